"""The dense C ABI's argument checks and workspace sizes (host only: every call
here is refused, or only asks for a size)."""

import ctypes
import os
import re

import pytest
import torch

from vectra_amd.kernels import _native
from vectra_amd.kernels import dense_capi as capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
POINTER = 1 << 20  # 16-byte aligned; never read: no call here reaches a kernel


def forward_args(**changes):
    a = capi.DenseArgs(struct_size=ctypes.sizeof(capi.DenseArgs), x=POINTER, weight=POINTER, bias=None, residual=None,
                       out=POINTER, dtype=capi.BF16, bias_dtype=capi.BF16, activation=0, gated=0, rows=64,
                       width_in=128, width_out=256, x_stride=128, weight_stride=128, residual_stride=256,
                       out_stride=256)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


def grad_args(**changes):
    a = capi.DenseGradArgs(struct_size=ctypes.sizeof(capi.DenseGradArgs), x=POINTER, weight=POINTER, grad=POINTER,
                           dx=POINTER, dweight=POINTER, dbias=POINTER, dtype=capi.BF16, bias_dtype=capi.BF16,
                           activation=2, gated=0, rows=64, width_in=128, width_out=256, x_stride=128,
                           weight_stride=128, grad_stride=256, dx_stride=128, dweight_stride=128)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


def status(args):
    """The size query's status: 0, or what the call itself would return."""
    lib = _native.dense_library()
    name = 'vectra_dense_forward' if isinstance(args, capi.DenseArgs) else 'vectra_dense_backward'
    need = getattr(lib, name + '_workspace_bytes')(ctypes.byref(args))
    return max(0, -need)


def test_exports_match_the_header():
    with open(os.path.join(ROOT, 'include', 'vectra_dense.h'), encoding='utf-8') as f:
        text = re.sub(r'/\*.*?\*/', '', f.read(), flags=re.S)
    declared = set(re.findall(r'\b(vectra_\w+)\s*\(', text))
    assert declared == set(capi.EXPORTS)
    lib = _native.dense_library()
    for name in capi.EXPORTS:
        assert hasattr(lib, name)
    assert capi.abi_version() == (1, 0)
    texts = [capi.status_string(s) for s in range(9)]
    assert len(set(texts)) == 9 and capi.status_string(99) == 'unknown status'


BAD_FORWARD = [
    (dict(struct_size=8), capi.ERR_BAD_STRUCT),
    (dict(dtype=3), capi.ERR_BAD_DTYPE),
    (dict(bias=POINTER, bias_dtype=capi.F16), capi.ERR_BAD_DTYPE),
    (dict(activation=5), capi.ERR_BAD_ACTIVATION),
    (dict(activation=-1), capi.ERR_BAD_ACTIVATION),
    (dict(gated=2), capi.ERR_BAD_SHAPE),
    (dict(gated=1, residual=POINTER), capi.ERR_BAD_SHAPE),
    (dict(rows=-1), capi.ERR_BAD_SHAPE),
    (dict(width_in=-1), capi.ERR_BAD_SHAPE),
    (dict(x=None), capi.ERR_NULL_ARGUMENT),
    (dict(weight=None), capi.ERR_NULL_ARGUMENT),
    (dict(out=None), capi.ERR_NULL_ARGUMENT),
    (dict(x_stride=127), capi.ERR_BAD_SHAPE),
    (dict(weight_stride=0), capi.ERR_BAD_SHAPE),
    (dict(out_stride=255), capi.ERR_BAD_SHAPE),
    (dict(residual=POINTER, residual_stride=255), capi.ERR_BAD_SHAPE),
    (dict(rows=1 << 31), capi.ERR_TOO_LARGE),
    (dict(width_out=1 << 22, out_stride=1 << 22), capi.ERR_TOO_LARGE),
    (dict(rows=1 << 29), capi.ERR_TOO_LARGE),
    (dict(x_stride=1 << 22), capi.ERR_TOO_LARGE),
    (dict(x_stride=1 << 60), capi.ERR_TOO_LARGE),
    (dict(weight_stride=1 << 60), capi.ERR_TOO_LARGE),
    (dict(gated=1, weight_stride=1 << 22), capi.ERR_TOO_LARGE),
]


@pytest.mark.parametrize('changes,want', BAD_FORWARD, ids=str)
def test_forward_refusals(changes, want):
    args = forward_args(**changes)
    assert status(args) == want
    lib = _native.dense_library()
    assert lib.vectra_dense_forward(ctypes.byref(args), None, 0, None) == want


BAD_BACKWARD = [
    (dict(struct_size=8), capi.ERR_BAD_STRUCT),
    (dict(dtype=7), capi.ERR_BAD_DTYPE),
    (dict(bias_dtype=capi.F16), capi.ERR_BAD_DTYPE),
    (dict(activation=9), capi.ERR_BAD_ACTIVATION),
    (dict(gated=-1), capi.ERR_BAD_SHAPE),
    (dict(x=None), capi.ERR_NULL_ARGUMENT),
    (dict(x=None, codes=POINTER), capi.ERR_NULL_ARGUMENT),
    (dict(x=None, codes=POINTER, scales=POINTER, codes_stride=127, scales_stride=4), capi.ERR_BAD_SHAPE),
    (dict(x=None, codes=POINTER, scales=POINTER, codes_stride=128, scales_stride=3), capi.ERR_BAD_SHAPE),
    (dict(weight=None), capi.ERR_NULL_ARGUMENT),
    (dict(grad=None), capi.ERR_NULL_ARGUMENT),
    (dict(grad_stride=200), capi.ERR_BAD_SHAPE),
    (dict(dx_stride=100), capi.ERR_BAD_SHAPE),
    (dict(dweight_stride=100), capi.ERR_BAD_SHAPE),
    (dict(grad_stride=1 << 22), capi.ERR_TOO_LARGE),
    (dict(rows=1 << 33), capi.ERR_TOO_LARGE),
]


@pytest.mark.parametrize('changes,want', BAD_BACKWARD, ids=str)
def test_backward_refusals(changes, want):
    args = grad_args(**changes)
    assert status(args) == want
    lib = _native.dense_library()
    assert lib.vectra_dense_backward(ctypes.byref(args), None, 0, None) == want


def test_null_arguments():
    lib = _native.dense_library()
    assert lib.vectra_dense_forward(None, None, 0, None) == capi.ERR_NULL_ARGUMENT
    assert lib.vectra_dense_forward_workspace_bytes(None) == -capi.ERR_NULL_ARGUMENT
    assert lib.vectra_dense_backward(None, None, 0, None) == capi.ERR_NULL_ARGUMENT
    assert lib.vectra_dense_backward_workspace_bytes(None) == -capi.ERR_NULL_ARGUMENT


def test_a_missing_or_small_workspace_is_refused():
    lib = _native.dense_library()
    args = grad_args()
    need = lib.vectra_dense_backward_workspace_bytes(ctypes.byref(args))
    assert need >= 64 * 256 * 2  # dz
    for workspace, size in ((None, 0), (POINTER, need - 1), (POINTER + 16, need)):
        assert lib.vectra_dense_backward(ctypes.byref(args), workspace, size, None) == capi.ERR_WORKSPACE


def test_unaligned_rows_need_room_for_their_copies():
    lib = _native.dense_library()
    size = lib.vectra_dense_forward_workspace_bytes
    plain = size(ctypes.byref(forward_args()))
    odd = size(ctypes.byref(forward_args(weight_stride=129)))
    assert odd >= plain


def test_nothing_to_do_is_no_error():
    lib = _native.dense_library()
    for args in (forward_args(rows=0, x=None, out=None), forward_args(width_out=0, weight=None, out=None)):
        assert lib.vectra_dense_forward(ctypes.byref(args), None, 0, None) == capi.OK
    args = grad_args(dx=None, dweight=None, dbias=None)
    assert lib.vectra_dense_backward(ctypes.byref(args), None, 0, None) == capi.OK


def test_an_input_that_no_gradient_reads_may_be_missing():
    lib = _native.dense_library()
    need = lib.vectra_dense_backward_workspace_bytes
    plain = dict(x=None, x_stride=0, activation=capi.ACTIVATIONS['none'], bias=None)
    assert need(ctypes.byref(grad_args(**plain, dweight=None))) >= 0
    assert need(ctypes.byref(grad_args(**plain))) == -capi.ERR_NULL_ARGUMENT
    plain['activation'] = capi.ACTIVATIONS['relu']
    assert need(ctypes.byref(grad_args(**plain, dweight=None))) == -capi.ERR_NULL_ARGUMENT


def test_row_refusals():
    lib = _native.dense_library()

    def quantize(x=POINTER, dtype=capi.F32, rows=4, width=64, stride=64, codes=POINTER, codes_stride=64, scales=POINTER,
                 scales_stride=2):
        return lib.vectra_rows_quantize(x, dtype, rows, width, stride, codes, codes_stride, scales, scales_stride, None)

    assert quantize(dtype=3) == capi.ERR_BAD_DTYPE
    assert quantize(rows=-1) == capi.ERR_BAD_SHAPE
    assert quantize(x=None) == capi.ERR_NULL_ARGUMENT
    assert quantize(scales=None) == capi.ERR_NULL_ARGUMENT
    assert quantize(stride=63) == capi.ERR_BAD_SHAPE
    assert quantize(codes_stride=63) == capi.ERR_BAD_SHAPE
    assert quantize(scales_stride=1) == capi.ERR_BAD_SHAPE
    assert quantize(rows=1 << 30) == capi.ERR_TOO_LARGE
    assert quantize(rows=0, x=None) == capi.OK

    def dequantize(codes=POINTER, dtype=capi.F32, rows=4, width=64, out=POINTER, out_stride=64):
        return lib.vectra_rows_dequantize(codes, 64, POINTER, 2, dtype, rows, width, out, out_stride, None)

    assert dequantize(dtype=-1) == capi.ERR_BAD_DTYPE
    assert dequantize(codes=None) == capi.ERR_NULL_ARGUMENT
    assert dequantize(out=None) == capi.ERR_NULL_ARGUMENT
    assert dequantize(out_stride=10) == capi.ERR_BAD_SHAPE
    assert dequantize(rows=1 << 30) == capi.ERR_TOO_LARGE
    assert dequantize(width=0) == capi.OK


def test_the_binding_fills_the_structures():
    x, w, out = torch.zeros(3, 8), torch.zeros(10, 8), torch.zeros(3, 5)
    a = capi.make_args(x, w, None, None, out, 'silu', True)
    assert (a.rows, a.width_in, a.width_out, a.gated, a.activation) == (3, 8, 5, 1, 4)
    g = capi.make_grad_args(out, x, w, None, x, w, None, 'gelu')
    assert (g.rows, g.width_in, g.width_out, g.dx_stride) == (3, 8, 5, 8)
