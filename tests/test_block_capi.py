"""The block C ABI: its argument checks and workspace sizes on the host (those calls
are refused, or only ask for a size), and its calls against the operators."""

import ctypes
import os
import re

import pytest
import torch

from vectra_amd.kernels import _native
from vectra_amd.kernels import block_capi as capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
POINTER = 1 << 20  # 256-byte aligned; never read: no call of the host tests reaches a kernel


def forward_args(**changes):
    a = capi.NormArgs(struct_size=ctypes.sizeof(capi.NormArgs), x=POINTER, residual=POINTER, h=POINTER, n=POINTER,
                      dtype=capi.BF16, stream_dtype=capi.F32, norm=1, post=0, eps=1e-6, residual_scale=1.0, rows=64,
                      width=128, gate_rows=64, x_stride=128, residual_stride=128, gate_stride=128, h_stride=128,
                      n_stride=128)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


def grad_args(**changes):
    a = capi.NormGradArgs(struct_size=ctypes.sizeof(capi.NormGradArgs), grad_h=POINTER, grad_n=POINTER, x=POINTER,
                          residual=POINTER, h=POINTER, dx=POINTER, dresidual=POINTER, dweight=POINTER,
                          dtype=capi.BF16, stream_dtype=capi.F32, norm=2, post=0, eps=1e-6, residual_scale=1.0, rows=64,
                          width=128, gate_rows=64, grad_h_stride=128, grad_n_stride=128, x_stride=128,
                          residual_stride=128, h_stride=128, gate_stride=128, dx_stride=128, dresidual_stride=128,
                          dgate_stride=128)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


def linear_args(**changes):
    a = capi.Linear8Args(struct_size=ctypes.sizeof(capi.Linear8Args), x=POINTER, weight=POINTER, weight_scales=POINTER,
                         out=POINTER, dtype=capi.BF16, bias_dtype=capi.BF16, rows=64, width=200, width_out=96,
                         x_stride=200, residual_stride=96, out_stride=96)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


def linear_size(args):
    return _native.block_library().vectra_linear8_workspace_bytes(ctypes.byref(args))


def grad_size(args):
    return _native.block_library().vectra_norm_backward_workspace_bytes(ctypes.byref(args))


def test_exports_match_the_header():
    with open(os.path.join(ROOT, 'include', 'vectra_block.h'), encoding='utf-8') as f:
        text = re.sub(r'/\*.*?\*/', '', f.read(), flags=re.S)
    declared = set(re.findall(r'\b(vectra_\w+)\s*\(', text))
    assert declared == set(capi.EXPORTS)
    lib = _native.block_library()
    for name in capi.EXPORTS:
        assert hasattr(lib, name)
    assert capi.abi_version() == (1, 0)
    texts = [capi.status_string(s) for s in range(9)]
    assert len(set(texts)) == 9 and capi.status_string(99) == 'unknown status'


BAD_NORM = [
    (dict(struct_size=8), capi.ERR_BAD_STRUCT),
    (dict(dtype=3), capi.ERR_BAD_DTYPE),
    (dict(stream_dtype=capi.F16), capi.ERR_BAD_DTYPE),
    (dict(dtype=capi.F32, stream_dtype=capi.BF16), capi.ERR_BAD_DTYPE),
    (dict(norm=0), capi.ERR_BAD_OPTION),
    (dict(norm=3), capi.ERR_BAD_OPTION),
    (dict(post=-1), capi.ERR_BAD_OPTION),
    (dict(threshold=65536), capi.ERR_BAD_OPTION),
    (dict(threshold=-1), capi.ERR_BAD_OPTION),
    (dict(eps=-1e-6), capi.ERR_BAD_OPTION),
    (dict(eps=float('nan')), capi.ERR_BAD_OPTION),
    (dict(eps=float('inf')), capi.ERR_BAD_OPTION),
    (dict(rows=-1), capi.ERR_BAD_SHAPE),
    (dict(width=-1), capi.ERR_BAD_SHAPE),
    (dict(rows=1 << 31), capi.ERR_TOO_LARGE),
    (dict(rows=1 << 28), capi.ERR_TOO_LARGE),
    (dict(rows=1 << 62), capi.ERR_TOO_LARGE),
    (dict(width=capi.NORM_WIDTH + 1, x_stride=1 << 15, residual_stride=1 << 15), capi.ERR_TOO_LARGE),
    (dict(weight=POINTER, weight_dtype=capi.F16), capi.ERR_BAD_DTYPE),
    (dict(gate=POINTER, gate_dtype=capi.F16), capi.ERR_BAD_DTYPE),
    (dict(post_bias=POINTER, post=1, post_bias_dtype=7), capi.ERR_BAD_DTYPE),
    (dict(gate=POINTER, gate_dtype=capi.F32, gate_rows=0), capi.ERR_BAD_SHAPE),
    (dict(gate=POINTER, gate_dtype=capi.F32, gate_rows=32, gate_stride=127), capi.ERR_BAD_SHAPE),
    (dict(threshold=7), capi.ERR_NULL_ARGUMENT),
]


@pytest.mark.parametrize('changes,want', BAD_NORM + [
    (dict(x=None), capi.ERR_NULL_ARGUMENT),
    (dict(residual=None), capi.ERR_NULL_ARGUMENT),
    (dict(h=None), capi.ERR_NULL_ARGUMENT),
    (dict(n=None), capi.ERR_NULL_ARGUMENT),
    (dict(n=None, codes=POINTER), capi.ERR_NULL_ARGUMENT),
    (dict(n=None, codes=POINTER + 8, scales=POINTER), capi.ERR_BAD_SHAPE),
    (dict(x_stride=127), capi.ERR_BAD_SHAPE),
    (dict(n_stride=-1), capi.ERR_BAD_SHAPE),
    (dict(h_stride=1 << 60), capi.ERR_TOO_LARGE),
], ids=str)
def test_norm_refusals(changes, want):
    assert _native.block_library().vectra_norm_forward(ctypes.byref(forward_args(**changes)), None) == want


@pytest.mark.parametrize('changes,want', BAD_NORM + [
    (dict(h=None), capi.ERR_NULL_ARGUMENT),
    (dict(post=1, x=None), capi.ERR_NULL_ARGUMENT),
    (dict(gate=POINTER, gate_dtype=capi.F32, residual=None), capi.ERR_NULL_ARGUMENT),
    (dict(dgate=POINTER, gate_dtype=capi.F32), capi.ERR_NULL_ARGUMENT),
    (dict(dpost_weight=POINTER, post_weight_dtype=capi.F32), capi.ERR_BAD_OPTION),
    (dict(dweight=POINTER, weight_dtype=capi.F16), capi.ERR_BAD_DTYPE),
    (dict(grad_n_stride=127), capi.ERR_BAD_SHAPE),
    (dict(dx_stride=0), capi.ERR_BAD_SHAPE),
    (dict(gate=POINTER, gate_dtype=capi.F32, gate_rows=1, dgate=POINTER, dgate_stride=1), capi.ERR_BAD_SHAPE),
], ids=str)
def test_norm_gradient_refusals(changes, want):
    args = grad_args(**changes)
    assert grad_size(args) == -want
    assert _native.block_library().vectra_norm_backward(ctypes.byref(args), None, 0, None) == want


@pytest.mark.parametrize('changes,want', [
    (dict(struct_size=8), capi.ERR_BAD_STRUCT),
    (dict(dtype=3), capi.ERR_BAD_DTYPE),
    (dict(bias=POINTER, bias_dtype=capi.F16), capi.ERR_BAD_DTYPE),
    (dict(activation=5), capi.ERR_BAD_OPTION),
    (dict(activation=-1), capi.ERR_BAD_OPTION),
    (dict(gated=2), capi.ERR_BAD_SHAPE),
    (dict(gated=1, residual=POINTER), capi.ERR_BAD_SHAPE),
    (dict(rows=-1), capi.ERR_BAD_SHAPE),
    (dict(width=-1), capi.ERR_BAD_SHAPE),
    (dict(width_out=-1), capi.ERR_BAD_SHAPE),
    (dict(rows=1 << 31), capi.ERR_TOO_LARGE),
    (dict(width_out=1 << 22), capi.ERR_TOO_LARGE),
    (dict(width_out=1 << 62), capi.ERR_TOO_LARGE),
    (dict(width_out=(1 << 62) + 8, gated=1), capi.ERR_TOO_LARGE),
    (dict(width=1 << 21, x_stride=1 << 21, width_out=1 << 14, gated=1), capi.ERR_TOO_LARGE),
    (dict(x=None), capi.ERR_NULL_ARGUMENT),
    (dict(x=None, codes=POINTER), capi.ERR_NULL_ARGUMENT),
    (dict(x=None, codes=POINTER + 8, scales=POINTER), capi.ERR_BAD_SHAPE),
    (dict(x=None, codes=POINTER, scales=POINTER + 2), capi.ERR_BAD_SHAPE),
    (dict(weight=None), capi.ERR_NULL_ARGUMENT),
    (dict(weight_scales=None), capi.ERR_NULL_ARGUMENT),
    (dict(weight=POINTER + 8), capi.ERR_BAD_SHAPE),
    (dict(weight_scales=POINTER + 1), capi.ERR_BAD_SHAPE),
    (dict(out=None), capi.ERR_NULL_ARGUMENT),
    (dict(x_stride=199), capi.ERR_BAD_SHAPE),
    (dict(out_stride=95), capi.ERR_BAD_SHAPE),
    (dict(residual=POINTER, residual_stride=95), capi.ERR_BAD_SHAPE),
], ids=str)
def test_linear_refusals(changes, want):
    args = linear_args(**changes)
    assert linear_size(args) == -want
    assert _native.block_library().vectra_linear8_forward(ctypes.byref(args), None, 0, None) == want


def test_dropout_and_quantize_refusals():
    lib = _native.block_library()

    def dropout(x=POINTER, dtype=capi.F32, rows=4, width=64, stride=64, y=POINTER, y_stride=64, threshold=100, rng=POINTER):
        return lib.vectra_dropout(x, dtype, rows, width, stride, y, y_stride, threshold, rng, 0, None)

    assert dropout(dtype=3) == capi.ERR_BAD_DTYPE
    assert dropout(threshold=65536) == dropout(threshold=-1) == capi.ERR_BAD_OPTION
    assert dropout(rows=-1) == dropout(stride=63) == dropout(y_stride=63) == capi.ERR_BAD_SHAPE
    assert dropout(x=None) == dropout(y=None) == dropout(rng=None) == capi.ERR_NULL_ARGUMENT
    assert dropout(rows=1 << 30, width=1) == dropout(rows=1, width=1 << 22) == capi.ERR_TOO_LARGE
    assert dropout(rows=0, x=None) == dropout(width=0, y=None) == capi.OK

    def quantize(x=POINTER, dtype=capi.F32, rows=4, width=64, stride=64, tiles=0, codes=POINTER, scales=POINTER):
        return lib.vectra_blocks_quantize(x, dtype, rows, width, stride, tiles, codes, scales, None)

    assert quantize(dtype=-1) == capi.ERR_BAD_DTYPE
    assert quantize(tiles=2) == capi.ERR_BAD_OPTION
    assert quantize(width=-1) == quantize(stride=63) == quantize(codes=POINTER + 8) == capi.ERR_BAD_SHAPE
    assert quantize(x=None) == quantize(codes=None) == quantize(scales=None) == capi.ERR_NULL_ARGUMENT
    assert quantize(rows=1 << 31) == capi.ERR_TOO_LARGE
    assert quantize(rows=0, x=None, tiles=1) == capi.OK


def test_null_arguments():
    lib = _native.block_library()
    assert lib.vectra_norm_forward(None, None) == capi.ERR_NULL_ARGUMENT
    for name in ('vectra_norm_backward', 'vectra_linear8_forward'):
        assert getattr(lib, name)(None, None, 0, None) == capi.ERR_NULL_ARGUMENT
    assert lib.vectra_norm_backward_workspace_bytes(None) == -capi.ERR_NULL_ARGUMENT
    assert lib.vectra_linear8_workspace_bytes(None) == -capi.ERR_NULL_ARGUMENT


def test_a_missing_or_small_workspace_is_refused():
    lib = _native.block_library()
    for args, call, size in ((grad_args(weight_dtype=capi.F32), lib.vectra_norm_backward, grad_size),
                             (linear_args(), lib.vectra_linear8_forward, linear_size)):
        need = size(args)
        assert need >= 128 * 4
        for workspace, n in ((None, 0), (POINTER, need - 1), (POINTER + 16, need)):
            assert call(ctypes.byref(args), workspace, n, None) == capi.ERR_WORKSPACE


def test_the_workspace_holds_what_is_asked_for():
    assert grad_size(grad_args(dweight=None)) == 0
    one = grad_size(grad_args(weight_dtype=capi.F32))
    assert grad_size(grad_args(weight_dtype=capi.F32, dbias=POINTER, bias_dtype=capi.F32)) == 2 * one
    # 8-bit rows of x, 200 wide: 64 of 256 codes and 4 scales; none where the caller has them.
    assert linear_size(linear_args()) >= 64 * 256 + 64 * 4
    assert linear_size(linear_args(x=None, codes=POINTER, scales=POINTER)) < linear_size(linear_args())
    assert linear_size(linear_args(rows=1)) == 0


def test_nothing_to_do_is_no_error():
    lib = _native.block_library()
    for args in (forward_args(rows=0, x=None, h=None), forward_args(width=0, residual=None)):
        assert lib.vectra_norm_forward(ctypes.byref(args), None) == capi.OK
    for args in (grad_args(width=0), grad_args(dx=None, dresidual=None, dweight=None), grad_args(rows=0, dweight=None)):
        assert lib.vectra_norm_backward(ctypes.byref(args), None, 0, None) == capi.OK
    for args in (linear_args(rows=0, x=None, out=None), linear_args(width_out=0, weight=None, out=None)):
        assert lib.vectra_linear8_forward(ctypes.byref(args), None, 0, None) == capi.OK


def test_the_binding_fills_the_structures():
    x, r, gate = torch.zeros(6, 8, dtype=torch.bfloat16), torch.zeros(6, 16)[:, :8], torch.zeros(2, 8)
    a = capi.make_norm_args(x, r, h=r, n=x, gate=gate, gate_rows=3, norm='layer', post='rms', p=0.5)
    assert (a.rows, a.width, a.gate_rows, a.norm, a.post, a.threshold) == (6, 8, 3, 2, 1, 32768)
    assert (a.dtype, a.stream_dtype, a.gate_dtype, a.weight_dtype) == (capi.BF16, capi.F32, capi.F32, capi.BF16)
    assert (a.x_stride, a.residual_stride, a.h_stride, a.n_stride, a.gate_stride) == (8, 16, 16, 8, 8)
    g = capi.make_norm_grad_args(x, None, h=r, dx=x, dresidual=r, dweight=gate[0])
    assert (g.grad_h, g.stream_dtype, g.weight_dtype, g.gate_rows, g.dresidual_stride) == (None, capi.F32, capi.F32, 6, 16)
    codes = torch.zeros(6, 128, dtype=torch.uint8)
    l = capi.make_linear8_args(codes, codes, codes, out=x, scales=codes, width=100, activation='silu', gated=True)
    assert (l.x, l.width, l.width_out, l.activation, l.gated, l.dtype) == (None, 100, 8, 4, 1, capi.BF16)


# ----------------------------------------------------------------------- on the GPU


def _strided(*shape, dtype, lead=3):
    """A matrix in a wider one, off its start by a few elements."""
    rows, width = shape
    return torch.randn(rows, width + 24, device='cuda').to(dtype)[:, lead:lead + width]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16], ids=str)
def test_dropout_through_the_c_abi(dtype):
    torch.manual_seed(0)
    rng = torch.tensor([5, 9], device='cuda')
    x = _strided(33, 77, dtype=dtype)
    want = torch.ops.vectra.dropout(x, 0.25, rng, 3)
    wide = torch.full((33, 90), 7.0, device='cuda', dtype=dtype)
    out = wide[:, 5:82]
    capi.dropout(x, 0.25, rng, out=out, stream_id=3)
    assert torch.equal(out, want)
    assert (wide[:, :5] == 7).all() and (wide[:, 82:] == 7).all()
    capi.dropout(x, 0.25, rng, out=x, stream_id=3)  # in place
    assert torch.equal(x, want)
    with pytest.raises(capi.BlockError) as e:
        capi.dropout(x, 1.0, rng, out=x)
    assert e.value.status == capi.ERR_BAD_OPTION


@pytest.mark.gpu
@pytest.mark.parametrize('gate_rows,post', [(None, 'none'), (10, 'layer'), (1, 'rms')], ids=str)
def test_norms_through_the_c_abi(gate_rows, post):
    torch.manual_seed(1)
    rows, width = 30, 203
    x, r = _strided(rows, width, dtype=torch.bfloat16), _strided(rows, width, dtype=torch.float32, lead=1)
    w, b = torch.randn(width, device='cuda'), torch.randn(width, device='cuda', dtype=torch.bfloat16)
    pw = torch.randn(width, device='cuda') if post != 'none' else None
    gate = None if gate_rows is None else torch.randn(rows // gate_rows, width, device='cuda')
    rng = torch.tensor([1, 2], device='cuda')
    options = dict(norm='layer', post=post, eps=1e-5, residual_scale=0.5, p=0.125, rng=rng)

    # Through the operators, with the rows in groups as the gate has them.
    groups = 1 if gate is None else gate.shape[0]
    leaves = [t.detach().clone().requires_grad_() if t is not None else None
              for t in (x.reshape(groups, -1, width), r.reshape(groups, -1, width), w, b,
                        None if gate is None else gate[:, None], pw)]
    h, n = torch.ops.vectra.residual_norm(*leaves[:5], leaves[5], None, **options)
    gh, gn = torch.randn_like(h), torch.randn_like(n)
    given = [t for t in leaves if t is not None]
    wanted = torch.autograd.grad([h, n], given, [gh, gn])

    out_h, out_n = torch.empty(rows, width + 5, device='cuda')[:, :width], torch.empty_like(n).reshape(rows, width)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    capi.norm_forward(x, r, h=out_h, n=out_n, weight=w, bias=b, gate=gate, post_weight=pw, gate_rows=gate_rows,
                      stream=stream.cuda_stream, **options)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(out_h, h.reshape(rows, width)) and torch.equal(out_n, n.reshape(rows, width))

    grads = dict(dx=torch.empty_like(out_n), dresidual=torch.empty_like(out_h), dweight=torch.empty_like(w),
                 dbias=torch.empty_like(b))
    if gate is not None:
        grads['dgate'] = torch.empty_like(gate)
    if pw is not None:
        grads['dpost_weight'] = torch.empty_like(pw)
    branch = dict(x=x, residual=r) if gate is not None or post != 'none' else dict(h=out_h)
    capi.norm_backward(gn.reshape(rows, width), gh.reshape(rows, width), weight=w, gate=gate, post_weight=pw,
                       gate_rows=gate_rows, **branch, **grads, **options)
    for got, want in zip(grads.values(), wanted):
        assert torch.equal(got, want.reshape(got.shape))
    with pytest.raises(capi.BlockError) as e:
        capi.norm_backward(gn.reshape(rows, width), gh.reshape(rows, width), weight=w, gate=gate, post_weight=pw,
                           gate_rows=gate_rows, workspace=torch.empty(256, dtype=torch.uint8, device='cuda'),
                           **branch, **grads, **options)
    assert e.value.status == capi.ERR_WORKSPACE


@pytest.mark.gpu
@pytest.mark.parametrize('rows', [5, 70])
@pytest.mark.parametrize('gated', [False, True])
def test_8_bit_layers_through_the_c_abi(rows, gated):
    torch.manual_seed(2)
    width, out_width = 200, 96
    x = _strided(rows, width, dtype=torch.float16)
    w = torch.randn((1 + gated) * out_width, width, device='cuda')
    codes = torch.empty(w.shape[0], 256, dtype=torch.float8_e4m3fn, device='cuda')
    scales = torch.empty((w.shape[0] + 127) // 128, 4, dtype=torch.uint8, device='cuda')
    capi.quantize(w, codes=codes, scales=scales, tiles=True)
    want_codes, want_scales = torch.ops.vectra.quantize_blocks(w, True)
    assert torch.equal(codes.view(torch.uint8), want_codes.view(torch.uint8))
    assert torch.equal(scales, want_scales.view(torch.uint8))
    op = torch.ops.vectra.gated_linear_8bit if gated else torch.ops.vectra.linear_8bit
    want = op(x, want_codes, want_scales, activation='silu')
    out = torch.zeros(rows, out_width + 9, dtype=torch.float16, device='cuda')
    capi.linear8(x, codes, scales, out=out[:, 2:2 + out_width], activation='silu', gated=gated)
    assert torch.equal(out[:, 2:2 + out_width], want)
    assert not out[:, :2].any() and not out[:, 2 + out_width:].any()

    # Rows in 8 bits from a norm, whose h and n the program has in another call.
    r = torch.randn(rows, width, device='cuda', dtype=torch.float16)
    h = torch.empty_like(r)
    row_codes = torch.empty(rows, 256, dtype=torch.float8_e4m3fn, device='cuda')
    row_scales = torch.empty(rows, 4, dtype=torch.uint8, device='cuda')
    capi.norm_forward(x, r, h=h, codes=row_codes, scales=row_scales)
    want_h, want_c, want_s = torch.ops.vectra.residual_norm_8bit(x, r)
    assert torch.equal(h, want_h) and torch.equal(row_codes.view(torch.uint8), want_c.view(torch.uint8))
    assert torch.equal(row_scales, want_s.view(torch.uint8))
    out = torch.empty(rows, out_width, dtype=torch.float16, device='cuda')
    capi.linear8(row_codes, codes, scales, out=out, scales=row_scales, width=width, gated=gated)
    assert torch.equal(out, op(want_c, want_codes, want_scales, activation='none', scales=want_s, dtype=torch.float16))
