"""Workspace sizes of products whose operands cannot be read in whole 16-byte
chunks and are copied first (host only: sizes are asked for, nothing runs)."""

import ctypes

import pytest

from tests.test_dense_capi import POINTER, forward_args, grad_args
from vectra_amd.kernels import _native
from vectra_amd.kernels import dense_capi as capi

# Wide enough for large tiles, which read whole chunks only.
ROWS = N = K = 4096


def need(args):
    lib = _native.dense_library()
    name = 'vectra_dense_forward' if isinstance(args, capi.DenseArgs) else 'vectra_dense_backward'
    size = getattr(lib, name + '_workspace_bytes')(ctypes.byref(args))
    assert size >= 0
    return size


def forward(**changes):
    return forward_args(**{**dict(rows=ROWS, width_in=K, width_out=N, x_stride=K, weight_stride=K, out_stride=N), **changes})


def backward(**changes):
    return grad_args(**{**dict(rows=ROWS, width_in=K, width_out=N, x_stride=K, weight_stride=K, grad_stride=N, dx_stride=K,
                               dweight_stride=K, activation=0), **changes})


COPIED = {
    'stride of W': (dict(weight_stride=K + 1), N * K * 2),
    'stride of x': (dict(x_stride=K + 3), ROWS * K * 2),
    'start of W': (dict(weight=POINTER + 2), N * K * 2),
    'start of x': (dict(x=POINTER + 8), ROWS * K * 2),
    'both': (dict(x=POINTER + 8, weight_stride=K + 1), (ROWS + N) * K * 2),
    'odd width': (dict(width_in=K - 3), (ROWS + N) * K * 2),
}


@pytest.mark.parametrize('name', COPIED)
def test_a_forward_call_asks_for_room_for_its_copies(name):
    changes, copied = COPIED[name]
    assert need(forward()) == 0
    assert need(forward(**changes)) >= copied
    lib = _native.dense_library()
    args = forward(**changes)
    # Refused before anything is launched.
    assert lib.vectra_dense_forward(ctypes.byref(args), POINTER, copied - 1, None) == capi.ERR_WORKSPACE
    assert lib.vectra_dense_forward(ctypes.byref(args), None, 0, None) == capi.ERR_WORKSPACE


@pytest.mark.parametrize('name', COPIED)
def test_a_backward_call_asks_for_room_for_its_copies(name):
    """x and W are read by one product each (dW, dx) of a layer without activation."""
    changes, copied = COPIED[name]
    assert need(backward(**changes)) >= need(backward()) + copied
    assert need(backward(grad=POINTER + 2)) >= need(backward()) + ROWS * N * 2


def test_a_copy_is_made_once_and_only_where_it_is_read():
    odd_x = dict(x=POINTER + 2)
    assert need(backward(**odd_x, dweight=None)) == need(backward(dweight=None))  # dx and db do not read x
    # With an activation x is read twice, for z and for dW, and copied once.
    slope = dict(activation=capi.ACTIVATIONS['gelu'])
    extra = need(backward(**odd_x, **slope)) - need(backward(**slope))
    assert ROWS * K * 2 <= extra < 2 * ROWS * K * 2


def test_small_calls_copy_nothing():
    assert need(forward_args(weight_stride=129)) == 0
    assert need(forward_args(x=POINTER + 2)) == 0
