"""The block C ABI at the ends of its integers: no size is added to before it is known
to be in range."""

import ctypes

import pytest

from vectra_amd.kernels import _native
from vectra_amd.kernels import block_capi as capi

POINTER = 1 << 20  # never read: these calls only ask for a size, or are refused


@pytest.mark.parametrize('rows', [0, 1, 64])
@pytest.mark.parametrize('gate_rows', [2 ** 31, 2 ** 62, 2 ** 63 - 1])
def test_a_gate_row_for_more_rows_than_there_are(gate_rows, rows):
    """It serves all of them, as one for exactly as many does."""
    lib = _native.block_library()

    def size(of):
        a = capi.NormGradArgs(struct_size=ctypes.sizeof(capi.NormGradArgs), grad_n=POINTER, x=POINTER, residual=POINTER,
                              gate=POINTER, dgate=POINTER, dtype=capi.BF16, stream_dtype=capi.F32, gate_dtype=capi.F32,
                              norm=1, eps=1e-6, residual_scale=1.0, rows=rows, width=128, gate_rows=of, grad_n_stride=128,
                              x_stride=128, residual_stride=128, gate_stride=128, dgate_stride=128)
        return lib.vectra_norm_backward_workspace_bytes(ctypes.byref(a))

    assert size(gate_rows) == size(max(rows, 1)) >= 0
    a = capi.NormArgs(struct_size=ctypes.sizeof(capi.NormArgs), x=POINTER, residual=POINTER, h=POINTER, n=POINTER, gate=POINTER,
                      dtype=capi.BF16, stream_dtype=capi.F32, gate_dtype=capi.F32, norm=1, eps=1e-6, residual_scale=1.0,
                      rows=rows, width=128, gate_rows=gate_rows, x_stride=128, residual_stride=128, gate_stride=-1,
                      h_stride=128, n_stride=128)
    assert lib.vectra_norm_forward(ctypes.byref(a), None) == (capi.ERR_BAD_SHAPE if rows else capi.OK)
