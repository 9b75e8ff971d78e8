"""Refusals of the dense operators that need more than one dimension of rows."""

import pytest
import torch

from vectra_amd.kernels import dense

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
ops = torch.ops.vectra


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('sizes', [(3, 2, 2), (6, 2), (1, 6, 2), (2, 3, 1), (2, 3, 2, 1), (2,)], ids=str)
def test_scales_of_other_leading_dimensions_are_refused(sizes, device):
    """Codes [2, 3, 33]: as many rows in another shape are not their scales."""
    codes = torch.zeros(2, 3, 33, device=device).to(torch.float8_e4m3fn)
    scales = torch.ones(*sizes, device=device).to(torch.float8_e8m0fnu)
    with pytest.raises(RuntimeError, match='scales must be'):
        dense.dequantize_rows(codes, scales, torch.float32)
    w = torch.zeros(4, 33, device=device)
    with pytest.raises(RuntimeError, match='scales must be'):
        ops.linear_backward(torch.zeros(2, 3, 4, device=device), codes, scales, w, None, 'none', False, [True, True, False])
    fit = torch.ones(2, 3, 2, device=device).to(torch.float8_e8m0fnu)
    assert dense.dequantize_rows(codes, fit, torch.float32).shape == codes.shape
    ops.linear_backward(torch.zeros(2, 3, 4, device=device), codes, fit, w, None, 'none', False, [True, True, False])
