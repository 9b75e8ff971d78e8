"""Sums of an 8-bit layer in which large products cancel: within the bounds that the
contract's words on the matrix cores give, element by element, and exact in fp32 sums
where it promises them."""

import pytest
import torch

from oracle import block as oracle
from vectra_amd.kernels import block

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def cancelling(rows, depth, n, device):
    """Codes of ordinary values beside pairs of columns whose products are some hundred
    times a result and cancel: within 16 of a block, within a block, and across blocks."""
    gen = torch.Generator().manual_seed(rows)
    x, w = torch.randn(rows, depth, generator=gen), torch.randn(n, depth, generator=gen) * depth ** -0.5
    for a, b in ((0, 1), (5, 40), (17, 127), (64, 300), (200, depth - 1)):
        x[:, a] = x[:, b] = 100 * torch.randn(rows, generator=gen).abs().add(0.5)
        w[:, a] *= 8
        w[:, b] = -w[:, a]
    xc, xs = block.quantize_blocks(x.to(device))
    wc, ws = block.quantize_blocks(w.to(device), True)
    xv, wv = oracle.values(xc, xs, 1, depth), oracle.values(wc, ws, 128, depth)
    z = xv @ wv.t()
    assert float((xv.abs().amax(1) * wv.abs().max() / z.abs().median(1).values).median()) > 100
    return (xc, wc, ws, xs), (xv, wv)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('rows,depth,n', [(1, 512, 40), (17, 1024, 70), (32, 512, 300), (33, 512, 130), (300, 1024, 257),
                                          (1030, 2048, 520)])
def test_large_products_that_cancel(rows, depth, n, dtype, device):
    (xc, wc, ws, xs), (xv, wv) = cancelling(rows, depth, n, device)
    cores = device != 'cpu' and dtype != F32 and rows > 32
    y = block.linear_8bit(xc, wc, ws, scales=xs, dtype=dtype)
    oracle.assert_within(y, *oracle.layer(xv, wv, dtype=dtype, cores=cores))
    y = block.gated_linear_8bit(xc, wc, ws, activation='relu', scales=xs, dtype=dtype) if n % 2 == 0 else None
    if y is not None:
        oracle.assert_within(y, *oracle.layer(xv, wv, activation='relu', gated=True, dtype=dtype, cores=cores))


@pytest.mark.gpu
def test_fp32_results_are_the_way_to_exact_sums():
    """The same call with fp32 results, rounded by the program: within fp32's error of the
    sum, whatever the rows."""
    (xc, wc, ws, xs), (xv, wv) = cancelling(300, 1024, 257, 'cuda')
    y = block.linear_8bit(xc, wc, ws, scales=xs, dtype=F32).to(BF16)
    want, bound = oracle.layer(xv, wv)
    oracle.assert_within(y, want, bound + oracle.rounding(want, bound, BF16))
