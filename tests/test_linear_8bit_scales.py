"""What scale bytes stand for in an 8-bit layer, whoever made them: 2^(byte - 127), and
NaN for 255."""

import pytest
import torch

from oracle import block as oracle
from vectra_amd.kernels import block

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ROWS = [3, 20, 100, 400]  # single tokens, a few rows, small and larger tiles


def operands(rows, x_byte, w_byte, device, depth=256, n=150):
    """Small integers, and whole blocks of one scale byte."""
    gen = torch.Generator().manual_seed(rows)
    x = torch.randint(-4, 5, (rows, depth), generator=gen).float()
    w = torch.randint(-2, 3, (n, depth), generator=gen).float()
    xs, ws = torch.full((rows, 4), x_byte, dtype=torch.uint8), torch.full((2, 4), w_byte, dtype=torch.uint8)
    return [t.to(device) for t in (x.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn), xs, ws)]


def run(xc, wc, xs, ws, dtype):
    return block.linear_8bit(xc, wc, ws.view(torch.float8_e8m0fnu), scales=xs.view(torch.float8_e8m0fnu), dtype=dtype)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows', ROWS)
def test_every_power_of_two(rows, dtype, device):
    """Integers times powers of two, bit for bit, also below the least power that
    quantize_blocks makes (byte 10) and below fp32's normal range (2^-127): in products
    that are large enough, nothing is flushed."""
    for w_byte, x_byte in ((0, 247), (1, 247), (9, 246), (10, 240), (127, 127), (247, 10), (253, 1), (248, 4), (250, 10)):
        xc, wc, xs, ws = operands(rows, x_byte, w_byte, device)
        want = oracle.values(xc, xs, 1, 256) @ oracle.values(wc, ws, 128, 256).t()
        assert torch.equal(run(xc, wc, xs, ws, dtype).cpu(), want.to(dtype)), (w_byte, x_byte)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows', ROWS)
def test_255_is_nan(rows, dtype, device):
    for of_weight in (False, True):
        xc, wc, xs, ws = operands(rows, 127, 127, device)
        (ws if of_weight else xs)[1, 1] = 255
        y = run(xc, wc, xs, ws, dtype)
        bad = torch.zeros(rows, 150, dtype=torch.bool)
        if of_weight:
            bad[:, 128:] = True
        else:
            bad[1] = True
        assert torch.equal(torch.isnan(y).cpu(), bad)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('rows', ROWS)
def test_bytes_behind_the_width_are_not_used(rows, device):
    xc, wc, xs, ws = operands(rows, 127, 127, device)
    want = run(xc, wc, xs, ws, torch.bfloat16)
    for byte in (0, 200, 255):
        xs[:, 2:] = byte
        ws[:, 2:] = byte
        assert torch.equal(run(xc, wc, xs, ws, torch.bfloat16), want)
