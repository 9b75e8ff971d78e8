"""torch.ops.vectra.residual_norm_8bit past 4096 columns, where a lane holds two or four
chunks of a row: codes and scales bit for bit those of the unrounded norm, h the same as
residual_norm's, with every kind of gate and every pair of types."""

import pytest
import torch

from oracle import block as oracle
from vectra_amd.kernels import block

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)]
# Odd ones end within a block, and leave blocks and scales of a word to be filled.
WIDTHS = [4097, 4224, 5000, 8191, 8192, 8193, 9001, 12300, 16383, 16384]


def arguments(width, dtype, stream, gate, norm, post, device, p=0.0):
    gen = torch.Generator().manual_seed(width)

    def normal(*sizes, to=F32, plus=0.0, factor=1.0):
        return torch.randn(*sizes, generator=gen).mul(factor).add(plus).to(to).to(device)

    t = dict(x=normal(3, 2, width, to=dtype), residual=normal(3, 2, width, to=stream, factor=2.0), weight=normal(width, factor=0.3, plus=1.0),
             bias=normal(width, factor=0.3), norm=norm, post=post, residual_scale=0.75, p=p)
    if post != 'none':
        t.update(post_weight=normal(width, factor=0.3, plus=0.5), post_bias=normal(width, factor=0.3))
    if gate is not None:
        t['gate'] = normal(*{'vector': (width,), 'sequence': (3, 1, width), 'row': (3, 2, width)}[gate], factor=0.5, plus=0.2)
    if p:
        t['rng'] = torch.tensor([width, 1], device=device)
    return t


def check(t):
    wide = {**t, 'x': t['x'].float(), 'residual': t['residual'].float()}
    n = block.residual_norm(**wide)[1]  # in fp32, as both have it before they round
    h, codes, scales = block.residual_norm_8bit(**t)
    assert torch.equal(h, block.residual_norm(**t)[0])
    width = n.shape[-1]
    want = oracle.quantize(n.reshape(-1, width), 1)
    assert codes.shape == (3, 2, want[0].shape[1]) and scales.shape == (3, 2, want[1].shape[1])
    assert torch.equal(codes.view(torch.uint8).cpu().reshape(6, -1), want[0])
    assert torch.equal(scales.view(torch.uint8).cpu().reshape(6, -1), want[1])


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('gate', [None, 'vector', 'sequence', 'row'])
@pytest.mark.parametrize('width', WIDTHS)
def test_widths_and_gates(width, gate, device):
    check(arguments(width, BF16, F32, gate, 'layer', 'rms', device))
    check(arguments(width, F32, F32, gate, 'rms', 'none', device, p=0.25))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype,stream', TYPES, ids=str)
@pytest.mark.parametrize('width', [4097, 8192, 9001, 16383])
def test_types(width, dtype, stream, device):
    check(arguments(width, dtype, stream, 'sequence', 'rms', 'layer', device))
    check(arguments(width, dtype, stream, None, 'layer', 'none', device, p=0.5))
