"""8-bit layers that are told their weight's width refuse an input of another."""

import pytest
import torch

from vectra_amd.kernels import block

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('layer', [block.linear_8bit, block.gated_linear_8bit])
def test_an_input_of_another_width(layer, device):
    gen = torch.Generator().manual_seed(0)
    for wide in (40, 128, 300):
        codes, scales = block.quantize_blocks(torch.randn(6, wide, generator=gen).to(device), True)
        for rows in (3, 50):
            x = torch.randn(rows, wide, generator=gen).to(device)
            want = layer(x, codes, scales)
            assert torch.equal(layer(x, codes, scales, width=wide), want)
            with pytest.raises(RuntimeError, match=f'x must be {wide} wide'):
                layer(x[:, :wide - 33], codes, scales, width=wide)
            # Without its width: as an input that ends in zeros.
            short = torch.nn.functional.pad(x[:, :wide - 3], (0, 3))
            assert torch.equal(layer(x[:, :wide - 3], codes, scales), layer(short, codes, scales))
            xc, xs = block.quantize_blocks(x)
            given = dict(scales=xs, dtype=torch.float32)
            assert torch.equal(layer(xc, codes, scales, **given, width=wide), layer(xc, codes, scales, **given))
            for other in (wide + 128, wide - 128, -1):
                with pytest.raises(RuntimeError, match='x must be .* wide'):
                    layer(xc, codes, scales, **given, width=other)


def test_opcheck():
    codes, scales = block.quantize_blocks(torch.randn(6, 40), True)
    for op in (torch.ops.vectra.linear_8bit.default, torch.ops.vectra.gated_linear_8bit.default):
        torch.library.opcheck(op, (torch.randn(3, 40), codes, scales), {'width': 40}, test_utils=('test_faketensor',))
