"""The dense operators' kernels for large sizes: rows whose tile spans more than
2^31 bytes."""

import pytest
import torch

from vectra_amd.kernels import dense  # noqa: F401  (registers the operators)

pytestmark = pytest.mark.gpu
ops = torch.ops.vectra


def test_gated_gradients_whose_tile_spans_more_than_31_bits():
    """dz of a gated layer is twice as wide as the gradient that the caller
    brings: 256 of its rows are 2.7 GB here.  Zeros but for a few columns, whose
    small integers fp32 holds exactly; the rows behind those that 2^31 bytes
    hold (the 205th of a tile on) are the ones in question."""
    rows, width_in, width_out = 1024, 256, 5 << 18
    at = torch.tensor([0, 1, 77, width_out // 2, width_out - 130, width_out - 1], device='cuda')
    gen = torch.Generator(device='cuda').manual_seed(1)

    def integers(*shape):
        return torch.randint(-2, 3, shape, generator=gen, device='cuda').float()

    x = integers(rows, width_in)
    gate, up = integers(len(at), width_in), integers(len(at), width_in)
    w = torch.zeros(2 * width_out, width_in, device='cuda')
    w[at], w[width_out + at] = gate, up
    dy = torch.zeros(rows, width_out, device='cuda')
    dy[:, at] = integers(rows, len(at))
    dx, dw = ops.linear_backward(dy, x, None, w, None, 'none', True, [True, True, False])
    xd, gd, ud, dyd = x.double(), gate.double(), up.double(), dy[:, at].double()
    da, du = dyd * (xd @ ud.t()), dyd * (xd @ gd.t())
    want = da @ gd + du @ ud
    assert float(want.abs().max()) < 2 ** 24 and float((da.t() @ xd).abs().max()) < 2 ** 24
    wrong = torch.nonzero((dx != want.float()).any(1)).flatten()
    assert len(wrong) == 0, f'{len(wrong)} rows of dx are wrong, the first ones {wrong[:4].tolist()}'
    assert torch.equal(dw[at], (da.t() @ xd).float()) and torch.equal(dw[width_out + at], (du.t() @ xd).float())
    assert int(torch.count_nonzero(dw)) == int(torch.count_nonzero(dw[at])) + int(torch.count_nonzero(dw[width_out + at]))
