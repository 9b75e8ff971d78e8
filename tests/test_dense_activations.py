"""The activations of the dense operators: the normal tail's polynomials (the
constants as they stand in the source, evaluated in 64 bits, against the tail
itself), and values far from zero."""

import os
import re

import numpy as np
import pytest
import torch
from scipy import special

from oracle import dense as oracle
from vectra_amd.kernels import dense

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'vectra_amd', 'csrc', 'dense',
                      'dense_common.h')


def constants(which):
    """(c, coefficients from the highest power down) as the fp32 values they are."""
    with open(SOURCE, encoding='utf-8') as f:
        text = f.read()
    body = re.search(r'void normal_tail\(.*?\n}', text, re.S).group(0).split('} else {')[which]
    c = re.search(r'fmaf\((\S+)f, a, 1\.f\)', body).group(1)
    powers = [re.search(r'p = (-?\d\S*)f;', body).group(1), *re.findall(r'fmaf\(p, t, (-?\S+)f\)', body)]
    return float(np.float32(c)), [float(np.float32(v)) for v in powers]


# The figures that the source states, to their last digit.
@pytest.mark.parametrize('which,degree,bound', [(0, 8, 3.05e-8), (1, 6, 8.25e-7)], ids=['fp32', '16 bits'])
def test_the_tail_is_as_close_as_the_source_says(which, degree, bound):
    c, powers = constants(which)
    assert len(powers) == degree + 1
    a = np.linspace(0.0, 14.0, 400001)
    t = 1.0 / (1.0 + c * a)
    # Phi(-a) / exp(-a^2 / 2) = erfcx(a / sqrt(2)) / 2, which underflows nowhere.
    want = special.erfcx(a / np.sqrt(2.0)) / 2
    assert np.abs(np.polyval(powers, t) * t / want - 1.0).max() < bound


FAR = [30.0, 1e3, 1e9, 1e13, 4e18, 1e19, 1e20, 1e30, 3e38]


@pytest.mark.parametrize('device', ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize('activation', dense.ACTIVATIONS)
@pytest.mark.parametrize('gated', [False, True])
def test_far_from_zero_an_activation_is_the_identity_or_zero(gated, activation, dtype, device):
    """z and slope 1 on one side, 0 and 0 on the other (none: z and 1), up to the
    type's largest values: exp(-30) z is below fp32's half step of z, and the
    other side's exp(-30) 30 below 1e-11."""
    z = torch.tensor([*FAR, *(-v for v in FAR)]).to(dtype).to(device)
    b = torch.zeros(2 if gated else 1, dtype=dtype, device=device)
    w = torch.ones(1, 1, dtype=dtype, device=device)
    if gated:  # an up projection of 1
        w = torch.tensor([[1.0], [0.0]], dtype=dtype, device=device)
        b[1] = 1.0
    x = z[:, None].clone().requires_grad_()
    y = dense.gated_linear(x, w, b, activation) if gated else dense.linear(x, w, b, activation=activation)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    keeps = (z > 0) | (activation == 'none')
    for got, want in ((y.detach()[:, 0], torch.where(keeps, z, torch.zeros_like(z))),
                      (dx[:, 0], keeps.to(dtype))):
        assert got.isfinite().all(), got
        assert ((got - want).abs().float() <= 1e-11 + 4 * oracle.U * want.abs().float()).all(), got


def test_the_oracle_allows_either_slope_where_a_gate_is_within_its_error_of_zero():
    """a = x W of one term is exact but for the order of its rounding with the
    bias: z = 1 - 1 = 0 here, where relu's slope may be taken as 0 or 1."""
    x, w = torch.ones(1, 1), torch.tensor([[1.0], [1.0]])
    layer = oracle.Layer.of(x, w, torch.tensor([-1.0, 0.0]), None, 'relu', True)
    want, bound = layer.backward(torch.ones(1, 1), torch.float32, torch.float32)['x']
    assert float(want) == 0 and float(bound) >= 1
    far = oracle.Layer.of(x, w, torch.tensor([-0.5, 0.0]), None, 'relu', True)
    assert float(far.backward(torch.ones(1, 1), torch.float32, torch.float32)['x'][1]) < 1e-4
