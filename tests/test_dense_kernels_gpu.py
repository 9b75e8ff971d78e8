"""The dense operators' kernels for many rows and for large tiles: ordinary
values against the 64-bit oracle with every activation, results that do not
depend on the run, and rows whose tile spans more than 2^31 bytes.

The 64-bit side runs on the GPU (matrix products of doubles).
"""

import numpy as np
import pytest
import torch

from oracle import dense as oracle
from tests import test_dense_activations
from vectra_amd.kernels import dense

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
ops = torch.ops.vectra


def normal(*shape, seed=0, scale=1.0, dtype=torch.float32):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device='cuda') * scale).to(dtype)


def within(got, want, bound, name):
    off = (got.detach().double() - want).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), (
        f'{name}: {int(bad.sum())} of {bad.numel()} outside; worst {float((off / bound).max()):.3g} times the bound, '
        f'first at {torch.nonzero(bad)[0].tolist()}')


def arguments(rows, width_in, width_out, dtype, gated, bias_dtype=None):
    n = width_out * (1 + gated)
    return dict(x=normal(rows, width_in, seed=1, dtype=dtype).requires_grad_(),
                w=normal(n, width_in, seed=2, scale=width_in ** -0.5, dtype=dtype).requires_grad_(),
                b=normal(n, seed=3, scale=0.2, dtype=bias_dtype or dtype).requires_grad_(),
                r=None if gated else normal(rows, width_out, seed=4, dtype=dtype),
                dy=normal(rows, width_out, seed=5, dtype=dtype))


def call(t, activation, gated, checkpoint='none'):
    if gated:
        return dense.gated_linear(t['x'], t['w'], t['b'], activation, checkpoint)
    return dense.linear(t['x'], t['w'], t['b'], t['r'], activation, checkpoint)


def check(t, activation, gated):
    y = call(t, activation, gated)
    grads = torch.autograd.grad(y, (t['x'], t['w'], t['b']), t['dy'])
    wide = [None if t[k] is None else t[k].detach().double() for k in ('x', 'w', 'b', 'r')]
    layer = oracle.Layer(*wide, activation, gated)
    dtype = t['x'].dtype
    within(y, *layer.forward(dtype), 'y')
    # (The oracle's own backward() brings the gradient to the CPU.)
    on_host = oracle.Layer(*[None if v is None else v.cpu() for v in wide], activation, gated)
    for g, (name, (want, bound)) in zip(grads, on_host.backward(t['dy'], dtype, t['b'].dtype).items()):
        within(g, want.cuda(), bound.cuda(), name)


SMOOTH = ['gelu', 'gelu_tanh', 'silu']


# Many rows by a weight that stays in LDS: contractions of every length that
# such a kernel exists for, widths inside and at the end of a tile, a last unit
# of 16 rows that is short, rows that leave waves unequal.
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('activation', SMOOTH)
@pytest.mark.parametrize('gated', [False, True])
@pytest.mark.parametrize('size', [(16391, 60, 70), (16640, 128, 256), (16400, 141, 100), (17003, 250, 128)], ids=str)
def test_many_rows_stay_in_their_bounds(size, gated, activation, dtype):
    t = arguments(*size, dtype, gated, torch.float32 if activation == 'gelu' else dtype)
    check(t, activation, gated)


# Tiles of 256 and 192 rows in the forward product, dx and dW, whole and not.
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('gated,activation', [(False, a) for a in SMOOTH] + [(True, a) for a in SMOOTH])
@pytest.mark.parametrize('size', [(2048, 1024, 4096), (2051, 1000, 4090)], ids=str)
def test_large_tiles_stay_in_their_bounds(size, gated, activation, dtype):
    t = arguments(*size, dtype, gated, torch.float32 if activation == 'gelu' else dtype)
    check(t, activation, gated)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('gated', [False, True])
@pytest.mark.parametrize('checkpoint', dense.CHECKPOINTS)
@pytest.mark.parametrize('size', [(16640, 128, 256), (3001, 1000, 2730), (300, 2048, 520), (40, 512, 96)], ids=str)
def test_a_step_gives_the_same_bits_every_time(size, checkpoint, gated, dtype):
    t = arguments(*size, dtype, gated)
    first = None
    for _ in range(4):
        y = call(t, 'silu', gated, checkpoint)
        now = (y.detach(), *torch.autograd.grad(y, (t['x'], t['w'], t['b']), t['dy']))
        first = first or now
        assert all(torch.equal(a, c) for a, c in zip(first, now))


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


@pytest.mark.parametrize('dtype', DTYPES[:2], ids=str)
def test_a_fp32_bias_gradient_has_fp32_slopes(dtype):
    """x = 0, so z is the fp32 bias itself, and the only row of dy that is not
    zero is ones: db is gelu'(z), of which nothing is rounded to 16 bits.  Its
    error holds none of the error of the polynomial that serves 16-bit results
    (e6, up to 8e-7 of the tail): projected on e6 it is near 0, where it would
    be 1; roundings, of 1 / 7 of e6's size and uncorrelated with it, leave less
    than a half."""
    rows, width_in, n = 40, 64, 4096
    b = torch.linspace(-4, 4, n, device='cuda')
    dy = torch.zeros(rows, n, dtype=dtype, device='cuda')
    dy[7] = 1
    x = torch.zeros(rows, width_in, dtype=dtype, device='cuda')
    db, = ops.linear_backward(dy, x, None, normal(n, width_in, dtype=dtype), b, 'gelu', False, [False, False, True])
    assert db.dtype == torch.float32
    z = b.double().cpu()
    error = db.double().cpu() - oracle.activation(z, 'gelu')[1]
    assert float(error.abs().max()) < 32 * oracle.U
    # e6: the tail by degree 6 less the tail, with the sign that the slope takes it with.
    c, powers = test_dense_activations.constants(1)
    t = 1 / (1 + c * z.abs().numpy())
    tail = 0.5 * torch.special.erfc(z.abs() / 2 ** 0.5)
    e6 = torch.exp(-z * z / 2) * torch.from_numpy(np.polyval(powers, t) * t) - tail
    e6 = torch.where(z < 0, e6, -e6)
    assert abs(float((error * e6).sum() / (e6 * e6).sum())) < 0.5


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('size', [(2051, 1000, 2056), (4096, 4096, 1024)], ids=str)
def test_large_operands_that_start_anywhere(size, dtype):
    """Rows of whole chunks whose first element is not 16-byte aligned, of x, W
    and dy: copied first, exact integers, NaN around them."""
    rows, width_in, width_out = size
    gen = torch.Generator(device='cuda').manual_seed(1)

    def shifted(r, c, most):
        wide = torch.full((r, c + 16), float('nan'), dtype=dtype, device='cuda')
        wide[:, 1:c + 1] = torch.randint(-most, most + 1, (r, c), generator=gen, device='cuda').to(dtype)
        return wide[:, 1:c + 1]

    x, w, dy = shifted(rows, width_in, 2), shifted(width_out, width_in, 1), shifted(rows, width_out, 3)
    assert torch.equal(dense.linear(x, w), (x.double() @ w.double().t()).to(dtype))
    dx, dw = ops.linear_backward(dy, x, None, w, None, 'none', False, [True, True, False])
    assert torch.equal(dx, (dy.double() @ w.double()).to(dtype))
    assert torch.equal(dw, (dy.double().t().contiguous() @ x.double()).to(dtype))
