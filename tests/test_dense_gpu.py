"""The dense operators on the GPU against the 64-bit oracle.

Two kinds of checks: bit-exact ones, on small integers whose products and sums
fp32 holds exactly (any wrong index, missing element or element too many shows
as a different integer), and bounded ones on ordinary values, with bounds that
follow from the roundings (oracle/dense.py).
"""

import pytest
import torch

from oracle import dense as oracle
from vectra_amd.kernels import _native
from vectra_amd.kernels import dense
from vectra_amd.kernels import dense_capi as capi

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
ops = torch.ops.vectra


def normal(*shape, seed=0, scale=1.0, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * scale).to(dtype).cuda()


def integers(*shape, most, seed=0, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=gen).to(dtype).cuda()


def view_of(x, pad):
    """The same values as columns of a wider tensor full of NaN."""
    wide = torch.full((x.shape[0] + 2, x.shape[1] + 2 * pad), float('nan'), dtype=x.dtype, device=x.device)
    out = wide[1:-1, pad:pad + x.shape[1]]
    out.copy_(x)
    return out


# rows, width_in, width_out: one of everything, tiles that are full, one short
# and one over, widths of no whole 16-byte chunk, long contractions.
SIZES = [
    (1, 1, 1), (1, 8, 1), (2, 16, 24), (1, 64, 64), (5, 40, 72), (16, 128, 16), (17, 129, 130), (33, 64, 48),
    (63, 65, 31), (64, 64, 64), (65, 128, 384), (127, 72, 129), (128, 128, 128), (129, 136, 257), (255, 200, 256),
    (256, 64, 512), (300, 33, 7), (1, 4096, 520), (4, 2048, 77), (40, 1000, 200), (513, 264, 1000), (2048, 8, 8),
    (5000, 24, 40),
    # Many rows by a weight that fits LDS.
    (16384, 128, 256), (16391, 141, 33), (17000, 72, 100), (16500, 256, 128), (16400, 30, 65),
]


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('size', SIZES, ids=str)
def test_integers_are_exact(size, dtype):
    """x, W in [-2, 2], dy in [-3, 3]: at most 4096 * 4 + ... per sum, below
    2^24, and dz = dy (or dy times an integer of at most 256 in magnitude,
    which 16 bits hold) exactly."""
    rows, width_in, width_out = size
    x, w = integers(rows, width_in, most=2, seed=1, dtype=dtype), integers(width_out, width_in, most=2, seed=2, dtype=dtype)
    b, r = integers(width_out, most=9, seed=3, dtype=dtype), integers(rows, width_out, most=9, seed=4, dtype=dtype)
    dy = integers(rows, width_out, most=3, seed=5, dtype=dtype)
    for activation in ('none', 'relu'):
        leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
        y = dense.linear(*leaves, activation)
        got = torch.autograd.grad(y, leaves, dy)
        xd, wd, bd, rd, dyd = (t.double().cpu() for t in (x, w, b, r, dy))
        z = xd @ wd.t() + bd
        dz = dyd if activation == 'none' else dyd * (z > 0)
        want = (dz @ wd, dz.t() @ xd, dz.sum(0), dyd)
        assert torch.equal(y.cpu(), ((z if activation == 'none' else z.clamp_min(0)) + rd).to(dtype))
        for name, g, v in zip(('x', 'weight', 'bias', 'residual'), got, want):
            assert torch.equal(g.cpu(), v.to(dtype)), (activation, name)


# Products of many large tiles, with rows, columns and contractions that end
# inside one: forward, dx and dW each take them at one of these.
LARGE = [(1100, 4104, 4104), (8200, 264, 4104), (8200, 4104, 264), (2051, 1000, 2056), (4096, 4096, 1024),
         (4090, 2056, 4090), (8190, 1543, 4090),
         (2995, 1032, 4090), (9990, 1000, 5460)]


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('size', LARGE, ids=str)
@pytest.mark.parametrize('gated', [False, True])
def test_large_integers_are_exact(size, dtype, gated):
    """As below 2^24 as the small ones: at most 8200 terms of at most 12.  The
    64-bit reference runs on the GPU, as matrix products of doubles."""
    rows, width_in, width_out = size
    n = width_out * (1 + gated)
    x, w = integers(rows, width_in, most=2, seed=1, dtype=dtype), integers(n, width_in, most=1, seed=2, dtype=dtype)
    b = integers(n, most=9, seed=3, dtype=dtype)
    if gated:  # an up projection of one-hot rows and a gate that passes all: dz stays a small integer
        w.zero_()
        w[torch.arange(n), torch.randint(0, width_in, (n,), generator=torch.Generator().manual_seed(6))] = 1
    dy = integers(rows, width_out, most=3, seed=5, dtype=dtype)
    r = None if gated else integers(rows, width_out, most=9, seed=4, dtype=dtype)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = dense.gated_linear(*leaves, 'relu') if gated else dense.linear(*leaves, r, 'relu')
    got = torch.autograd.grad(y, leaves, dy)
    xd, wd, bd, dyd = (t.double() for t in (x, w, b, dy))
    z = xd @ wd.t() + bd
    if gated:
        gate, up = z.chunk(2, 1)
        want_y = gate.clamp_min(0) * up
        dz = torch.cat([dyd * up * (gate > 0), dyd * gate.clamp_min(0)], 1)
    else:
        want_y = z.clamp_min(0) + r.double()
        dz = dyd * (z > 0)
    assert torch.equal(y, want_y.to(dtype))
    for name, g, v in zip(('x', 'weight', 'bias'), got, (dz @ wd, dz.t() @ xd, dz.sum(0))):
        assert torch.equal(g, v.to(dtype)), name


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('size', SIZES, ids=str)
def test_gated_integers_are_exact(size, dtype):
    """One-hot rows of W keep z, and so dz, small integers: the up projection
    picks elements of x (at most 4), dy is at most 4, dz at most 16 + 4."""
    rows, width_in, width_out = size
    x = integers(rows, width_in, most=4, seed=1, dtype=dtype)
    gen = torch.Generator().manual_seed(6)
    w = torch.zeros(2 * width_out, width_in, dtype=dtype)
    w[torch.arange(2 * width_out), torch.randint(0, width_in, (2 * width_out,), generator=gen)] = 1
    w = w.cuda()
    b = integers(2 * width_out, most=2, seed=3, dtype=dtype)
    dy = integers(rows, width_out, most=4, seed=5, dtype=dtype)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = dense.gated_linear(*leaves, 'relu')
    got = torch.autograd.grad(y, leaves, dy)
    xd, wd, bd, dyd = (t.double().cpu() for t in (x, w, b, dy))
    gate, up = (xd @ wd.t() + bd).chunk(2, 1)
    dz = torch.cat([dyd * up * (gate > 0), dyd * gate.clamp_min(0)], 1)
    assert torch.equal(y.cpu(), (gate.clamp_min(0) * up).to(dtype))
    for g, v in zip(got, (dz @ wd, dz.t() @ xd, dz.sum(0))):
        assert torch.equal(g.cpu(), v.to(dtype))


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('activation', dense.ACTIVATIONS)
@pytest.mark.parametrize('gated', [False, True])
@pytest.mark.parametrize('size', [(1, 300, 40), (70, 141, 90), (257, 128, 256), (900, 520, 333)], ids=str)
def test_layers_and_gradients_stay_in_their_bounds(size, gated, activation, dtype):
    rows, width_in, width_out = size
    n = width_out * (1 + gated)
    x = view_of(normal(rows, width_in, seed=1, dtype=dtype), 5).requires_grad_()
    w = normal(n, width_in, seed=2, scale=width_in ** -0.5, dtype=dtype).requires_grad_()
    b = normal(n, seed=3, scale=0.2, dtype=torch.float32 if activation == 'gelu' else dtype).requires_grad_()
    r = None if gated else normal(rows, width_out, seed=4, dtype=dtype)
    dy = normal(rows, width_out, seed=5, dtype=dtype)
    y = dense.gated_linear(x, w, b, activation) if gated else dense.linear(x, w, b, r, activation)
    grads = torch.autograd.grad(y, (x, w, b), dy)
    layer = oracle.Layer.of(x, w, b, r, activation, gated)
    oracle.assert_within(y, *layer.forward(dtype))
    for g, (want, bound) in zip(grads, layer.backward(dy, dtype, b.dtype).values()):
        oracle.assert_within(g, want, bound)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('width', [1, 31, 32, 33, 100, 256, 1000])
@pytest.mark.parametrize('layout', ['rows', 'view'])
def test_8_bit_rows_equal_the_host_operators(dtype, width, layout):
    """Codes, scales and their values, bit for bit (the host operator is held
    to the oracle)."""
    gen = torch.Generator().manual_seed(width)
    x = torch.randn(257, width, generator=gen) * torch.exp2(torch.randint(-140, 128, (257, 1), generator=gen).float())
    x[3] = 0.0
    x[4, 0], x[5, 0], x[8] = float('inf'), float('nan'), float('-inf')
    x[6], x[7], x[9] = torch.finfo(dtype).max, torch.finfo(dtype).tiny, -torch.finfo(dtype).max
    x = x.to(dtype)
    dev = view_of(x.cuda(), 3) if layout == 'view' else x.cuda()
    codes, scales = dense.quantize_rows(dev)
    want_codes, want_scales = dense.quantize_rows(x)
    assert torch.equal(scales.cpu().view(torch.uint8), want_scales.view(torch.uint8))
    a, b = codes.cpu().view(torch.uint8), want_codes.view(torch.uint8)
    nan = (b & 0x7F) == 0x7F
    assert torch.equal((a & 0x7F) == 0x7F, nan) and torch.equal(a[~nan], b[~nan])
    back = dense.dequantize_rows(codes, scales, dtype).cpu()
    want = dense.dequantize_rows(want_codes, want_scales, dtype)
    assert torch.equal(back.isnan(), want.isnan()) and torch.equal(back[~want.isnan()], want[~want.isnan()])


def test_every_scale_byte_is_read_as_its_power_of_two():
    scales = torch.arange(256, dtype=torch.uint8)[:, None]
    codes = torch.arange(256, dtype=torch.uint8)[None, :32].repeat(256, 1) + 40
    args = codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)
    got = dense.dequantize_rows(args[0].cuda(), args[1].cuda(), torch.float32).cpu()
    want = torch.from_numpy(oracle.dequantize(codes.numpy(), scales.numpy())).float()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[~want.isnan()], want[~want.isnan()])


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('gated', [False, True])
@pytest.mark.parametrize('width_in', [96, 141])
def test_gradients_from_8_bits_are_those_at_the_kept_values(dtype, gated, width_in):
    rows, width_out = 333, 130
    n = width_out * (1 + gated)
    x = normal(rows, width_in, seed=1, dtype=dtype).requires_grad_()
    w = normal(n, width_in, seed=2, scale=width_in ** -0.5, dtype=dtype).requires_grad_()
    b = normal(n, seed=3, dtype=dtype).requires_grad_()
    dy = normal(rows, width_out, seed=5, dtype=dtype)

    def layer(rows_in, checkpoint):
        if gated:
            return dense.gated_linear(rows_in, w, b, 'silu', checkpoint)
        return dense.linear(rows_in, w, b, None, 'gelu', checkpoint)

    y = layer(x, 'e4m3')
    assert torch.equal(y, layer(x, 'none'))
    got = torch.autograd.grad(y, (x, w, b), dy)
    kept = dense.dequantize_rows(*dense.quantize_rows(x.detach()), dtype).requires_grad_()
    want = torch.autograd.grad(layer(kept, 'none'), (kept, w, b), dy)
    for g, v in zip(got, want):  # the same kernels on the same values
        assert torch.equal(g, v)


def test_what_lies_around_the_matrices_is_neither_read_nor_written():
    """x, W, dy and the residual lie in tensors full of NaN, the outputs in
    tensors of a marker: exact results, markers as they were."""
    for dtype in DTYPES:
        for rows, width_in, width_out in ((130, 72, 136), (37, 33, 50), (1, 264, 70)):
            x, w = integers(rows, width_in, most=2, seed=1, dtype=dtype), integers(width_out, width_in, most=2, seed=2, dtype=dtype)
            r, dy = integers(rows, width_out, most=9, seed=4, dtype=dtype), integers(rows, width_out, most=3, seed=5, dtype=dtype)
            xv, wv, rv, dyv = (view_of(t, 8) for t in (x, w, r, dy))

            def marked(*shape):
                whole = torch.full((shape[0] + 2, shape[1] + 16), 77.0, dtype=dtype, device='cuda')
                return whole, whole[1:-1, 8:8 + shape[1]]

            whole, out = marked(rows, width_out)
            capi.forward(xv, wv, None, rv, out=out)
            wholes = [whole]
            whole_dx, dx = marked(rows, width_in)
            whole_dw, dw = marked(width_out, width_in)
            capi.backward(dyv, xv, wv, dx=dx, dweight=dw)
            wholes += [whole_dx, whole_dw]
            xd, wd, rd, dyd = (t.double().cpu() for t in (x, w, r, dy))
            assert torch.equal(out.cpu(), (xd @ wd.t() + rd).to(dtype))
            assert torch.equal(dx.cpu(), (dyd @ wd).to(dtype))
            assert torch.equal(dw.cpu(), (dyd.t() @ xd).to(dtype))
            for whole, inner in zip(wholes, (out, dx, dw)):
                inner.fill_(77.0)
                assert bool((whole == 77.0).all())


def test_a_nan_stays_in_its_row():
    x, w = normal(200, 96, seed=1, dtype=torch.bfloat16), normal(80, 96, seed=2, dtype=torch.bfloat16)
    clean = dense.linear(x, w, activation='gelu')
    x[17, 5], x[150, 95] = float('nan'), float('inf')
    y = dense.linear(x, w, activation='gelu')
    rows = torch.ones(200, dtype=torch.bool)
    rows[[17, 150]] = False
    assert torch.equal(y[rows], clean[rows]) and bool(y[17].isnan().all())


@pytest.mark.parametrize('size', [(300, 96, 100), (16400, 96, 33), (16400, 128, 72)], ids=str)
@pytest.mark.parametrize('gated', [False, True])
def test_an_infinity_of_the_input_stays_out_of_the_inputs_gradient(size, gated):
    """z = +inf where x is and W > 0, and relu's slope there is 1: dx is that of
    a large finite x, at widths that end inside a tile too.  (Gated: the up half
    has zeros for that element, and x of -inf in the gate's place: slope 0.)"""
    rows, width_in, width_out = size
    for dtype in (torch.bfloat16, torch.float32):
        x = integers(rows, width_in, most=2, seed=1, dtype=dtype)
        w = integers(width_out, width_in, most=2, seed=2, dtype=dtype)
        dy = integers(rows, width_out, most=3, seed=3, dtype=dtype)
        w[:, 5] = 1
        if gated:
            up = integers(width_out, width_in, most=2, seed=4, dtype=dtype)
            up[:, 5] = 0
            w = torch.cat((w, up))
        x[7, 5] = x[rows - 1, 5] = 30000  # z > 0 whatever the rest is, and exact in fp32
        if gated:
            x[7, 5] = x[rows - 1, 5] = -30000
        wanted = [True, False, False]
        want, = ops.linear_backward(dy, x, None, w, None, 'relu', gated, wanted)
        x[7, 5] = x[rows - 1, 5] = float('-inf' if gated else 'inf')
        got, = ops.linear_backward(dy, x, None, w, None, 'relu', gated, wanted)
        live = torch.ones(rows, dtype=torch.bool)
        if gated:  # up = ... + inf * 0 is NaN in those rows, by the formula
            live[[7, rows - 1]] = False
        assert torch.equal(got[live], want[live])


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_a_single_row_may_have_any_stride(dtype):
    """Of x, dy and W: its stride is not a distance to another row."""
    for width_in, width_out in ((64, 48), (33, 8), (4104, 264)):
        x, dy = integers(1, width_in, most=2, seed=1, dtype=dtype), integers(1, width_out, most=3, seed=2, dtype=dtype)
        w = integers(width_out, width_in, most=2, seed=3, dtype=dtype)
        x0, dy0 = x.as_strided(x.shape, (0, 1)), dy.as_strided(dy.shape, (0, 1))
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        db = torch.empty(width_out, dtype=dtype, device='cuda')
        capi.backward(dy0, x0, w, dx=dx, dweight=dw, dbias=db)
        assert torch.equal(dx, (dy.double() @ w.double()).to(dtype))
        assert torch.equal(dw, (dy.double().t() @ x.double()).to(dtype)) and torch.equal(db, dy[0])
        rows = integers(70, width_in, most=2, seed=4, dtype=dtype)
        dz, w0 = integers(70, 1, most=3, seed=5, dtype=dtype), x.as_strided(x.shape, (0, 1))
        dx = torch.empty_like(rows)
        capi.backward(dz, rows, w0, dx=dx)
        assert torch.equal(dx, (dz.double() @ x.double()).to(dtype))


def test_rows_far_apart_are_copied():
    for dtype, stride in ((torch.bfloat16, (1 << 22) + 8), (torch.float32, (1 << 21) + 4)):
        store = torch.zeros(stride * 40 + 64, dtype=dtype, device='cuda')
        x = store.as_strided((40, 64), (stride, 1))
        x.copy_(integers(40, 64, most=2, seed=1, dtype=dtype))
        w, dy = integers(48, 64, most=2, seed=2, dtype=dtype), integers(40, 48, most=3, seed=3, dtype=dtype)
        assert torch.equal(dense.linear(x, w), (x.double() @ w.double().t()).to(dtype))
        dw, = ops.linear_backward(dy, x, None, w, None, 'none', False, [False, True, False])
        assert torch.equal(dw, (dy.double().t() @ x.double()).to(dtype))


# rows, width_in, width_out: an operand or a result of more than 2^32 bytes on
# the products' tiles, on the kernel of resident weights, and on both sides.
@pytest.mark.parametrize('size', [(1100007, 2048, 64), (1100007, 64, 2048), (17000003, 136, 128)], ids=str)
def test_offsets_past_32_bits(size):
    """Rows of zeros but for a few, the last ones among them: exact integers."""
    rows, width_in, width_out = size
    dtype = torch.bfloat16
    at = torch.tensor([0, 1, rows // 2, rows - 130, rows - 2, rows - 1], device='cuda')
    x = torch.zeros(rows, width_in, dtype=dtype, device='cuda')
    dy = torch.zeros(rows, width_out, dtype=dtype, device='cuda')
    x[at], dy[at] = (integers(len(at), n, most=2, seed=n, dtype=dtype) for n in (width_in, width_out))
    w = integers(width_out, width_in, most=2, seed=3, dtype=dtype)
    xd, wd, dyd = x[at].double(), w.double(), dy[at].double()
    y = dense.linear(x, w, activation='relu')
    assert torch.equal(y[at], (xd @ wd.t()).clamp_min(0).to(dtype))
    assert int(torch.count_nonzero(y)) == int(torch.count_nonzero(y[at]))
    del y
    dz = dyd * (xd @ wd.t() > 0)
    dx, dw, db = ops.linear_backward(dy, x, None, w, None, 'relu', False, [True, True, True])
    assert torch.equal(dw, (dz.t() @ xd).to(dtype)) and torch.equal(db, dz.sum(0).to(dtype))
    assert torch.equal(dx[at], (dz @ wd).to(dtype))
    assert int(torch.count_nonzero(dx)) == int(torch.count_nonzero(dx[at]))


def test_8_bit_rows_past_32_bits():
    rows, width = 2200003, 2048  # 4.5e9 codes
    at = torch.tensor([0, rows // 2, rows - 1], device='cuda')
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device='cuda')
    x[at] = normal(3, width, seed=1, dtype=torch.bfloat16)
    codes, scales = dense.quantize_rows(x)
    want = dense.quantize_rows(x[at])
    for got, few in zip((codes, scales), want):
        assert torch.equal(got[at].view(torch.uint8), few.view(torch.uint8))
    assert int(torch.count_nonzero(codes.view(torch.uint8))) == int(torch.count_nonzero(want[0].view(torch.uint8)))
    back = dense.dequantize_rows(codes, scales, torch.bfloat16)
    assert torch.equal(back[at], dense.dequantize_rows(*want, torch.bfloat16))
    assert int(torch.count_nonzero(back)) == int(torch.count_nonzero(back[at]))


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('size', [(0, 40, 24), (5, 0, 24), (5, 40, 0), (0, 0, 0), (0, 512, 4104), (300, 0, 600)], ids=str)
@pytest.mark.parametrize('gated', [False, True])
def test_empty_sizes(size, gated, dtype):
    """No rows: gradients of the weight and the bias are zero.  No inputs: z = b."""
    rows, width_in, width_out = size
    n = width_out * (1 + gated)
    x, w = integers(rows, width_in, most=2, seed=1, dtype=dtype), integers(n, width_in, most=2, seed=2, dtype=dtype)
    b, dy = integers(n, most=3, seed=3, dtype=dtype), integers(rows, width_out, most=3, seed=4, dtype=dtype)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = dense.gated_linear(*leaves, 'relu') if gated else dense.linear(*leaves, None, 'relu')
    got = torch.autograd.grad(y, leaves, dy)
    z = b.double().expand(rows, n)
    if gated:
        gate, up = z.chunk(2, 1)
        want_y, dz = gate.clamp_min(0) * up, torch.cat([dy * up * (gate > 0), dy * gate.clamp_min(0)], 1)
    else:
        want_y, dz = z.clamp_min(0), dy.double() * (z > 0)
    assert torch.equal(y, want_y.to(dtype))
    assert got[0].shape == x.shape and got[1].shape == w.shape
    assert not got[0].any() and not got[1].any() and torch.equal(got[2], dz.sum(0).to(dtype))


@pytest.mark.parametrize('checkpoint', dense.CHECKPOINTS)
def test_a_broadcast_gradient_is_read_as_its_rows(checkpoint):
    """y.sum() gives a gradient of stride zero, as an expanded x has."""
    x = integers(1, 72, most=2, seed=1, dtype=torch.bfloat16).expand(130, 72).requires_grad_()
    w = integers(40, 72, most=2, seed=2, dtype=torch.bfloat16).requires_grad_()
    dx, dw = torch.autograd.grad(dense.linear(x, w, checkpoint=checkpoint).sum(), (x, w))
    assert torch.equal(dx, w.double().sum(0).to(dx.dtype).expand(130, 72))
    assert torch.equal(dw, (130 * x[0].double()).to(dw.dtype).expand(40, 72))


# On a few rows, a small, a medium and a large tile, in parts, and by resident weights.
@pytest.mark.parametrize('size', [(1, 300, 40), (65, 64, 128), (300, 4096, 520), (1100, 1024, 2100), (4096, 512, 4104),
                                  (16400, 128, 100)], ids=str)
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_the_residual_may_be_the_output(size, dtype):
    rows, width_in, width_out = size
    x, w = integers(rows, width_in, most=2, seed=1, dtype=dtype), integers(width_out, width_in, most=2, seed=2, dtype=dtype)
    out = integers(rows, width_out, most=5, seed=3, dtype=dtype)
    want = (x.float() @ w.float().t() + out.float()).to(dtype)
    capi.forward(x, w, None, out, out=out)
    assert torch.equal(out, want)


def test_results_do_not_depend_on_the_run():
    for dtype in (torch.bfloat16, torch.float32):
        x = normal(3000, 200, seed=1, dtype=dtype).requires_grad_()
        w = normal(264, 200, seed=2, scale=0.1, dtype=dtype).requires_grad_()
        b = normal(264, seed=3, dtype=dtype).requires_grad_()
        dy = normal(3000, 264, seed=4, dtype=dtype)
        first = None
        for _ in range(3):
            y = dense.linear(x, w, b, activation='gelu')
            now = (y.detach(), *torch.autograd.grad(y, (x, w, b), dy))
            if first is None:
                first = now
            assert all(torch.equal(a, c) for a, c in zip(first, now))


def test_calls_on_two_streams_do_not_share_scratch():
    sets = [(normal(2000, 141, seed=s), normal(200, 141, seed=s + 10, scale=0.1)) for s in (1, 2)]
    dys = [normal(2000, 200, seed=s + 20) for s in (1, 2)]

    def both(x, w, dy):
        return [dense.linear(x, w, activation='silu'),
                *ops.linear_backward(dy, x, None, w, None, 'silu', False, [True, True, False])]

    want = [both(x, w, dy) for (x, w), dy in zip(sets, dys)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for stream, (x, w), dy in zip(streams, sets, dys):
            with torch.cuda.stream(stream):
                got.append(both(x, w, dy))
        torch.cuda.synchronize()
        for g, v in zip(got, want):
            assert all(torch.equal(a, c) for a, c in zip(g, v))


def test_a_captured_step_replays():
    """Forward and gradients in one graph, replayed on new inputs with eager
    work between the replays."""
    x, w, b = normal(1000, 72, seed=1), normal(160, 72, seed=2, scale=0.1), normal(160, seed=3)
    dy = normal(1000, 80, seed=4)

    def step():
        y = dense.gated_linear(x, w, b, 'silu')
        codes, scales = dense.quantize_rows(x)
        return [y, *ops.linear_backward(dy, x, None, w, b, 'silu', True, [True, True, True]),
                *ops.linear_backward(dy, codes, scales, w, b, 'silu', True, [True, True, True])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for seed in range(4):
        x.copy_(normal(1000, 72, seed=30 + seed))
        dy.copy_(normal(1000, 80, seed=40 + seed))
        want = step()
        torch.cuda.synchronize()
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_a_captured_autograd_step_replays():
    x, w = normal(300, 64, seed=1).requires_grad_(), normal(96, 64, seed=2, scale=0.1).requires_grad_()
    dy = normal(300, 96, seed=3)

    def step():
        return torch.autograd.grad(dense.linear(x, w, activation='gelu', checkpoint='e4m3'), (x, w), dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        with torch.no_grad():
            x.mul_(1.5)
        want = [g.clone() for g in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_compiled_training_step_equals_the_eager_one():
    x = normal(128, 64, seed=1, dtype=torch.bfloat16).requires_grad_()
    w = normal(96, 64, seed=2, scale=0.1, dtype=torch.bfloat16).requires_grad_()
    v = normal(64, 96, seed=3, scale=0.1, dtype=torch.bfloat16).requires_grad_()

    def block(x, w, v):
        return dense.linear(dense.linear(x, w, activation='gelu', checkpoint='e4m3'), v, None, x)

    dy = normal(128, 64, seed=4, dtype=torch.bfloat16)
    want = torch.autograd.grad(block(x, w, v), (x, w, v), dy)
    got = torch.autograd.grad(torch.compile(block, backend='aot_eager')(x, w, v), (x, w, v), dy)
    assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_refusals_on_the_gpu():
    x, w = torch.zeros(2, 8, device='cuda'), torch.zeros(4, 8, device='cuda')
    for call in (lambda: dense.linear(x, w.cpu()), lambda: dense.linear(x, w, torch.zeros(4)),
                 lambda: dense.linear(x, w, None, torch.zeros(2, 4)), lambda: dense.linear(x, w.half()),
                 lambda: dense.gated_linear(x, torch.zeros(5, 8, device='cuda'))):
        with pytest.raises(RuntimeError):
            call()
    need = torch.zeros(64, 72, device='cuda')
    with pytest.raises(capi.DenseError) as e:
        capi.backward(need, need, torch.zeros(72, 72, device='cuda'), dx=need.clone(), activation='relu',
                      workspace=torch.zeros(256, dtype=torch.uint8, device='cuda'))
    assert e.value.status == capi.ERR_WORKSPACE


def test_the_native_library_ran():
    dense.linear(torch.zeros(2, 8, device='cuda'), torch.zeros(4, 8, device='cuda'))
    assert _native.DENSE_LIBRARY in _native.loaded_libraries()
