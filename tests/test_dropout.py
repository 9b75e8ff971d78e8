"""torch.ops.vectra.dropout on the CPU and the GPU: which elements are kept, the
backward pass, shapes and strides, and what it refuses."""

import pytest
import torch

from oracle import block as oracle
from vectra_amd.kernels import block

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def rng_of(seed, offset=0, device='cpu'):
    return torch.tensor([seed, offset], device=device)


def test_philox_known_answers():
    """The generator against its published known answers (counter and key all zeros, all ones)."""
    assert oracle.philox((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = 0xFFFFFFFF
    assert oracle.philox((ones,) * 4, (ones,) * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_factors_are_the_generator_s():
    seed, offset, stream = 0x123456789ABCDEF, 77, 5
    got = oracle.factors(3, 11, 0.5, (seed, offset), stream)
    for row in range(3):
        for column in range(11):
            group = row * 2 + column // 8
            word = oracle.philox((group, 0, stream, offset), (seed & 0xFFFFFFFF, seed >> 32))[column % 8 // 2]
            bits = word >> 16 if column % 2 else word & 0xFFFF
            assert got[row, column] == (2.0 if bits >= 32768 else 0.0)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('shape', [(1, 1), (1, 7), (3, 8), (5, 9), (2, 3, 130), (257, 141), (4, 1024), (1, 4099)], ids=str)
def test_kept_elements_and_their_gradient(shape, dtype, device):
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(*shape, generator=gen).to(dtype).to(device).requires_grad_()
    dy = torch.randn(*shape, generator=gen).to(dtype).to(device)
    for p, seed, offset, stream in ((0.1, 5, 0, 0), (0.5, -3, 2 ** 33 + 9, 2 ** 32 - 1), (0.999, 2 ** 62, 1, 7)):
        rng = rng_of(seed, offset, device)
        y = block.dropout(x, p, rng, stream)
        k = oracle.factors(x.numel() // shape[-1], shape[-1], p, (seed, offset), stream).reshape(shape)
        u = 2 * oracle.U  # the factor's rounding and the product's
        for got, of in ((y, x), (torch.autograd.grad(y, x, dy)[0], dy)):
            want = of.detach().double().cpu() * k
            oracle.assert_within(got, want, want.abs() * u + oracle.rounding(want, want.abs() * u, dtype))
            assert torch.equal(got.cpu() == 0, (k == 0) | (of.cpu() == 0))


@pytest.mark.parametrize('device', DEVICES)
def test_probability_and_offsets(device):
    x = torch.ones(512, 512, device=device)
    for p in (0.0, 2 ** -16, 0.25, 0.9, 1 - 2 ** -16):
        y = block.dropout(x, p, rng_of(11, 3, device))
        kept = float((y != 0).double().mean())
        n = x.numel()
        assert abs(kept - (1 - p)) <= 6 * (p * (1 - p) / n) ** 0.5 + 1 / n, (p, kept)
        assert torch.equal(y[y != 0], torch.full_like(y[y != 0], 65536 / (65536 - round(65536 * p))))
    masks = [block.dropout(x, 0.5, rng_of(s, o, device), t) != 0 for s, o, t in
             ((1, 0, 0), (2, 0, 0), (1, 1, 0), (1, 0, 1), (1 + 2 ** 40, 0, 0))]
    for i, a in enumerate(masks):
        for b in masks[:i]:  # independent draws agree on half of the elements
            assert abs(float((a == b).double().mean()) - 0.5) < 6 * 0.5 / 512
    # Offsets that differ by 2^32 are one.
    assert torch.equal(masks[0], block.dropout(x, 0.5, rng_of(1, 2 ** 32, device)) != 0)


@pytest.mark.parametrize('device', DEVICES)
def test_strides_scalars_and_empty(device):
    rng = rng_of(9, 1, device)
    wide = torch.randn(6, 40, 50, device=device)
    for view in (wide[:, 3:30, 7:41], wide.transpose(1, 2), wide[::2, :, ::3], wide[:, :1].expand(6, 7, 50), wide[..., 0]):
        assert torch.equal(block.dropout(view, 0.4, rng, 2), block.dropout(view.contiguous(), 0.4, rng, 2))
    assert block.dropout(torch.tensor(2.0, device=device), 0.3, rng).shape == ()
    for shape in ((0,), (0, 5), (4, 0), (2, 0, 3)):
        x = torch.zeros(shape, device=device).requires_grad_()
        y = block.dropout(x, 0.3, rng)
        assert y.shape == x.shape
        torch.autograd.grad(y.sum(), x)
    pair = torch.tensor([9, -1, 1, -1], device=device)[::2]  # rng of any stride
    assert torch.equal(block.dropout(wide, 0.4, pair, 2), block.dropout(wide, 0.4, rng, 2))


@pytest.mark.parametrize('device', DEVICES)
def test_a_dropped_element_is_zero_whatever_it_held(device):
    x = torch.full((64, 64), float('inf'), device=device)
    x[::2] = float('nan')
    y = block.dropout(x, 0.5, rng_of(3, 0, device))
    k = oracle.factors(64, 64, 0.5, (3, 0), 0)
    assert torch.equal(y.cpu() == 0, k == 0)
    assert bool(torch.isnan(y[::2].cpu()[k[::2] != 0]).all()) and bool(torch.isinf(y[1::2].cpu()[k[1::2] != 0]).all())


def test_gradients_of_gradients():
    x, dy, v = (torch.randn(4, 9, dtype=torch.float32).requires_grad_() for _ in range(3))
    rng = rng_of(1)
    g, = torch.autograd.grad(block.dropout(x, 0.3, rng), x, dy, create_graph=True)
    gg, = torch.autograd.grad(g, dy, v)
    assert torch.equal(gg, block.dropout(v.detach(), 0.3, rng))


def test_rng_changed_between_the_passes_is_an_error():
    x, rng = torch.randn(4, 9).requires_grad_(), rng_of(1)
    y = block.dropout(x, 0.3, rng)
    rng[1].add_(1)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()


@pytest.mark.parametrize('device', DEVICES)
def test_refusals(device):
    x, rng = torch.randn(4, 9, device=device), rng_of(1, 0, device)
    for p in (-0.1, 1.0, 1 - 2 ** -18, float('nan')):
        with pytest.raises(ValueError, match='p must be'):
            block.dropout(x, p, rng)
    for stream in (-1, 2 ** 32):
        with pytest.raises(ValueError, match='stream must be'):
            block.dropout(x, 0.1, rng, stream)
    for bad in (rng.float(), rng[:1], rng[None], torch.zeros(3, dtype=torch.long, device=device)):
        with pytest.raises(RuntimeError, match='rng must be'):
            block.dropout(x, 0.1, bad)
    with pytest.raises(RuntimeError, match='x must be float'):
        block.dropout(x.double(), 0.1, rng)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError, match='forward-mode'):
        block.dropout(torch.autograd.forward_ad.make_dual(x, x), 0.1, rng)


def test_opcheck():
    x = torch.randn(3, 10).requires_grad_()
    torch.library.opcheck(torch.ops.vectra.dropout.default, (x, 0.4, rng_of(4), 2),
                          test_utils=('test_schema', 'test_faketensor', 'test_autograd_registration'))


@pytest.mark.gpu
def test_rng_of_another_device_is_refused():
    with pytest.raises(RuntimeError, match='rng must be on'):
        block.dropout(torch.randn(4, 9, device='cuda'), 0.1, rng_of(1))


@pytest.mark.gpu
def test_a_captured_graph_draws_anew_with_a_changed_rng():
    x = torch.randn(300, 100, device='cuda', dtype=torch.bfloat16)
    rng = rng_of(5, 0, 'cuda')
    dy = torch.randn_like(x)
    block.dropout(x, 0.2, rng, 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block.dropout(x, 0.2, rng, 4)
        dx = block.dropout(dy, 0.2, rng, 4)
        rng[1].add_(1)
    for step in range(4):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        again = rng_of(5, step, 'cuda')
        assert torch.equal(y, block.dropout(x, 0.2, again, 4)) and torch.equal(dx, block.dropout(dy, 0.2, again, 4))
        assert torch.equal(rng.cpu(), rng_of(5, step + 1))


@pytest.mark.gpu
def test_positions_past_32_bits_of_bytes():
    """2^32 bytes in: the elements there draw by their own positions, and are read from them."""
    rows, width = 2 ** 17 + 3, 2 ** 14 + 8
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device='cuda')
    x[-3:] = torch.randn(3, width, device='cuda').to(x.dtype)
    rng = rng_of(8, 2, 'cuda')
    y = block.dropout(x, 0.3, rng, 1)
    groups = width // 8
    k = torch.empty(3, width, dtype=torch.float64)
    for r in range(3):
        for g in (0, 1, groups // 2, groups - 1):
            group = (rows - 3 + r) * groups + g
            words = oracle.philox((group & 0xFFFFFFFF, group >> 32, 1, 2), (8, 0))
            for e in range(8):
                bits = words[e // 2] >> 16 if e % 2 else words[e // 2] & 0xFFFF
                want = 0.0 if bits < round(0.3 * 65536) else 65536 / (65536 - round(0.3 * 65536))
                k[r, g * 8 + e] = want
                v = float(x[rows - 3 + r, g * 8 + e].double()) * want
                assert abs(float(y[rows - 3 + r, g * 8 + e].double()) - v) <= abs(v) * 2.0 ** -8
    assert not bool(y[:-3].any())
