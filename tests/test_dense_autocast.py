"""The dense operators and the price model on them under torch.autocast: what
torch's own linear layers do there, in autocast's type."""

import copy

import pytest
import torch

from vectra_amd.kernels import dense
from vectra_amd.price_transformer import model as model_lib

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
TYPES = [torch.bfloat16, torch.float16]


def randn(*shape, seed=0, device='cpu', scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(device)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('gated', [False, True])
def test_a_layer_is_that_of_its_cast_arguments(gated, dtype, device):
    """Bit for bit, with gradients in the arguments' own types; a fp32 bias is not rounded."""
    x, w, b = randn(5, 24, seed=1, device=device), randn(6, 24, seed=2, device=device), randn(6, seed=3, device=device)

    def layer(*t):
        return dense.gated_linear(*t, 'silu') if gated else dense.linear(*t, activation='gelu')

    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    with torch.autocast(device, dtype):
        y = layer(*leaves)
    dy = randn(*y.shape, seed=4, device=device).to(dtype)
    got = torch.autograd.grad(y, leaves, dy)
    cast = [x.to(dtype).requires_grad_(), w.to(dtype).requires_grad_(), b.clone().requires_grad_()]
    want_y = layer(*cast)
    want = torch.autograd.grad(want_y, cast, dy)
    assert y.dtype == dtype and torch.equal(y, want_y)
    for g, v in zip(got, want):
        assert g.dtype == torch.float32 and torch.equal(g, v.float())


@pytest.mark.parametrize('device', DEVICES)
def test_a_wider_residual_stays_in_its_type(device):
    """As `residual + layer(x)` is under autocast; one of autocast's type joins the epilogue."""
    x, w = randn(2, 5, 24, seed=1, device=device), randn(6, 24, seed=2, device=device)
    r = randn(2, 5, 6, seed=3, device=device).requires_grad_()
    with torch.autocast(device, torch.bfloat16):
        alone = dense.linear(x, w)
        y = dense.linear(x, w, None, r)
        narrow = dense.linear(x, w, None, r.detach().bfloat16())
        with pytest.raises(RuntimeError, match='residual'):
            dense.linear(x, w, None, r[:1])
    assert y.dtype == torch.float32 and torch.equal(y, r + alone)
    assert torch.equal(torch.autograd.grad(y.sum(), r)[0], torch.ones_like(r))
    assert narrow.dtype == torch.bfloat16
    assert torch.equal(narrow, dense.linear(x.bfloat16(), w.bfloat16(), None, r.detach().bfloat16()))


@pytest.mark.parametrize('device', DEVICES)
def test_outside_and_in_a_disabled_region_nothing_is_cast(device):
    x, w = randn(5, 24, seed=1, device=device), randn(6, 24, seed=2, device=device)
    want = dense.linear(x, w)
    with torch.autocast(device, torch.bfloat16), torch.autocast(device, enabled=False):
        assert torch.equal(dense.linear(x, w), want)
    assert want.dtype == torch.float32


def relative(a, b):
    return float((a - b).norm() / b.norm().clamp_min(1e-12))


def step(model, inputs, device, dtype):
    model.zero_grad(set_to_none=True)
    with torch.autocast(device, dtype):
        out = model(*inputs)
    (out * torch.linspace(0.5, 1.5, out.numel(), device=out.device)).sum().backward()
    return out.detach(), {name: p.grad for name, p in model.named_parameters()}


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('gate', [False, True])
@pytest.mark.parametrize('checkpoint', dense.CHECKPOINTS)
def test_the_price_model_runs_and_trains_under_autocast(checkpoint, gate, device):
    """Both models round every layer's output to bf16, the plain one z before
    its activation too: a few steps of 2^-8 per layer.  A gradient kept from
    8 bits is off by what half a code's step of its inputs does to it (0.25, as
    without autocast) on top."""
    torch.manual_seed(0)
    config = model_lib.ModelConfig(d_model=48, num_heads=4, num_layers=2, ffn_dim=80, num_candidates=12,
                                   embedding_dim=24, attribute_dim=7, ffn_gate=gate)
    plain = model_lib.PriceTransformer(config).to(device)
    model = copy.deepcopy(plain).set_dense_kernels(checkpoint=checkpoint)
    inputs = model_lib.example_inputs(config, 9, device, seed=1)
    y0, g0 = step(plain, inputs, device, torch.bfloat16)
    y1, g1 = step(model, inputs, device, torch.bfloat16)
    assert y1.dtype == y0.dtype and relative(y1, y0) < 2 ** -8
    for name in g0:
        assert g1[name].dtype == g0[name].dtype and g1[name].isfinite().all()
        assert relative(g1[name], g0[name]) < (0.1 if checkpoint == 'none' else 0.35), name


@pytest.mark.parametrize('device', DEVICES)
def test_a_compiled_layer_under_autocast_equals_the_eager_one(device):
    x, w = randn(5, 24, seed=1, device=device), randn(6, 24, seed=2, device=device).requires_grad_()
    r = randn(5, 6, seed=3, device=device)

    def f(x, w, r):
        with torch.autocast(device, torch.bfloat16):
            return dense.linear(x, w, None, r, 'gelu')

    want = f(x, w, r)
    got = torch.compile(f, backend='aot_eager', fullgraph=True)(x, w, r)
    assert got.dtype == want.dtype and torch.equal(got, want)
    assert torch.equal(torch.autograd.grad(got.sum(), w)[0], torch.autograd.grad(want.sum(), w)[0])
