"""The dense operators where they have no derivative (forward mode, through the
8-bit rows, a second time): an error, never a derivative that is dropped."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from vectra_amd.kernels import dense
from vectra_amd.price_transformer import model as model_lib

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


def randn(*shape, seed=0, device='cpu'):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(device)


def layer_arguments(gated, device):
    t = {'x': randn(3, 8, seed=1, device=device), 'weight': randn(4, 8, seed=2, device=device),
         'bias': randn(4, seed=3, device=device)}
    if not gated:
        t['residual'] = randn(3, 4, seed=4, device=device)
    return t


def call(gated, t):
    return dense.gated_linear(**t) if gated else dense.linear(**t, activation='gelu')


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('other', [False, True], ids=['alone', 'beside a leaf'])
@pytest.mark.parametrize('gated,name', [(g, n) for g in (False, True) for n in layer_arguments(g, 'cpu')])
def test_a_tangent_is_refused_and_not_dropped(gated, name, other, device):
    t = layer_arguments(gated, device)
    if other:  # an argument that needs a reverse gradient changes nothing
        t['weight' if name != 'weight' else 'x'].requires_grad_()
    with forward_ad.dual_level():
        t[name] = forward_ad.make_dual(t[name], torch.ones_like(t[name]))
        for grad_mode in (True, False):
            with torch.set_grad_enabled(grad_mode), pytest.raises(NotImplementedError, match='forward-mode'):
                call(gated, t)
    # Outside the level the tangent is gone, and the call is an ordinary one.
    call(gated, t)


@pytest.mark.parametrize('gated', [False, True])
def test_jvp_and_jacfwd_are_refused(gated):
    t = layer_arguments(gated, 'cpu')
    x = t.pop('x')

    def f(a):
        return call(gated, {'x': a, **t})

    for transform in (lambda: torch.func.jvp(f, (x,), (x,)), lambda: torch.func.jacfwd(f)(x),
                      lambda: torch.func.jvp(lambda a: torch.func.jvp(lambda b: f(a) + b, (x[:, :1],), (x[:, :1],))[0],
                                             (x,), (x,))):
        with pytest.raises((NotImplementedError, RuntimeError)):
            transform()


def test_jvp_of_the_price_model_is_that_of_its_plain_layers_or_refused():
    config = model_lib.ModelConfig(d_model=16, num_heads=2, num_layers=1, ffn_dim=24, num_candidates=6, embedding_dim=8,
                                   attribute_dim=3)
    torch.manual_seed(0)
    model = model_lib.PriceTransformer(config).requires_grad_(False)
    inputs = model_lib.example_inputs(config, 3, 'cpu', seed=1)

    def price(embedding):
        return model(embedding, *inputs[1:])

    tangents = (randn(*inputs[0].shape, seed=5),)
    assert torch.func.jvp(price, (inputs[0],), tangents)[1].abs().min() > 0
    model.set_dense_kernels()
    with pytest.raises(NotImplementedError, match='forward-mode'):
        torch.func.jvp(price, (inputs[0],), tangents)


# The operators without a derivative, as a function of one tensor.
def eight_bits(x):
    return dense.dequantize_rows(*dense.quantize_rows(x), torch.float32)


def second(x):
    w = randn(4, 8, seed=2, device=x.device)
    dy = randn(3, 4, seed=3, device=x.device)
    return torch.ops.vectra.linear_backward(dy, x, None, w, None, 'gelu', False, [True, False, False])[0]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('f', [eight_bits, second])
def test_a_gradient_through_an_operator_without_one_is_refused(f, device):
    x = randn(3, 8, seed=1, device=device)
    want = f(x)
    leaf = x.clone().requires_grad_()
    y = f(leaf)
    assert torch.equal(y, want) and y.requires_grad
    with pytest.raises(RuntimeError, match='not implemented'):
        torch.autograd.grad((y * leaf).sum(), leaf)
    with torch.no_grad():
        assert not f(leaf).requires_grad
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match='forward AD'):
        f(forward_ad.make_dual(x, torch.ones_like(x)))


def test_8_bit_rows_are_well_formed_where_a_gradient_is_asked_for():
    x = randn(3, 40, seed=1).requires_grad_()
    torch.library.opcheck(torch.ops.vectra.quantize_rows.default, (x,),
                          test_utils=('test_schema', 'test_faketensor', 'test_autograd_registration'))
    codes, scales = dense.quantize_rows(x.detach())
    torch.library.opcheck(torch.ops.vectra.dequantize_rows.default, (codes, scales, torch.float32),
                          test_utils=('test_faketensor',))
