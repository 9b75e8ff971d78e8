"""The dense operators are well-formed PyTorch operators (CPU checks): schemas,
the CPU implementation against the 64-bit oracle, gradients against
differences, tracing, and every refusal."""

import numpy as np
import pytest
import torch

from oracle import dense as oracle
from vectra_amd.kernels import dense

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ops = torch.ops.vectra


def make(rows, width_in, width_out, dtype=torch.float32, gated=False, bias=True, residual=False, seed=0):
    gen = torch.Generator().manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen)

    n = width_out * (2 if gated else 1)
    return dict(
        x=randn(rows, width_in).to(dtype),
        weight=(randn(n, width_in) * max(width_in, 1) ** -0.5).to(dtype),
        bias=(0.1 * randn(n)).to(dtype) if bias else None,
        residual=randn(rows, width_out).to(dtype) if residual else None,
        grad=randn(rows, width_out).to(dtype),
    )


def test_schemas():
    assert str(ops.linear.default._schema) == (
        "vectra::linear(Tensor x, Tensor weight, Tensor? bias=None, Tensor? residual=None, "
        'str activation="none", str checkpoint="none") -> Tensor')
    assert str(ops.gated_linear.default._schema) == (
        'vectra::gated_linear(Tensor x, Tensor weight, Tensor? bias=None, str activation="silu", '
        'str checkpoint="none") -> Tensor')
    assert str(ops.quantize_rows.default._schema) == 'vectra::quantize_rows(Tensor x) -> (Tensor, Tensor)'


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('activation', dense.ACTIVATIONS)
@pytest.mark.parametrize('gated', [False, True])
def test_cpu_layer_and_gradients_match_the_oracle(dtype, activation, gated):
    t = make(7, 13, 6, dtype, gated, residual=not gated)
    leaves = {k: v.requires_grad_() for k, v in t.items() if k != 'grad' and v is not None}
    if gated:
        y = dense.gated_linear(t['x'], t['weight'], t['bias'], activation)
    else:
        y = dense.linear(t['x'], t['weight'], t['bias'], t['residual'], activation)
    layer = oracle.Layer.of(t['x'], t['weight'], t['bias'], t['residual'], activation, gated)
    oracle.assert_within(y, *layer.forward(dtype))
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), t['grad'])))
    for name, (want, bound) in layer.backward(t['grad'], dtype, dtype).items():
        assert grads[name].dtype == dtype
        oracle.assert_within(grads[name], want, bound)
    if not gated:
        assert torch.equal(grads['residual'], t['grad'])


@pytest.mark.parametrize('activation', dense.ACTIVATIONS)
@pytest.mark.parametrize('gated', [False, True])
def test_the_oracles_gradients_are_its_differences(activation, gated):
    """The formulas themselves: a central difference of the 64-bit layer.  With
    step s the difference of a smooth f is off by s^2 f''' / 6 and by
    2^-52 |f| / s; s = 1e-5 leaves 1e-9 of the O(1) values here."""
    t = make(3, 5, 4, torch.float64, gated, seed=3)
    layer = oracle.Layer.of(t['x'], t['weight'], t['bias'], None, activation, gated)
    got = layer.backward(t['grad'], torch.float32, torch.float32)
    step = 1e-5
    for name in ('x', 'weight', 'bias'):
        at = getattr(layer, name)
        want = torch.zeros_like(at)
        for i in np.ndindex(*at.shape):
            kept = at[i].item()
            values = []
            for s in (step, -step):
                at[i] = kept + s
                values.append(float((layer.forward(torch.float32)[0] * t['grad']).sum()))
            at[i] = kept
            want[i] = (values[0] - values[1]) / (2 * step)
        assert float((got[name][0] - want).abs().max()) < 1e-7


@pytest.mark.parametrize('shape', [(4,), (2, 3, 5, 4), (0, 4), (3, 0)])
def test_leading_dimensions_and_empty_sizes(shape):
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(*shape, generator=gen, requires_grad=True)
    w = torch.randn(6, shape[-1], generator=gen, requires_grad=True)
    b = torch.randn(6, generator=gen, requires_grad=True)
    for y, want in ((dense.linear(x, w, b), torch.nn.functional.linear(x, w, b)),
                    (dense.gated_linear(x, w, b, 'relu'), None)):
        assert y.shape == (*shape[:-1], 6 if want is not None else 3)
        if want is not None:
            torch.testing.assert_close(y, want)
        grads = torch.autograd.grad(y.sum(), (x, w, b))
        assert [g.shape for g in grads] == [x.shape, w.shape, b.shape]
        if x.numel() == 0:
            assert not grads[1].any()


def test_a_wide_view_and_a_transposed_view():
    gen = torch.Generator().manual_seed(2)
    wide = torch.randn(9, 30, generator=gen)
    w = torch.randn(30, 8, generator=gen).t()
    for x in (wide[:, 11:22], torch.randn(11, 9, generator=gen).t()):
        weight = w[:, :11]
        torch.testing.assert_close(dense.linear(x, weight), x @ weight.t())


@pytest.mark.parametrize('checkpoint', dense.CHECKPOINTS)
@pytest.mark.parametrize('gated', [False, True])
def test_opcheck(checkpoint, gated):
    t = make(5, 12, 4, gated=gated)
    for name in ('x', 'weight', 'bias'):
        t[name].requires_grad_()
    tests = ('test_schema', 'test_faketensor', 'test_aot_dispatch_static')
    if gated:
        torch.library.opcheck(ops.gated_linear.default, (t['x'], t['weight'], t['bias'], 'silu', checkpoint),
                              test_utils=tests)
    else:
        torch.library.opcheck(ops.linear.default, (t['x'], t['weight'], t['bias'], None, 'gelu', checkpoint),
                              test_utils=tests)
    torch.library.opcheck(ops.quantize_rows.default, (t['x'].detach(),), test_utils=tests[:2])


def test_8_bit_gradients_are_those_at_the_kept_values():
    t = make(6, 70, 5, residual=True, seed=4)
    for name in ('x', 'weight', 'bias', 'residual'):
        t[name].requires_grad_()
    y = dense.linear(t['x'], t['weight'], t['bias'], t['residual'], 'gelu', 'e4m3')
    assert torch.equal(y, dense.linear(t['x'], t['weight'], t['bias'], t['residual'], 'gelu'))
    grads = torch.autograd.grad(y, (t['x'], t['weight'], t['bias']), t['grad'])
    kept = dense.dequantize_rows(*dense.quantize_rows(t['x'].detach()), torch.float32)
    layer = oracle.Layer.of(kept, t['weight'], t['bias'], None, 'gelu')
    for got, (want, bound) in zip(grads, layer.backward(t['grad'], torch.float32, torch.float32).values()):
        oracle.assert_within(got, want, bound)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('width', [1, 31, 32, 33, 100])
def test_8_bit_rows_match_the_oracle(dtype, width):
    gen = torch.Generator().manual_seed(width)
    x = torch.randn(40, width, generator=gen) * torch.exp2(torch.randint(-30, 16, (40, 1), generator=gen).float())
    x[3] = 0.0
    x[4, 0] = float('inf')
    x[5, 0] = float('nan')
    x[6] = torch.finfo(dtype).max
    x[7] = torch.finfo(dtype).tiny
    x = x.to(dtype)
    codes, scales = dense.quantize_rows(x)
    want_codes, want_scales = oracle.quantize(x)
    assert np.array_equal(scales.view(torch.uint8).numpy(), want_scales)
    got = codes.view(torch.uint8).numpy()
    nan = (want_codes & 0x7F) == 0x7F
    assert np.array_equal((got & 0x7F) == 0x7F, nan)
    assert np.array_equal(got[~nan], want_codes[~nan])
    back = dense.dequantize_rows(codes, scales, dtype)
    assert back.dtype == dtype
    want = oracle.dequantize(want_codes, want_scales)
    assert np.array_equal(back.double().numpy(), want, equal_nan=True)  # exact in the rows' own type
    # An element is off by at most half a code's step: 2^-4 of it, or 2^-10 of its block's power of two.
    xv = x.double().numpy()
    ok = np.isfinite(xv)
    power = np.exp2(np.repeat(want_scales.astype(np.float64) - 127, 32, axis=1)[:, :width])
    off = np.abs(want - xv)
    ok &= np.abs(xv) < 248 * 2.0 ** (8 if dtype == torch.float16 else 120)  # past it: the type's largest code, 240
    assert (off[ok] <= np.maximum(np.abs(xv) / 16, power / 1024)[ok]).all()


REFUSALS = {
    'width': (lambda: dense.linear(torch.zeros(2, 3), torch.zeros(4, 5)), RuntimeError, "not weight's"),
    'weight rank': (lambda: dense.linear(torch.zeros(2, 3), torch.zeros(3)), RuntimeError, 'weight'),
    'odd gate': (lambda: dense.gated_linear(torch.zeros(2, 3), torch.zeros(5, 3)), RuntimeError, 'up projection'),
    'dtype': (lambda: dense.linear(torch.zeros(2, 3).double(), torch.zeros(4, 3).double()), RuntimeError, 'float32'),
    'mixed': (lambda: dense.linear(torch.zeros(2, 3), torch.zeros(4, 3).half()), RuntimeError, 'share a dtype'),
    'bias shape': (lambda: dense.linear(torch.zeros(2, 3), torch.zeros(4, 3), torch.zeros(3)), RuntimeError, 'bias'),
    'bias dtype': (lambda: dense.linear(torch.zeros(2, 3), torch.zeros(4, 3), torch.zeros(4).half()), RuntimeError,
                   'bias'),
    'residual shape': (lambda: dense.linear(torch.zeros(2, 3), torch.zeros(4, 3), None, torch.zeros(1, 4)),
                       RuntimeError, 'residual'),
    'residual dtype': (lambda: dense.linear(torch.zeros(2, 3), torch.zeros(4, 3), None, torch.zeros(2, 4).half()),
                       RuntimeError, 'residual'),
    'activation': (lambda: dense.linear(torch.zeros(2, 3), torch.zeros(4, 3), activation='tanh'), ValueError,
                   'activation'),
    'checkpoint': (lambda: dense.gated_linear(torch.zeros(2, 3), torch.zeros(4, 3), checkpoint='int8'), ValueError,
                   'checkpoint'),
    'rows dtype': (lambda: dense.quantize_rows(torch.zeros(2, 3).double()), RuntimeError, 'float32'),
    'codes dtype': (lambda: dense.dequantize_rows(torch.zeros(2, 3), torch.zeros(2, 1), torch.float32), RuntimeError,
                    'float8'),
    'scales shape': (lambda: dense.dequantize_rows(torch.zeros(2, 33).to(torch.float8_e4m3fn),
                                                   torch.ones(2, 1).to(torch.float8_e8m0fnu), torch.float32),
                     RuntimeError, 'ceil'),
    'grad shape': (lambda: ops.linear_backward(torch.zeros(3, 4), torch.zeros(2, 3), None, torch.zeros(4, 3), None,
                                               'none', False, [True, True, False]), RuntimeError, 'grad'),
}


@pytest.mark.parametrize('name', REFUSALS)
def test_refusals(name):
    call, error, match = REFUSALS[name]
    with pytest.raises(error, match=match):
        call()


def test_gradients_of_gradients_are_refused():
    x = torch.randn(2, 3, requires_grad=True)
    w = torch.randn(4, 3, requires_grad=True)
    with pytest.raises(RuntimeError, match='gradients of gradients'):
        torch.autograd.grad(dense.linear(x, w, activation='silu').sum(), x, create_graph=True)


@pytest.mark.parametrize('wanted', [('x',), ('weight',), ('bias',), ('residual',), ('x', 'residual')])
def test_only_what_requires_a_gradient_gets_one(wanted):
    t = make(4, 6, 3, residual=True, seed=5)
    for name in wanted:
        t[name].requires_grad_()
    for activation in ('none', 'gelu'):
        y = dense.linear(t['x'], t['weight'], t['bias'], t['residual'], activation)
        got = torch.autograd.grad(y, [t[name] for name in wanted], t['grad'])
        layer = oracle.Layer.of(t['x'], t['weight'], t['bias'], t['residual'], activation)
        want = layer.backward(t['grad'], torch.float32, torch.float32)
        for name, g in zip(wanted, got):
            if name == 'residual':
                assert torch.equal(g, t['grad'])
            else:
                oracle.assert_within(g, *want[name])
