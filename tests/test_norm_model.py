"""The price model on torch.ops.vectra.residual_norm and with dropout: the same
function and gradients as its plain layers, alone and beside the dense operators, and
what users put on its layers."""

import copy

import pytest
import torch
from torch import nn

from vectra_amd.compiler import backend
from vectra_amd.kernels import block as block_ops
from vectra_amd.kernels import dense as dense_ops
from vectra_amd.price_transformer import checkpoint
from vectra_amd.price_transformer import model as model_lib
from vectra_amd.price_transformer import plain_modules

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


def build(device='cpu', gate=False, dropout=0.0, layers=3):
    torch.manual_seed(0)
    config = model_lib.ModelConfig(d_model=48, num_heads=4, num_layers=layers, ffn_dim=80, num_candidates=12,
                                   embedding_dim=24, attribute_dim=7, ffn_gate=gate, dropout=dropout)
    model = model_lib.PriceTransformer(config).to(device)
    with torch.no_grad():  # (norms that do something)
        for name, p in model.named_parameters():
            if 'norm' in name:
                p.add_(0.2 * torch.randn(p.shape).to(device))
    return model, model_lib.example_inputs(config, 9, device, seed=1)


def gradients(model, inputs, autocast=None):
    model.zero_grad(set_to_none=True)
    with torch.autocast(inputs[0].device.type, autocast or torch.bfloat16, enabled=autocast is not None):
        out = model(*inputs)
    # Weighted so that no parameter's gradient cancels.
    (out * torch.linspace(0.5, 1.5, out.numel(), device=out.device)).sum().backward()
    return out.detach(), {name: p.grad for name, p in model.named_parameters()}


def relative(a, b):
    a, b = a.detach().float(), b.detach().float()
    return float((a - b).norm() / b.norm().clamp_min(1e-12))


def count(model, inputs, key='vectra::residual_norm'):
    with torch.no_grad(), torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        model(*inputs)
    return sum(e.count for e in prof.key_averages() if e.key == key)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dropout', [0.0, 0.25])
@pytest.mark.parametrize('gate', [False, True])
@pytest.mark.parametrize('dense', [False, True])
def test_same_outputs_and_gradients_as_the_plain_layers(dense, gate, dropout, device):
    """fp32: two orders of the same sums, of up to 80 terms in the layers, 48 in the norms
    and 9 * 13 rows in the weights' gradients; fifteen layers of them, each off by about
    sqrt(terms) 2^-24 of its size, stay below 1e-5; the softmax and the square distances
    between them amplify by less than 10.  With dropout both draw the same elements."""
    plain, inputs = build(device, gate, dropout)
    fused = copy.deepcopy(plain).set_norm_kernels()
    if dense:
        fused.set_dense_kernels()
    for _ in range(2):  # (the second pass draws anew)
        y0, g0 = gradients(plain, inputs)
        y1, g1 = gradients(fused, inputs)
        assert relative(y1, y0) < 1e-5
        assert g0.keys() == g1.keys()
        for name in g0:
            assert relative(g1[name], g0[name]) < 1e-4, name
    assert count(fused, inputs) == 2 * 3 - 1
    with torch.no_grad():
        assert torch.equal(fused.set_norm_kernels(False).set_dense_kernels(False).eval()(*inputs), plain.eval()(*inputs))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dense', [False, True])
def test_half_precision_and_autocast_train(dense, device):
    """Against the plain layers in the same precision: both round every layer's output, in
    other places; a few steps of 2^-8 (bf16) per layer, and the stream itself with the
    blocks in bf16."""
    plain, inputs = build(device, True, 0.25)
    fused = copy.deepcopy(plain).set_norm_kernels()
    if dense:
        fused.set_dense_kernels()
    for autocast in (torch.bfloat16, None):
        if autocast is None:
            plain.set_block_dtype(torch.bfloat16)
            fused.set_block_dtype(torch.bfloat16)
        y0, g0 = gradients(plain, inputs, autocast)
        y1, g1 = gradients(fused, inputs, autocast)
        assert y1.dtype == y0.dtype and relative(y1, y0) < 2 ** -8
        for name in g0:
            assert g1[name].dtype == g0[name].dtype and g1[name].isfinite().all()
            assert relative(g1[name], g0[name]) < 0.1, name
    assert count(fused, inputs) == 2 * 3 - 1


@pytest.mark.parametrize('device', DEVICES)
def test_the_compiled_model_keeps_its_attention_sites(device):
    plain, inputs = build(device, dropout=0.5)
    fused = copy.deepcopy(plain).set_norm_kernels().set_dense_kernels().eval()
    with torch.no_grad():
        compiled, report = backend.compile_for_serving(fused, tuple(inputs), expected_sites=3)
        got, want = compiled(*inputs), plain.eval()(*inputs)
    assert report.sites == 3 and report.graph_break_count == 0
    assert relative(got, want) < 1e-5


# ------------------------------------------------------------------------ dropout


@pytest.mark.parametrize('fused', [False, True])
def test_dropout_draws_anew_with_each_pass_and_again_from_its_seed(fused):
    model, inputs = build(dropout=0.5)
    model.set_norm_kernels(fused).seed_dropout(11)
    with torch.no_grad():
        first, second = model(*inputs), model(*inputs)
        assert not torch.equal(first, second)
        assert model.dropout_rng.tolist() == [11, 2]
        assert torch.equal(model.seed_dropout(11)(*inputs), first)
        assert torch.equal(model.seed_dropout(11, 1)(*inputs), second)
        assert not torch.equal(model.seed_dropout(12)(*inputs), first)
        still = model.eval()(*inputs)
        assert torch.equal(model(*inputs), still) and model.dropout_rng.tolist() == [12, 1]


def test_each_branch_of_each_block_has_a_stream_of_its_own():
    model, inputs = build(dropout=0.5)
    seen = []
    real = torch.ops.vectra.dropout
    rng = torch.tensor([3, 0])
    x = torch.ones(9, 13, 48)
    for b in model.blocks:
        seen += [b._drop(x, rng, 2 * b.index), b._drop(x, rng, 2 * b.index + 1)]
    assert all(torch.equal(s, real(x, 0.5, rng, i)) for i, s in enumerate(seen))
    assert len({tuple(s.flatten().tolist()) for s in seen}) == 2 * 3


@pytest.mark.parametrize('fused', [False, True])
def test_two_passes_before_their_backward_passes(fused):
    """Each backward pass drops what its own forward pass dropped."""
    model, inputs = build(dropout=0.5)
    model.set_norm_kernels(fused)
    weights = list(model.parameters())
    want = [torch.autograd.grad(model.seed_dropout(5, i)(*inputs).sum(), weights) for i in range(2)]
    model.seed_dropout(5)
    outs = [model(*inputs) for _ in range(2)]
    for out, w in zip(outs, want):
        for a, b in zip(torch.autograd.grad(out.sum(), weights), w):
            assert torch.equal(a, b)


def test_configuration_and_checkpoints(tmp_path):
    assert 'dropout' not in model_lib.ModelConfig().to_dict()
    assert model_lib.ModelConfig.from_dict(model_lib.ModelConfig(dropout=0.1).to_dict()).dropout == 0.1
    plain, inputs = build()
    with_dropout, _ = build(dropout=0.25)
    assert plain.state_dict().keys() == with_dropout.state_dict().keys()
    assert not list(plain.buffers())
    checkpoint.save(str(tmp_path), with_dropout)
    again = checkpoint.load(str(tmp_path))
    assert again.config == with_dropout.config
    with torch.no_grad():
        assert torch.equal(again(*inputs), plain.eval()(*inputs))
    for bad in (-0.1, 1.0, 1 - 2 ** -18, float('nan')):
        with pytest.raises(ValueError, match='dropout'):
            build(dropout=bad)
    with pytest.raises(ValueError, match='no dropout'):
        plain.seed_dropout(1)


def test_a_model_too_wide_for_the_norms_is_refused():
    config = model_lib.ModelConfig(d_model=block_ops.NORM_WIDTH + 4, num_layers=0)
    with torch.device('meta'):
        model = model_lib.PriceTransformer(config)
    with pytest.raises(ValueError, match='widest'):
        model.set_norm_kernels()


def test_modules_restored_without_the_switches_run_plain():
    """A module pickled before they existed holds none of their attributes."""
    model, inputs = build()
    with torch.no_grad():
        want = model(*inputs)
        for m in model.modules():
            for name in ('norm_kernels', 'dropout', 'index'):
                m.__dict__.pop(name, None)
        model.config.__dict__.pop('dropout')
        assert torch.equal(model(*inputs), want)


# ------------------------------------------------- hooks, wrappers and replacements


@pytest.mark.parametrize('register', ['register_forward_hook', 'register_forward_pre_hook',
                                      'register_full_backward_hook', 'register_full_backward_pre_hook'])
def test_every_hook_runs_as_on_the_plain_model(register):
    model, inputs = build()

    def calls(m):
        seen = []
        for name, sub in m.named_modules():
            getattr(sub, register)(lambda *args, name=name: seen.append(name))
        out = m(*inputs)
        out.sum().backward()
        return seen, out.detach()

    want, want_y = calls(copy.deepcopy(model))
    got, y = calls(copy.deepcopy(model).set_norm_kernels())
    assert got == want and len(want) > 20
    assert relative(y, want_y) < 1e-5


@pytest.mark.parametrize('name', ['blocks.0', 'blocks.1', 'blocks.0.norm1', 'blocks.1.norm1', 'blocks.1.norm2',
                                  'blocks.2.norm2', 'blocks.1.attention', 'blocks.1.ffn', 'norm'])
def test_a_hook_may_change_what_a_layer_gives(name):
    model, inputs = build()
    pair = [copy.deepcopy(model), copy.deepcopy(model).set_norm_kernels()]
    for m in pair:
        m.get_submodule(name).register_forward_hook(lambda module, args, out: out * 1.5)
    with torch.no_grad():
        want, got = (m(*inputs) for m in pair)
        assert not torch.equal(want, model(*inputs))
    assert relative(got, want) < 1e-5


class Forwarding(nn.Module):
    """A wrapper that hands on its inner module's attributes, as those for
    recomputation and sharding do, and takes two arguments."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, *args):
        return 1.5 * self.inner(*args)

    def __getattr__(self, name):
        try:
            return super().__getattr__(name)
        except AttributeError:
            return getattr(super().__getattr__('inner'), name)


def rms_norm(m):
    return nn.RMSNorm(m.normalized_shape[0])


def unscaled(m):
    return nn.LayerNorm(m.normalized_shape, elementwise_affine=False)


def of_more(m):
    return nn.LayerNorm((13, *m.normalized_shape))


@pytest.mark.parametrize('name,change,sites', [
    ('blocks.1', Forwarding, 3), ('blocks.0', Forwarding, 4), ('blocks.2', Forwarding, 4),
    ('blocks.1.norm1', Forwarding, 4), ('blocks.1.norm2', Forwarding, 4), ('blocks.1.norm1', rms_norm, 4),
    ('blocks.1.norm2', rms_norm, 4), ('blocks.1.norm1', of_more, 4), ('blocks.1.norm2', of_more, 4),
    ('blocks.1.norm1', unscaled, 5), ('blocks.1.norm2', unscaled, 5), ('blocks.0.norm1', rms_norm, 5),
    ('blocks.1.attention', Forwarding, 5), ('blocks.1.ffn', Forwarding, 5)])
@pytest.mark.parametrize('dense', [False, True])
def test_replaced_layers_run_as_they_are(name, change, sites, dense):
    model, inputs = build()
    model.set_submodule(name, change(model.get_submodule(name)))
    with torch.no_grad():
        want = model(*inputs)
        model.set_norm_kernels()
        if dense:
            model.set_dense_kernels()
        assert relative(model(*inputs), want) < 1e-5
        assert count(model, inputs) == sites
        model.set_norm_kernels(False)
        assert count(model, inputs) == 0


def test_which_norms_are_plain():
    assert plain_modules.is_plain_norm(nn.LayerNorm(8), 8)
    assert not plain_modules.is_plain_norm(nn.LayerNorm(8), 16)
    assert not plain_modules.is_plain_norm(nn.LayerNorm((2, 8)), 8)
    assert not plain_modules.is_plain_norm(nn.RMSNorm(8), 8)


# ------------------------------------------------------- a run of the operators together


def training_pass(leaves, x, rng):
    """Two branches of a block, a gated feed-forward and a dense layer, with their
    residual sums, norms and dropout, on a stream of fp32 beside bf16 branches."""
    w_gate_up, w_down, w_out, norm_a, norm_b, scale = leaves
    first = torch.ops.vectra.dropout(x, 0.125, rng, 0)
    h, n = torch.ops.vectra.residual_norm(first, x.float(), norm_a, norm='rms')
    hidden = torch.ops.vectra.gated_linear(n, w_gate_up, None, 'silu')
    branch = torch.ops.vectra.linear(hidden, w_down)
    h, n = torch.ops.vectra.residual_norm(branch, h, norm_b, None, scale, norm='rms', post='rms', p=0.25, rng=rng, stream=1)
    return h, torch.ops.vectra.linear(n, w_out)


def make_pass(device, rows=70, width=136, hidden=200):
    torch.manual_seed(3)
    shapes = [(2 * hidden, width), (width, hidden), (width, width)]
    leaves = [(torch.randn(s) / s[1] ** 0.5).to(device, torch.bfloat16).requires_grad_() for s in shapes]
    leaves += [(1 + 0.1 * torch.randn(width)).to(device).requires_grad_() for _ in range(3)]
    return leaves, torch.randn(2, rows // 2, width).to(device, torch.bfloat16), torch.tensor([17, 4], device=device)


@pytest.mark.parametrize('device', DEVICES)
def test_a_run_of_them_together_against_plain_products(device):
    """In float64 from the same elements dropped.  Six roundings to bf16 (2^-9 of each
    value at most in the mean square) lie between a leaf and the loss, forward and
    backward: 0.03 of a gradient's norm holds several times that."""
    leaves, x, rng = make_pass(device)
    h, y = training_pass(leaves, x, rng)
    gh, gy = torch.randn_like(h), torch.randn_like(y)
    got = torch.autograd.grad([h, y], leaves, [gh, gy])

    kept = [torch.ops.vectra.dropout(torch.ones_like(x), p, rng, i).cpu().double() for i, p in enumerate((0.125, 0.25))]
    l64 = [t.detach().cpu().double().requires_grad_() for t in leaves]
    w_gate_up, w_down, w_out, norm_a, norm_b, scale = l64

    def rms(t):
        return t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt()

    x64 = x.cpu().double()
    h64 = x64 + x64 * kept[0]
    gate, up = ((rms(h64) * norm_a) @ w_gate_up.t()).chunk(2, -1)
    branch = (nn.functional.silu(gate) * up) @ w_down.t()
    h64 = h64 + scale * kept[1] * rms(branch)
    y64 = (rms(h64) * norm_b) @ w_out.t()
    assert relative(h.cpu(), h64) < 0.01 and relative(y.cpu(), y64) < 0.02
    want = torch.autograd.grad([h64, y64], l64, [gh.cpu().double(), gy.cpu().double()])
    for i, (a, b) in enumerate(zip(got, want)):
        assert a.isfinite().all() and relative(a.cpu(), b) < 0.03, i


@pytest.mark.gpu
def test_a_captured_run_draws_as_the_eager_one():
    """Forward and backward in a HIP graph, its generator counted on by the program
    between the replays; each replay equals the eager pass with the same counter."""
    assert dense_ops.CHECKPOINTS  # (the dense operators are registered)
    leaves, x, rng = make_pass('cuda')
    h, y = training_pass(leaves, x, rng)
    gh, gy = torch.randn_like(h), torch.randn_like(y)

    def eager(offset):
        own = torch.tensor([17, offset], device='cuda')
        h, y = training_pass(leaves, x, own)
        return [h.detach(), y.detach(), *torch.autograd.grad([h, y], leaves, [gh, gy])]

    want = [eager(4 + i) for i in range(4)]
    del h, y  # (no eager graph over the leaves lives on)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager(4)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, y = training_pass(leaves, x, rng)
        got = [h.detach(), y.detach(), *torch.autograd.grad([h, y], leaves, [gh, gy])]
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want[i]):
            assert torch.equal(a, b), i
        rng[1].add_(1)
        for t in got:
            t.zero_()


@pytest.mark.parametrize('device', DEVICES)
def test_a_run_of_the_serving_forms(device):
    """A block's feed-forward part in 8 bits, one token at a time and in a batch: a norm
    into 8 bits, the gated layer, the next layer onto the stream.  Against the same with
    its operands' 8-bit values in float64: sums of exact products, the hidden values
    rounded once to bf16 and once to codes, half a step of 2^-4 each at most."""
    torch.manual_seed(4)
    width, hidden = 200, 136
    up = torch.ops.vectra.quantize_blocks((torch.randn(2 * hidden, width) / width ** 0.5).to(device), True)
    down = torch.ops.vectra.quantize_blocks((torch.randn(width, hidden) / hidden ** 0.5).to(device), True)
    weight = (1 + 0.1 * torch.randn(width)).to(device)

    def values(codes, scales, rows, columns, tiles):
        c = codes[:rows].cpu().double()
        s = torch.exp2(scales.view(torch.uint8).cpu().double() - 127)
        if tiles:
            s = s.repeat_interleave(128, 0)[:rows]
        return (c * s.repeat_interleave(128, 1)[:, :c.shape[1]])[:, :columns]

    for rows in (1, 3, 70):
        x, r = torch.randn(rows, width).to(device, torch.bfloat16), torch.randn(rows, width).to(device, torch.bfloat16)
        h, codes, scales = torch.ops.vectra.residual_norm_8bit(x, r, weight)
        mid = torch.ops.vectra.gated_linear_8bit(codes, *up, scales=scales, dtype=torch.bfloat16)
        out = torch.ops.vectra.linear_8bit(mid, *down, None, h)
        n64 = values(codes, scales, rows, width, False)
        a, b = (n64 @ values(*up, 2 * hidden, width, True).t()).chunk(2, -1)
        mid64 = nn.functional.silu(a) * b
        assert relative(mid.cpu(), mid64) < 2 ** -8
        out64 = h.cpu().double() + values(*torch.ops.vectra.quantize_blocks(mid), rows, hidden, False) @ values(
            *down, width, hidden, True).t()
        assert out.shape == (rows, width) and relative(out.cpu(), out64) < 2 ** -8
