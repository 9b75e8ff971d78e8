"""How a program draws dropout anew with each pass: torch.ops.vectra.dropout_pass, and
the price model that uses it, eager, compiled and captured.  The gradients belong to the
elements that the forward pass dropped."""

import copy

import pytest
import torch
import torch.distributed as dist
from torch import multiprocessing
from torch import nn

from torch.utils._python_dispatch import TorchDispatchMode
from torch.utils.checkpoint import checkpoint

from vectra_amd.compiler import backend  # noqa: F401  (registers the backend 'vectra')
from vectra_amd.kernels import block
from vectra_amd.price_transformer import model as model_lib

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


def build(device='cpu', dropout=0.5, layers=2, gate=False):
    torch.manual_seed(0)
    config = model_lib.ModelConfig(d_model=48, num_heads=4, num_layers=layers, ffn_dim=80, num_candidates=12,
                                   embedding_dim=24, attribute_dim=7, ffn_gate=gate, dropout=dropout)
    return model_lib.PriceTransformer(config).to(device), model_lib.example_inputs(config, 9, device, seed=1)


def gradients(outs, parameters):
    """One backward pass per output, after all the forward passes."""
    weights = [torch.linspace(0.5, 1.5, out.numel(), device=out.device) for out in outs]
    return [torch.autograd.grad((out * w).sum(), parameters) for out, w in zip(outs, weights)]


def relative(a, b):
    a, b = a.detach().float(), b.detach().float()
    return float((a - b).norm() / b.norm().clamp_min(1e-12))


# ------------------------------------------------------------------- the operator


@pytest.mark.parametrize('device', DEVICES)
def test_a_pass_is_a_copy_and_the_state_is_counted_on(device):
    state = torch.tensor([-5, 2 ** 40 - 1], device=device)
    passes = [block.dropout_pass(state) for _ in range(3)]
    assert [p.tolist() for p in passes] == [[-5, 2 ** 40 - 1 + i] for i in range(3)]
    assert state.tolist() == [-5, 2 ** 40 + 2]
    apart = torch.tensor([[3, 9], [4, 9]], device=device)[:, 0]  # (of any stride)
    assert block.dropout_pass(apart).tolist() == [3, 4] and apart.tolist() == [3, 5]
    for bad in (state.float(), state[:1], state[None], state.int()):
        with pytest.raises(RuntimeError, match='state must be two int64'):
            block.dropout_pass(bad)


def test_a_state_that_was_drawn_from_itself_is_noticed():
    x, state = torch.randn(4, 9).requires_grad_(), torch.tensor([3, 0])
    y = block.dropout(x, 0.3, state)
    block.dropout_pass(state)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()


def test_opcheck():
    torch.library.opcheck(torch.ops.vectra.dropout_pass.default, (torch.tensor([3, 0]),),
                          test_utils=('test_schema', 'test_faketensor'))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('compiler', ['aot_eager', 'inductor'])
def test_compiled_passes_of_a_program(compiler, device):
    """Dropout alone and in a norm; the backward passes after both forward passes.  Two
    orders of fp32 sums over 48 and 640 terms: below 1e-5."""
    x, w = (torch.randn(n, 48, generator=torch.Generator().manual_seed(n)).to(device).requires_grad_() for n in (640, 48))

    def step(x, w, state):
        rng = block.dropout_pass(state)
        y = block.dropout(x @ w.t(), 0.5, rng, 1)
        h, n = block.residual_norm(y @ w, x, p=0.25, rng=rng, stream=2)
        return (h.sin() * n).sum(1)

    torch._dynamo.reset()
    compiled = torch.compile(step, backend=compiler, fullgraph=True)
    runs = []
    for f in (step, compiled):
        state = torch.tensor([3, 7], device=device)
        outs = [f(x, w, state) for _ in range(2)]
        assert state.tolist() == [3, 9]
        runs.append((outs, gradients(outs, [x, w])))
    for a, b in zip(runs[1][0], runs[0][0]):
        assert relative(a, b) < 1e-5
    for got, want in zip(runs[1][1], runs[0][1]):
        assert all(relative(a, b) < 1e-5 for a, b in zip(got, want))


# ------------------------------------------------------------------ the price model


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('fused', [False, True])
@pytest.mark.parametrize('compiler', ['inductor', 'vectra'])
def test_the_compiled_model_trains_as_the_eager_one(compiler, fused, device):
    """fp32, two orders of the same sums through two blocks: outputs within 1e-5, gradients
    within 1e-4 (as the fused model's against the plain one's)."""
    model, inputs = build(device)
    model.set_norm_kernels(fused).seed_dropout(11)
    twin = copy.deepcopy(model)
    torch._dynamo.reset()
    compiled = torch.compile(twin, backend=compiler)
    outs, own = ([m(*inputs) for _ in range(2)] for m in (model, compiled))
    assert twin.dropout_rng.tolist() == model.dropout_rng.tolist() == [11, 2]
    assert not torch.equal(outs[0], outs[1])
    for a, b in zip(own, outs):
        assert relative(a, b) < 1e-5
    want, got = gradients(outs, list(model.parameters())), gradients(own, list(twin.parameters()))
    for i in range(2):
        for (name, _), a, b in zip(model.named_parameters(), got[i], want[i]):
            assert relative(a, b) < 1e-4, (i, name)


@pytest.mark.gpu
@pytest.mark.parametrize('fused', [False, True])
def test_captured_passes_of_the_model_draw_anew(fused):
    model, inputs = build('cuda')
    model.set_norm_kernels(fused).seed_dropout(11)
    with torch.no_grad():
        want = [model(*inputs) for _ in range(4)]
        torch.cuda.synchronize()
        model.seed_dropout(11)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = model(*inputs)
        assert model.dropout_rng.tolist() == [11, 0]
        for i in range(4):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[i]), i
    assert model.dropout_rng.tolist() == [11, 4]


# ------------------------------------------------------------ passes that are run again


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('fused', [False, True])
def test_a_model_that_is_run_again_drops_the_same_elements(fused, device):
    """Activation checkpointing of the whole model, of a compiled one and in one; the same
    operations in the same order where nothing is compiled."""
    model, inputs = build(device)
    model.set_norm_kernels(fused).seed_dropout(11)
    weights = list(model.parameters())
    outs = [model(*inputs) for _ in range(2)]
    want = gradients(outs, weights)

    def again(m):
        return lambda *args: checkpoint(m, *args, use_reentrant=False)

    torch._dynamo.reset()
    for run, most in ((again(model), 0.0), (again(torch.compile(model)), 1e-4), (torch.compile(again(model)), 1e-4)):
        model.seed_dropout(11)
        own = [run(*inputs, model.dropout_pass()) for _ in range(2)]
        assert model.dropout_rng.tolist() == [11, 2]
        for got, expected in zip(gradients(own, weights), want):
            assert all(relative(a, b) <= most for a, b in zip(got, expected))
        assert model.dropout_rng.tolist() == [11, 2]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('fused', [False, True])
def test_a_model_that_would_draw_again_in_the_backward_pass_is_refused(fused, device):
    model, inputs = build(device)
    model.set_norm_kernels(fused).seed_dropout(11)
    out = checkpoint(model, *inputs, use_reentrant=False)
    with pytest.raises(RuntimeError, match='within a backward pass'):
        out.sum().backward()
    inputs[0].requires_grad_()
    out = checkpoint(model, *inputs, use_reentrant=True)
    with pytest.raises(RuntimeError, match='within a backward pass'):
        out.sum().backward()
    torch._dynamo.reset()
    compiled = torch.compile(model)
    for run in (lambda *args: checkpoint(compiled, *args, use_reentrant=False),
                torch.compile(lambda *args: checkpoint(model, *args, use_reentrant=False))):
        with pytest.raises(RuntimeError):
            run(*inputs).sum().backward()
    checkpoint(model.eval(), *inputs, use_reentrant=False).sum().backward()  # (nothing is dropped)


def test_single_blocks_that_are_run_again_drop_the_same_elements():
    model, inputs = build()
    twin = copy.deepcopy(model)
    for b in twin.blocks:
        b.forward = lambda *args, own=b.forward: checkpoint(own, *args, use_reentrant=False)
    want, got = (gradients([m.seed_dropout(11)(*inputs)], list(m.parameters()))[0] for m in (model, twin))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_draws_that_the_caller_takes():
    model, inputs = build()
    with torch.no_grad():
        rng = model.seed_dropout(11).dropout_pass()
        assert rng.tolist() == [11, 0] and model.dropout_rng.tolist() == [11, 1]
        first, again = model(*inputs, rng), model(*inputs, rng=rng)
        assert torch.equal(first, again) and torch.equal(first, model.seed_dropout(11)(*inputs))
        assert torch.equal(model.eval()(*inputs, rng), model(*inputs))  # (nothing is dropped)
        assert model.dropout_pass() is None and model.dropout_rng.tolist() == [11, 1]
        plain, _ = build(dropout=0.0)
        assert plain.dropout_pass() is None and torch.equal(plain(*inputs, rng), plain(*inputs))


# ------------------------------------------------------------------ what is dropped


class Draws(TorchDispatchMode):
    """The stream numbers that a run draws with, in order."""

    def __init__(self):
        super().__init__()
        self.streams = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        kwargs = kwargs or {}
        if func is torch.ops.vectra.dropout.default:
            self.streams.append(args[3] if len(args) > 3 else kwargs.get('stream', 0))
        elif func is torch.ops.vectra.residual_norm.default and kwargs.get('p', 0.0) > 0:
            self.streams.append(kwargs.get('stream', 0))
        return func(*args, **kwargs)


def draws(model, inputs):
    with torch.no_grad(), Draws() as seen:
        model(*inputs)
    return seen.streams


@pytest.mark.parametrize('fused', [False, True])
def test_a_block_in_eval_mode_drops_nothing(fused):
    """As nn.Dropout inside of it would: by its own flag, whatever the model's is."""
    model, inputs = build(layers=3)
    model.set_norm_kernels(fused)
    with torch.no_grad():
        still = copy.deepcopy(model).eval()(*inputs)
        model.blocks.eval()
        assert model.training and draws(model, inputs) == []
        assert torch.equal(model(*inputs), still) and model.dropout_rng[1] == 0
        assert torch.equal(model(*inputs, torch.tensor([1, 2])), still)
        model.blocks[1].train()
        assert draws(model, inputs) == [2, 3] and model.dropout_rng[1] == 1
        assert not torch.equal(model(*inputs), still)
        model.eval()
        model.blocks[2].train()
        assert draws(model, inputs) == [4, 5]


@pytest.mark.parametrize('dense', [False, True])
@pytest.mark.parametrize('gate', [False, True])
@pytest.mark.parametrize('fused', [False, True])
def test_a_run_draws_each_branch_with_a_number_of_its_own(fused, gate, dense):
    """In a whole forward pass, and as many in its backward one."""
    model, inputs = build(layers=3, gate=gate)
    model.set_norm_kernels(fused)
    if dense:
        model.set_dense_kernels()
    assert draws(model, inputs) == [0, 1, 2, 3, 4, 5]
    with Draws() as seen:
        model(*inputs).sum().backward()
    if not fused:  # (the fused backward operator draws the branches that it joins)
        assert sorted(seen.streams) == [i // 2 for i in range(12)]


# ------------------------------------------------------- where the generator's state is


class Loss(torch.nn.Module):
    """A model inside another, as a loss that wraps it."""

    def __init__(self, model):
        super().__init__()
        self.model = model

    def forward(self, *inputs):
        return self.model(*inputs)


def data_parallel_rank(rank, path):
    """Two replicas with seeds of their own drop by their own seeds and keep equal weights."""
    dist.init_process_group('gloo', init_method=f'file://{path}', rank=rank, world_size=2)
    torch.set_num_threads(1)
    for wrap in (lambda m: m, Loss):
        model, inputs = build()
        model.seed_dropout(100 + rank)
        alone = copy.deepcopy(model)
        replica = nn.parallel.DistributedDataParallel(wrap(model))
        for i in range(2):
            out = replica(*inputs)
            assert torch.equal(out, alone(*inputs)), (rank, i)
            assert model.dropout_rng.tolist() == [100 + rank, i + 1]
            out.sum().backward()
        grads = [torch.zeros_like(model.head.weight) for _ in range(2)]
        dist.all_gather(grads, model.head.weight.grad)
        assert torch.equal(grads[0], grads[1])
    dist.destroy_process_group()


def test_data_parallel_ranks_draw_by_their_own_seeds(tmp_path):
    multiprocessing.spawn(data_parallel_rank, (str(tmp_path / 'store'),), nprocs=2)


@pytest.mark.parametrize('device', DEVICES)
def test_the_state_moves_with_the_model(device, tmp_path):
    model, inputs = build()
    model.seed_dropout(11, 5)
    with torch.no_grad():
        want = model(*inputs)
        model.half().float()
        assert model.dropout_rng.dtype == torch.int64
        moved = copy.deepcopy(model).to(device).seed_dropout(11, 5)
        assert moved.dropout_rng.device.type == device and moved.dropout_rng is not model.dropout_rng
        moved(*(t.to(device) for t in inputs))
        assert moved.dropout_rng.tolist() == [11, 6] and moved.to('cpu').dropout_rng.tolist() == [11, 6]
        # Pickled and restored, and made without memory, which leaves the state as it was made.
        torch.save(model, tmp_path / 'model.pt')
        again = torch.load(tmp_path / 'model.pt', weights_only=False)
        assert again.dropout_rng.tolist() == [11, 6] and torch.equal(again.seed_dropout(11, 5).to('cpu')(*inputs), model.seed_dropout(11, 5)(*inputs))
        torch.manual_seed(77)
        with torch.device('meta'):
            empty = model_lib.PriceTransformer(model.config)
        assert empty.to_empty(device=device).dropout_rng.tolist() == [77, 0]
        assert empty.dropout_rng.device.type == device
        assert empty.to('meta').to_empty(device=device).dropout_rng.tolist() == [77, 0]
    assert relative(want, model.seed_dropout(11, 5)(*inputs)) < 1e-2  # (once through fp16)
    assert 'dropout_rng' not in model.state_dict()


@pytest.mark.gpu
def test_the_state_follows_weights_that_are_moved_one_by_one():
    """As wrappers that shard a model do."""
    model, inputs = build('cuda')
    with torch.no_grad():
        want = model.seed_dropout(11, 5)(*inputs)
        model.seed_dropout(11, 5)
        model.dropout_rng = model.dropout_rng.cpu()
        assert torch.equal(model(*inputs), want)
    assert model.dropout_rng.is_cuda and model.dropout_rng.tolist() == [11, 6]


@pytest.mark.parametrize('fused', [False, True])
def test_a_pass_makes_no_modules(fused, monkeypatch):
    """(A slice of a module list is a new one, 26 us of host time.)"""
    model, inputs = build()
    model.set_norm_kernels(fused)
    made = []
    real = nn.Module.__init__
    monkeypatch.setattr(nn.Module, '__init__', lambda self, *args, **kwargs: (made.append(type(self)), real(self, *args, **kwargs))[1])
    with torch.no_grad():
        model(*inputs)
    assert made == []
