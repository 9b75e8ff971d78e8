"""The price model on the dense operators: the same function and gradients as
its plain layers, alone and compiled, on the CPU and on the GPU."""

import copy

import pytest
import torch

from vectra_amd.compiler import backend
from vectra_amd.price_transformer import checkpoint
from vectra_amd.price_transformer import model as model_lib

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


def build(gate, device, layers=2):
    torch.manual_seed(0)
    config = model_lib.ModelConfig(d_model=48, num_heads=4, num_layers=layers, ffn_dim=80, num_candidates=12,
                                   embedding_dim=24, attribute_dim=7, ffn_gate=gate)
    plain = model_lib.PriceTransformer(config).to(device)
    inputs = model_lib.example_inputs(config, 9, device, seed=1)
    return config, plain, copy.deepcopy(plain).set_dense_kernels(), inputs


def gradients(model, inputs):
    model.zero_grad(set_to_none=True)
    out = model(*inputs)
    # Weighted so that no parameter's gradient cancels.
    (out * torch.linspace(0.5, 1.5, out.numel(), device=out.device)).sum().backward()
    return out.detach(), {name: p.grad for name, p in model.named_parameters()}


def relative(a, b):
    return float((a - b).norm() / b.norm().clamp_min(1e-12))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('gate', [False, True])
def test_same_outputs_and_gradients_as_the_plain_layers(device, gate):
    """fp32: two orders of the same sums.  Sums here have up to 80 terms in the
    layers and 9 * 13 rows in the weights' gradients; ten layers of them, each
    off by about sqrt(terms) 2^-24 of its size, stay below 1e-5; the softmax
    and the square distances between them amplify by less than 10."""
    _, plain, dense, inputs = build(gate, device)
    y0, g0 = gradients(plain, inputs)
    y1, g1 = gradients(dense, inputs)
    assert relative(y1, y0) < 1e-5
    assert g0.keys() == g1.keys()
    for name in g0:
        assert relative(g1[name], g0[name]) < 1e-4, name


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('gate', [False, True])
def test_training_with_inputs_kept_in_8_bits(device, gate):
    """The forward pass is unchanged; each gradient is off by what keeping
    inputs at half a code's step (2^-4 of an element, about 2^-5.5 of a row in
    the mean square) does to it."""
    _, _, dense, inputs = build(gate, device)
    y0, g0 = gradients(dense, inputs)
    y1, g1 = gradients(dense.set_dense_kernels(checkpoint='e4m3'), inputs)
    assert torch.equal(y0, y1)
    changed = 0
    for name in g0:
        assert g1[name].isfinite().all()
        assert relative(g1[name], g0[name]) < 0.25, name
        changed += not torch.equal(g1[name], g0[name])
    assert changed


@pytest.mark.parametrize('device', DEVICES)
def test_the_compiled_model_keeps_its_attention_sites(device):
    config, plain, dense, inputs = build(True, device)
    with torch.no_grad():
        compiled, report = backend.compile_for_serving(dense.eval(), tuple(inputs), expected_sites=config.num_layers)
        got, want = compiled(*inputs), plain.eval()(*inputs)
    assert report.sites == config.num_layers and report.graph_break_count == 0
    assert relative(got, want) < 1e-5


def test_switching_back_and_refusals():
    _, plain, dense, inputs = build(False, 'cpu')
    with torch.no_grad():
        assert torch.equal(dense.set_dense_kernels(False)(*inputs), plain(*inputs))
    with pytest.raises(ValueError, match='checkpoint'):
        dense.set_dense_kernels(checkpoint='int8')


def test_a_gated_checkpoint_round_trips(tmp_path):
    _, plain, _, inputs = build(True, 'cpu')
    checkpoint.save(str(tmp_path), plain)
    again = checkpoint.load(str(tmp_path))
    assert again.config == plain.config and again.config.ffn_gate
    with torch.no_grad():
        assert torch.equal(again(*inputs), plain.eval()(*inputs))


def test_a_plain_configuration_is_written_as_before():
    assert 'ffn_gate' not in model_lib.ModelConfig().to_dict()
    assert model_lib.ModelConfig.from_dict(model_lib.ModelConfig(ffn_gate=True).to_dict()).ffn_gate


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_half_precision_blocks_train(dtype):
    """Against the same half-precision model on plain layers: both round every
    layer's output, in other places; a few steps of 2^-8 (bf16) per layer."""
    _, plain, dense, inputs = build(True, 'cuda')
    y0, g0 = gradients(plain.set_block_dtype(dtype), inputs)
    y1, g1 = gradients(dense.set_block_dtype(dtype), inputs)
    assert relative(y1, y0) < 2 ** -8
    for name in g0:
        assert g1[name].dtype == g0[name].dtype and g1[name].isfinite().all()
        assert relative(g1[name].float(), g0[name].float()) < 0.1, name
