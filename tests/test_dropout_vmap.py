"""The operators that drop elements under torch.vmap: refused where every sample would
draw the same without a word, else each sample as a call of its own."""

import pytest
import torch

from vectra_amd.kernels import block

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]

CALLS = {
    'dropout': lambda x, r, rng, p: (block.dropout(x, p, rng, 3),),
    'residual_norm': lambda x, r, rng, p: block.residual_norm(x, r, p=p, rng=rng, stream=3),
    'residual_norm_8bit': lambda x, r, rng, p: block.residual_norm_8bit(x, r, p=p, rng=rng, stream=3),
}


def as_bytes(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('name', CALLS)
def test_samples_draw_by_their_own_rng_or_not_at_all(name, device):
    call = CALLS[name]
    x, r = (torch.randn(3, 5, 40, device=device) for _ in range(2))
    one, each = torch.tensor([3, 0], device=device), torch.tensor([[3, 0], [3, 1], [4, 0]], device=device)

    def same(got, rng_of, p=0.5):
        for i in range(3):
            want = call(x[i], r[i], rng_of(i), p)
            assert all(torch.equal(as_bytes(a[i]), as_bytes(b)) for a, b in zip(got, want))

    for randomness in ('error', 'different'):
        with pytest.raises(RuntimeError, match='same elements of every sample'):
            torch.vmap(lambda x, r: call(x, r, one, 0.5), randomness=randomness)(x, r)
        same(torch.vmap(lambda x, r, rng: call(x, r, rng, 0.5), randomness=randomness)(x, r, each), lambda i: each[i])
        same(torch.vmap(lambda x, r: call(x, r, one, 0.0), randomness=randomness)(x, r), lambda i: one, 0.0)
    same(torch.vmap(lambda x, r: call(x, r, one, 0.5), randomness='same')(x, r), lambda i: one)
    # An inner vmap over what is not dropped, and an rng of an outer one.
    shared = torch.vmap(lambda s: call(x[0], r[0], one, 0.5)[0].float() * s)(torch.ones(2, device=device))
    assert torch.equal(shared[0], call(x[0], r[0], one, 0.5)[0].float())
    with pytest.raises(RuntimeError, match='same elements of every sample'):
        torch.vmap(lambda rng: torch.vmap(lambda x, r: call(x, r, rng, 0.5))(x, r))(each)


@pytest.mark.parametrize('device', DEVICES)
def test_gradients_of_samples(device):
    x, each = torch.randn(3, 5, 40, device=device).requires_grad_(), torch.tensor([[3, 0], [3, 1], [4, 0]], device=device)
    y = torch.vmap(lambda x, rng: block.dropout(x, 0.5, rng))(x, each)
    dy = torch.randn_like(y)
    g, = torch.autograd.grad(y, x, dy)
    assert all(torch.equal(g[i], block.dropout(dy[i], 0.5, each[i])) for i in range(3))


@pytest.mark.parametrize('device', DEVICES)
def test_a_batch_of_gradients_of_one_pass_drops_what_the_pass_dropped(device):
    x, rng = torch.randn(5, 40, device=device).requires_grad_(), torch.tensor([3, 0], device=device)
    dy = torch.randn(4, 5, 40, device=device)
    g, = torch.autograd.grad(block.dropout(x, 0.5, rng), x, dy, is_grads_batched=True)
    assert all(torch.equal(g[i], block.dropout(dy[i], 0.5, rng)) for i in range(4))
