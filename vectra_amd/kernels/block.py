"""What stands between the dense operators of a Transformer block on MI355X:
dropout, and the residual stream with its norms.

  y = torch.ops.vectra.dropout(x, p, rng, stream=0)
  h, n = torch.ops.vectra.residual_norm(
      x, residual, weight=None, bias=None, gate=None, post_weight=None,
      post_bias=None, *, norm='rms', post='none', eps=1e-6,
      residual_scale=1.0, p=0.0, rng=None, stream=0)
      h = residual_scale * residual + gate * dropout(post_norm(x)),
      n = norm(h): a branch's output onto the residual stream, and what the
      next branch reads, in one pass
  h, codes, scales = torch.ops.vectra.residual_norm_8bit(...the same...)
      n in 8-bit rows, as torch.ops.vectra.linear_8bit reads them

x [..., width] is float32, float16 or bfloat16 (any strides; views without unit
element stride are copied); the residual, of x's shape, has x's type or float32
(a stream wider than its branches), and h has the residual's, n x's.  Rows of a
norm have at most 16,384 elements.  norm is 'rms' or 'layer', post 'none', 'rms'
or 'layer':

  rms    x / sqrt(mean(x^2) + eps) * weight + bias
  layer  (x - mean) / sqrt(var + eps) * weight + bias

weight, bias, post_weight, post_bias [width] and the gate are x's type or
float32, each by itself.  The gate is [width], or x's own shape with size 1 from
some dimension on: x [batch, tokens, width] takes [batch, 1, width] and
[batch, tokens, width].  Everything is computed in fp32; h and n are rounded
once each, n from the unrounded h.

Dropout keeps an element with probability 1 - t / 65536, t = round(65536 p), and
scales it by 65536 / (65536 - t); a dropped element is 0 whatever it held.  Which
are kept, a counter-based generator says (include/vectra_block.h states it):
its key and counter are the two int64 of `rng`, the seed and an offset (modulo
2^32), the number `stream` (one for each place of the program that draws) and the
element's position in x.  No mask is stored: the backward pass draws the same
again, from the same rng, which must therefore not be changed in place between
the two (autograd raises if it is).  dropout and residual_norm with equal rng,
stream and shape drop the same elements.  rng is read when the kernel runs, so a
program that replays a captured graph changes it between replays (rng[1].add_(1))
and draws anew.

dropout and residual_norm have gradients for every tensor argument but rng;
residual_norm keeps x and the residual for them where there is a gate or a post
norm, else h.  Gradients of gradients (of residual_norm) and forward-mode
derivatives are refused, and so is any derivative of residual_norm_8bit, a serving
form.  The gradients of the vectors are summed in fp32 in a fixed order.

A backward pass may be captured into a HIP graph through
torch.ops.vectra.residual_norm_backward, which autograd calls, and through
torch.ops.vectra.dropout on the gradient.  (Capturing torch.autograd.grad itself
while an eager graph over the same leaves is alive fails in autograd's own stream
bookkeeping: drop such graphs, outputs with a grad_fn, before the capture.)

The schemas, the CUDA-key implementations (libvectra_block.so on the current
stream), the CPU ones and the autograd rules live in
vectra_amd/csrc/ext/block_op.cpp.  This module registers the fake (meta)
implementations used while tracing and gives the operators Python names.
"""

import torch

from vectra_amd.kernels import _native

NORMS = ('rms', 'layer')
POST_NORMS = ('none', 'rms', 'layer')
BLOCK = 128  # elements of a row (and rows of a tile) that share a power of two

_native.load_torch_extension()


def _codes_shape(shape):
    return (*shape[:-1], (shape[-1] + BLOCK - 1) // BLOCK * BLOCK)


def _scales_shape(shape):
    return (*shape[:-1], (shape[-1] + 4 * BLOCK - 1) // (4 * BLOCK) * 4)


@torch.library.register_fake('vectra::dropout')
def _dropout_fake(x, p, rng, stream=0):
    del p, rng, stream
    return x.new_empty(x.shape)


@torch.library.register_fake('vectra::residual_norm')
def _residual_norm_fake(x, residual, weight=None, bias=None, gate=None, post_weight=None, post_bias=None, *, norm='rms',
                        post='none', eps=1e-6, residual_scale=1.0, p=0.0, rng=None, stream=0):
    del weight, bias, gate, post_weight, post_bias, norm, post, eps, residual_scale, p, rng, stream
    return residual.new_empty(x.shape), x.new_empty(x.shape)


@torch.library.register_fake('vectra::residual_norm_8bit')
def _residual_norm_8bit_fake(x, residual, weight=None, bias=None, gate=None, post_weight=None, post_bias=None, *,
                             norm='rms', post='none', eps=1e-6, residual_scale=1.0, p=0.0, rng=None, stream=0):
    del weight, bias, gate, post_weight, post_bias, norm, post, eps, residual_scale, p, rng, stream
    return (residual.new_empty(x.shape), x.new_empty(_codes_shape(x.shape), dtype=torch.float8_e4m3fn),
            x.new_empty(_scales_shape(x.shape), dtype=torch.float8_e8m0fnu))


@torch.library.register_fake('vectra::residual_norm_backward')
def _residual_norm_backward_fake(grad_h, grad_n, h, x, residual, weight, bias, gate, post_weight, post_bias, norm, post,
                                 eps, residual_scale, p, rng, stream, dtype, wanted):
    del grad_h, grad_n, x, norm, eps, residual_scale, p, rng, stream
    side = residual if gate is not None or post != 'none' else h
    made = [lambda: side.new_empty(side.shape, dtype=dtype), lambda: side.new_empty(side.shape)]
    made += [lambda t=t: t.new_empty(t.shape) for t in (weight, bias, gate, post_weight, post_bias)]
    return [make() for make, want in zip(made, wanted) if want]


def dropout(x, p, rng, stream=0):
    """x with elements dropped and the others scaled (torch.ops.vectra.dropout)."""
    return torch.ops.vectra.dropout(x, p, rng, stream)


def residual_norm(x, residual, weight=None, bias=None, gate=None, post_weight=None, post_bias=None, **options):
    """The residual stream with a branch, and its norm: (h, n) (torch.ops.vectra.residual_norm)."""
    return torch.ops.vectra.residual_norm(x, residual, weight, bias, gate, post_weight, post_bias, **options)


def residual_norm_8bit(x, residual, weight=None, bias=None, gate=None, post_weight=None, post_bias=None, **options):
    """residual_norm with n in 8-bit rows: (h, codes, scales) (torch.ops.vectra.residual_norm_8bit)."""
    return torch.ops.vectra.residual_norm_8bit(x, residual, weight, bias, gate, post_weight, post_bias, **options)
