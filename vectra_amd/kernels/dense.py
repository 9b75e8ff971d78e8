"""The dense operators of a Transformer block on MI355X: the linear layers
around its attention, forward and backward, in one pass each.

  y = torch.ops.vectra.linear(x, weight, bias=None, residual=None,
                              activation='none', checkpoint='none')
      act(x @ weight.T + bias) + residual
  y = torch.ops.vectra.gated_linear(x, weight, bias=None,
                                    activation='silu', checkpoint='none')
      act(x @ gate.T + b_g) * (x @ up.T + b_u), with weight = cat([gate, up])
      and bias = cat([b_g, b_u])
  codes, scales = torch.ops.vectra.quantize_rows(x)
  x_ = torch.ops.vectra.dequantize_rows(codes, scales, x.dtype)

x [..., width_in] and residual [..., width_out] (float32, float16 or bfloat16,
weight in the same type, any strides; views without unit element stride are
copied), bias in that type or float32.  activation is 'none', 'relu', 'gelu'
(the exact one), 'gelu_tanh' or 'silu'.  Products are accumulated in fp32 and
the result is rounded once.

Under torch.autocast the layers run in autocast's type, as torch's own linear
layers do; a float32 bias stays float32, and a residual of another type is added
to the layer's output by torch's rules (a float32 residual stream stays one).

Both layers have gradients for every tensor argument; the 8-bit rows and
linear_backward have none, and a backward pass through them raises (quantise
x.detach(), or under no_grad, what is kept beside a graph).  Nothing but their inputs
is kept for the backward pass: the pre-activation is computed again.  With
``checkpoint='e4m3'`` the input too is given up: its 8-bit form is kept (33
bytes for 32 elements), and the gradients are those of the layer at the values
that form stands for.  The 8-bit form, see include/vectra_dense.h: each 32
consecutive elements of a row share a power of two, an element is an OCP e4m3
code; codes are float8_e4m3fn [..., width], scales float8_e8m0fnu
[..., ceil(width / 32)].

dz, the gradient before the layer's products, is rounded once to x's type (a
16-bit matrix product reads 16-bit operands); dx = dz @ weight and dW = dz.T @ x
are formed from that in fp32 sums, db = dz.sum(0) from dz before or after that
rounding.  Gradients of gradients and forward-mode derivatives (an argument
that carries a tangent) are refused.

A backward pass may be captured into a HIP graph through
torch.ops.vectra.linear_backward, which autograd calls.  (Capturing
torch.autograd.grad itself while an eager graph over the same leaves is alive
fails in autograd's own stream bookkeeping: drop such graphs, outputs with a
grad_fn, before the capture.)

The schemas, the CUDA-key implementations (libvectra_dense.so on the current
stream), the CPU ones and the autograd rule live in
vectra_amd/csrc/ext/dense_op.cpp.  This module registers the fake (meta)
implementations used while tracing and gives the operators Python names.
"""

import torch

from vectra_amd.kernels import _native

ACTIVATIONS = ('none', 'relu', 'gelu', 'gelu_tanh', 'silu')
CHECKPOINTS = ('none', 'e4m3')
BLOCK = 32  # elements of a row that share a power of two in the 8-bit form

_native.load_torch_extension()


@torch.library.register_fake('vectra::linear')
def _linear_fake(x, weight, bias=None, residual=None, activation='none', checkpoint='none'):
    del bias, residual, activation, checkpoint
    return x.new_empty((*x.shape[:-1], weight.shape[0]))


@torch.library.register_fake('vectra::gated_linear')
def _gated_linear_fake(x, weight, bias=None, activation='silu', checkpoint='none'):
    del bias, activation, checkpoint
    return x.new_empty((*x.shape[:-1], weight.shape[0] // 2))


@torch.library.register_fake('vectra::linear_backward')
def _linear_backward_fake(grad, x, scales, weight, bias, activation, gated, wanted):
    del grad, scales, activation, gated
    made = (
        lambda: weight.new_empty(x.shape),
        lambda: weight.new_empty(weight.shape),
        lambda: (weight if bias is None else bias).new_empty((weight.shape[0],)),
    )
    return [make() for make, want in zip(made, wanted) if want]


@torch.library.register_fake('vectra::quantize_rows')
def _quantize_rows_fake(x):
    blocks = (x.shape[-1] + BLOCK - 1) // BLOCK
    return (x.new_empty(x.shape, dtype=torch.float8_e4m3fn),
            x.new_empty((*x.shape[:-1], blocks), dtype=torch.float8_e8m0fnu))


@torch.library.register_fake('vectra::dequantize_rows')
def _dequantize_rows_fake(codes, scales, dtype):
    del scales
    return codes.new_empty(codes.shape, dtype=dtype)


def linear(x, weight, bias=None, residual=None, activation='none', checkpoint='none'):
    """act(x @ weight.T + bias) + residual (torch.ops.vectra.linear)."""
    return torch.ops.vectra.linear(x, weight, bias, residual, activation, checkpoint)


def gated_linear(x, weight, bias=None, activation='silu', checkpoint='none'):
    """act(x @ gate.T + b_g) * (x @ up.T + b_u) (torch.ops.vectra.gated_linear)."""
    return torch.ops.vectra.gated_linear(x, weight, bias, activation, checkpoint)


def quantize_rows(x):
    """The 8-bit form of x's rows: (codes, scales) (torch.ops.vectra.quantize_rows)."""
    return torch.ops.vectra.quantize_rows(x)


def dequantize_rows(codes, scales, dtype):
    """What codes and scales stand for (torch.ops.vectra.dequantize_rows)."""
    return torch.ops.vectra.dequantize_rows(codes, scales, dtype)
