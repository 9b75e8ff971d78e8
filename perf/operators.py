"""Performance cases of the dense operators around the attention of a Transformer block.

* ``torch.ops.vectra.linear``: act(x @ weight.T + bias) + residual, one pass; with ``checkpoint='e4m3'`` the input is kept in 8 bits
  for the backward pass.
* ``torch.ops.vectra.gated_linear``: act(x @ gate.T + b_g) * (x @ up.T + b_u), ``weight`` holding the gate's rows, then the up
  projection's.
* ``torch.ops.vectra.quantize_rows`` / ``dequantize_rows``: the 8-bit form itself.

A case is a dict: the kind ('linear' and 'gated': a forward call, as serving makes it; 'linear_step' and 'gated_step': a forward and a
backward pass, with the gradients of all inputs; 'codes': rows to 8 bits and back), the sizes, the element type, the activation, whether
there is a bias and a residual, how the input lies ('rows': a tensor of its own; 'view': the middle columns of a wider one, as a split
projection hands it on) and the form in which a step keeps its input ('none': as it is, 'e4m3').  Tensors are resident on the GPU.

8-bit rows: each 32 consecutive elements of a row (the last block may be shorter) share a power of two 2^e, the smallest for which no
finite element exceeds 448 * 2^e in magnitude (e >= -117, for fp16 e >= -15); an element x is kept as x / 2^e rounded to e4m3 (ties to
even).
"""

import math

import numpy as np
import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
BLOCK = 32
CODE_MAX = 448.0
LOWEST_EXPONENT = {'bf16': -117, 'fp16': -15, 'fp32': -117}
STEPS = ('linear_step', 'gated_step')
GATED = ('gated', 'gated_step')


def _case(name, kind, rows, width_in, width_out, dtype, activation='none', bias=True, residual=False, layout='rows', checkpoint='none'):
    case = {'kind': kind, 'rows': rows, 'width_in': width_in, 'width_out': width_out, 'dtype': dtype, 'activation': activation,
            'bias': bias, 'residual': residual, 'layout': layout, 'checkpoint': checkpoint}
    return {'name': name, **case} if name else case


def listed():
    return [
        # The qkv projection of one price request: a subject and its 64 comparables at the price model's widths.  Launch latency.
        _case('qkv of one request', 'linear', 65, 128, 384, 'bf16'),
        # The candidate encoder's first layer over a full serving batch (1,024 requests of 64 comparables): odd rows, fp32.
        _case('candidate encoder', 'linear', 65536, 141, 256, 'fp32', 'gelu'),
        # The second projection of the price model's feed-forward block at the serving batch, onto the residual stream.
        _case('block output', 'linear', 66560, 256, 128, 'bf16', residual=True),
        # One token through a square projection of a wide model: the weight's bytes.
        _case('one row', 'linear', 1, 4096, 4096, 'fp16', residual=True),
        # Training: the first projection of the price model's feed-forward block, and its gradients.
        _case('block training', 'linear_step', 66560, 128, 256, 'bf16', 'gelu'),
        # Training: an output projection of a wide model onto the residual stream.
        _case('wide training', 'linear_step', 8192, 4096, 4096, 'bf16', residual=True),
        # A few tokens in flight through a gated feed-forward block's projections: the weights' bytes.
        _case('gated, a few rows', 'gated', 4, 4096, 11008, 'bf16', 'silu', bias=False),
        # A ragged prompt through a gated block.
        _case('gated, a prompt', 'gated', 2051, 2048, 5632, 'fp16', 'gelu_tanh', layout='view'),
        # Training: a gated block at the price model's widths.
        _case('gated block training', 'gated_step', 66560, 128, 256, 'bf16', 'silu'),
        # Training: a gated block of a wide model.
        _case('gated wide training', 'gated_step', 4096, 4096, 8192, 'bf16', 'silu', bias=False),
        # The block's hidden rows of a training batch to 8 bits and back.
        _case('rows to 8 bits', 'codes', 66560, 256, 0, 'bf16', bias=False),
        # Training with the input kept in 8 bits: a gated block at widths that fill no tile.
        _case('gated training from 8 bits', 'gated_step', 10007, 1000, 2730, 'bf16', 'silu', checkpoint='e4m3'),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    most = {k: max(work(c)[k] for c in listed()) for k in ('bytes', 'flops')}
    while True:
        kind = rng.choice(['linear', 'linear', 'linear_step', 'linear_step', 'gated', 'gated_step', 'gated_step', 'codes'])
        rows, width_in = _log_uniform(rng, 1, 131072), _log_uniform(rng, 16, 8192)
        width_out = _log_uniform(rng, 16, 12288)
        if rng.random() < 0.5:  # model widths: multiples of 16
            width_in, width_out = -(-width_in // 16) * 16, -(-width_out // 16) * 16
        activation = rng.choice(['silu', 'gelu', 'gelu_tanh'] + ([] if kind in GATED else ['none', 'none', 'relu']))
        case = _case('', kind, rows, width_in, width_out, rng.choice(['bf16', 'bf16', 'fp16', 'fp32']), activation, rng.random() < 0.7,
                     kind in ('linear', 'linear_step') and rng.random() < 0.5, rng.choice(['rows', 'rows', 'view']),
                     rng.choice(['none', 'e4m3']) if kind in STEPS else 'none')
        if kind == 'codes':
            case.update(width_out=0, activation='none', bias=False)
        w = work(case)
        if w['bytes'] <= most['bytes'] and w['flops'] <= most['flops']:
            return case


def work(case):
    m, k, n = case['rows'], case['width_in'], case['width_out']
    size = 4 if case['dtype'] == 'fp32' else 2
    if case['kind'] == 'codes':
        return {'bytes': 2 * m * k * size, 'flops': 3 * m * k}
    n_w = 2 * n if case['kind'] in GATED else n
    values = m * k + n_w * k + n_w * case['bias'] + m * n * (1 + case['residual'])
    flops = 2 * m * n_w * k
    if case['kind'] in STEPS:  # dy in, and a gradient for x, the weight and the bias (the residual's is dy)
        values += m * n + m * k + n_w * k + n_w * case['bias']
        flops *= 3
    return {'bytes': values * size, 'flops': flops}


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    dtype = DTYPES[case['dtype']]
    m, k, n = case['rows'], case['width_in'], case['width_out']
    n_w = 2 * n if case['kind'] in GATED else n
    step = case['kind'] in STEPS

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device='cuda').mul_(scale).to(dtype)

    # Normalised rows, a few of their features large, as a Transformer's hidden rows are.
    width = k if case['layout'] == 'rows' else k + 2 * (-(-k // 16) * 8)
    x = torch.randn(m, width, generator=gen, device='cuda')
    x.mul_(1.0 + 7.0 * (torch.rand(width, generator=gen, device='cuda') < 0.01))
    x = x.to(dtype)
    if case['layout'] == 'view':
        x = x[:, (width - k) // 2:(width - k) // 2 + k]
    state = {'case': dict(case), 'x': x}
    if case['kind'] == 'codes':
        return state
    state['weight'] = normal(n_w, k, scale=k ** -0.5)
    state['bias'] = normal(n_w, scale=0.1) if case['bias'] else None
    state['residual'] = normal(m, n) if case['residual'] else None
    if step:
        state['grad'] = normal(m, n, scale=0.05)
        for name in ('x', 'weight', 'bias', 'residual'):
            if state[name] is not None:
                state[name].requires_grad_()
    return state


# ------------------------------------------------------------------ plain form


def _activation(z, name):
    """The activation of z and its derivative."""
    if name == 'none':
        return z, torch.ones_like(z)
    if name == 'relu':
        return z.clamp_min(0.0), (z > 0).to(z.dtype)
    if name == 'silu':
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    if name == 'gelu':
        cdf = 0.5 * torch.erfc(z * -math.sqrt(0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    c = math.sqrt(2.0 / math.pi)  # gelu_tanh
    s = 1.0 / (1.0 + torch.exp(-2.0 * c * (z + 0.044715 * z * z * z)))
    return z * s, s + z * s * (1.0 - s) * 2.0 * c * (1.0 + 3.0 * 0.044715 * z * z)


def _eight_bit_rows(x, dtype):
    """What the 8-bit form of x stands for, in x's type."""
    rows, width = x.shape
    padded = torch.nn.functional.pad(x.float(), (0, -width % BLOCK)).reshape(rows, -1, BLOCK)
    mantissa, exponent = torch.frexp(padded.abs().amax(-1, keepdim=True))  # largest = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = exponent - 9 + (mantissa > CODE_MAX / 512).to(torch.int32)  # 448 * 2^e >= largest
    e = torch.where(mantissa > 0, e, LOWEST_EXPONENT[dtype]).clamp_min(LOWEST_EXPONENT[dtype])
    y = torch.ldexp(padded, -e)
    _, place = torch.frexp(y)
    step = place.clamp_min(-5) - 4  # three bits after the leading one; subnormals below 2^-6
    y = torch.ldexp(torch.round(torch.ldexp(y, -step)), step)
    return torch.ldexp(y, e).reshape(rows, -1)[:, :width].to(x.dtype)


def _plain(state):
    case, x = state['case'], state['x']
    if case['kind'] == 'codes':
        return _eight_bit_rows(x, case['dtype'])
    weight, bias = state['weight'], state['bias']
    w, dtype, n = weight.float(), x.dtype, case['width_out']
    gated = case['kind'] in GATED

    def before(rows):
        z = rows.float() @ w.t()
        return z if bias is None else z + bias.float()

    z = before(x)
    a, slope = _activation(z[:, :n], case['activation'])
    y = a * z[:, n:] if gated else a
    if state['residual'] is not None:
        y = y + state['residual'].float()
    y = y.to(dtype)
    if case['kind'] not in STEPS:
        return y
    if case['checkpoint'] == 'e4m3':
        x = _eight_bit_rows(x, case['dtype'])
        z = before(x)
        a, slope = _activation(z[:, :n], case['activation'])
    grad = state['grad'].float()
    dz = torch.cat([grad * z[:, n:] * slope, grad * a], dim=1) if gated else grad * slope
    out = {'y': y, 'x': (dz @ w).to(dtype), 'weight': (dz.t() @ x.float()).to(dtype)}
    if bias is not None:
        out['bias'] = dz.sum(0).to(dtype)
    if state['residual'] is not None:
        out['residual'] = state['grad']
    return out


# ---------------------------------------------------------- the framework's own


def _own(state):
    import vectra_amd.kernels  # noqa: F401  (registers the operators)

    case, x = state['case'], state['x']
    if case['kind'] == 'codes':
        codes, scales = torch.ops.vectra.quantize_rows(x)
        return torch.ops.vectra.dequantize_rows(codes, scales, x.dtype)
    weight, bias, residual = state['weight'], state['bias'], state['residual']
    if case['kind'] in GATED:
        y = torch.ops.vectra.gated_linear(x, weight, bias, case['activation'], case['checkpoint'])
    else:
        y = torch.ops.vectra.linear(x, weight, bias, residual, case['activation'], case['checkpoint'])
    if case['kind'] not in STEPS:
        return y
    leaves = {'x': x, 'weight': weight, 'bias': bias, 'residual': residual}
    leaves = {name: leaf for name, leaf in leaves.items() if leaf is not None}
    gradients = torch.autograd.grad(y, tuple(leaves.values()), state['grad'])
    return {'y': y, **dict(zip(leaves, gradients))}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


# ---------------------------------------------------------------------- 64 bits


def _eight_bit_exact(x, lowest):
    """The 8-bit form from the table of e4m3's values, in numpy."""
    x = x.detach().double().cpu().numpy()
    rows, width = x.shape
    blocks = np.pad(x, ((0, 0), (0, -width % BLOCK))).reshape(rows, -1, BLOCK)
    largest = np.abs(blocks).max(-1, keepdims=True)
    e = np.full(largest.shape, lowest)
    with np.errstate(divide='ignore'):
        guess = np.ceil(np.log2(largest / CODE_MAX))
    for near in (-1, 0, 1):  # the smallest of three that fits (the logarithm may be off by a rounding)
        candidate = np.where(largest > 0, guess - near, lowest).astype(np.int64)
        e = np.where(np.ldexp(CODE_MAX, candidate) >= largest, np.maximum(candidate, lowest), e)
    table = np.array([m * 2.0 ** -9 if p == 0 else (8 + m) * 2.0 ** (p - 10) for p in range(16) for m in range(8)][:127])
    y = np.abs(np.ldexp(blocks, -e))
    above = np.clip(np.searchsorted(table, y), 0, 126)
    below = np.maximum(above - 1, 0)
    to_above, to_below = table[above] - y, y - table[below]
    code = np.where((to_above < to_below) | ((to_above == to_below) & (above % 2 == 0)), above, below)
    return torch.from_numpy((np.copysign(np.ldexp(table[code], e), blocks)).reshape(rows, -1)[:, :width].copy()).cuda()


def exact(case, seed):
    functional = torch.nn.functional
    state = prepare(case, seed)
    if case['kind'] == 'codes':
        return _eight_bit_exact(state['x'], LOWEST_EXPONENT[case['dtype']])
    rows, weight, bias = (None if t is None else t.detach().double() for t in (state['x'], state['weight'], state['bias']))
    act = {'none': lambda t: t, 'relu': torch.relu, 'silu': functional.silu, 'gelu': functional.gelu,
           'gelu_tanh': lambda t: functional.gelu(t, approximate='tanh')}[case['activation']]

    def block(rows, weight, bias):
        z = functional.linear(rows, weight, bias)
        if case['kind'] in GATED:
            gate, up = z.chunk(2, dim=-1)
            return act(gate) * up
        return act(z)

    with torch.no_grad():
        y = block(rows, weight, bias)
        if state['residual'] is not None:
            y = y + state['residual'].detach().double()
    if case['kind'] not in STEPS:
        return y
    if case['checkpoint'] == 'e4m3':
        rows = _eight_bit_exact(state['x'], LOWEST_EXPONENT[case['dtype']])
    leaves = {name: t.requires_grad_() for name, t in (('x', rows), ('weight', weight), ('bias', bias)) if t is not None}
    grad = state['grad'].double()
    out = dict(zip(leaves, torch.autograd.grad(block(rows, weight, bias), tuple(leaves.values()), grad)))
    out['y'] = y
    if state['residual'] is not None:
        out['residual'] = grad
    return out
