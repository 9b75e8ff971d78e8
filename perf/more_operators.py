"""Performance cases of what stands between the dense operators of a Transformer block, and of the dense operators in 8 bits.

* ``torch.ops.vectra.dropout``: kept elements are scaled, the others zero; which ones, a counter-based generator says, here and again in
  the backward pass.
* ``torch.ops.vectra.residual_norm``: a branch's output onto the residual stream, and the stream normalised for the next branch, in one
  pass: h = residual_scale * r + gate * dropout(post_norm(x)), n = norm(h).
* ``torch.ops.vectra.linear_8bit``, ``gated_linear_8bit``: the dense operators on e4m3 codes.  The weight's 128 x 128 tiles and the
  input's rows of 128 share a power of two each; the input is brought into 8 bits within the call.
* ``torch.ops.vectra.residual_norm_8bit``: as ``residual_norm``, n in 8 bits for the product behind it.

A case is a dict: the kind ('dropout': a forward and a backward pass; 'norm': the forward call, as serving makes it; 'norm_step': a forward
and a backward pass, with the gradients of all inputs; 'product', 'gated_product': a layer in 8 bits; 'norm_product': the stream and the
next layer, the rows between them in 8 bits), the sizes ([batch, rows, width] inputs; a product's width_out), the element type, the
residual stream's type ('same' or 'fp32', the norms' weights likewise), which norms there are, the gate's form, the probability p of
dropping an element, and how the input lies ('rows': a tensor of its own; 'view': the middle columns of a wider one, as a split projection
hands it on).  Tensors are resident on the GPU.

The generator: Philox 4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: Parallel random numbers, as easy as 1, 2, 3; SC 2011), key: the
64-bit seed, counter: (group, group >> 32, stream, offset), one draw for each group of eight elements of a row, 16 bits for each.  An
element is kept where its 16 bits are at least t = round(65536 p), and scaled by 65536 / (65536 - t).

The 8-bit form: elements that share a power of two 2^e have the smallest e >= -117 for which none exceeds 448 * 2^e in magnitude; an
element x is kept as x / 2^e rounded to e4m3 (ties to even).  Codes are padded with zeros to whole blocks of 128, a row of scales to a
multiple of four.
"""

import functools
import math

import numpy as np
import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
BLOCK = 128
CODE_MAX = 448.0
LOWEST_EXPONENT = -117
EPS = 1e-6
STREAM = 3  # the dropout's own number in the program
LEAVES = ('x', 'residual', 'weight', 'bias', 'gate', 'post_weight', 'post_bias')


def _norm_case(name, kind, batch, rows, width, dtype, *, stream='same', norm='rms', post='none', gate='none', p=0.0, scale=1.0,
               layout='rows', width_out=0):
    case = {'kind': kind, 'batch': batch, 'rows': rows, 'width': width, 'dtype': dtype, 'stream': stream, 'norm': norm, 'post': post,
            'gate': gate, 'p': p, 'residual_scale': scale, 'layout': layout, 'width_out': width_out}
    return {'name': name, **case} if name else case


def _dropout_case(name, batch, rows, width, dtype, p, layout='rows'):
    case = {'kind': 'dropout', 'batch': batch, 'rows': rows, 'width': width, 'dtype': dtype, 'p': p, 'layout': layout}
    return {'name': name, **case} if name else case


def _product_case(name, kind, batch, rows, width, width_out, dtype, activation='none', bias=True, residual=False, layout='rows'):
    case = {'kind': kind, 'batch': batch, 'rows': rows, 'width': width, 'width_out': width_out, 'dtype': dtype, 'activation': activation,
            'bias': bias, 'residual': residual, 'layout': layout}
    return {'name': name, **case} if name else case


def listed():
    return [
        # Dropout behind the activation of the price model's feed-forward block, a full training batch (1,024 requests of 65 tokens).
        _dropout_case('dropout of a batch', 1024, 65, 256, 'bf16', 0.1),
        # Dropout of an fp32 encoder's features: rows of an odd width, not aligned.
        _dropout_case('dropout, odd rows', 10007, 1, 141, 'fp32', 0.3),
        # One token: the residual stream of a wide model between two branches.  Launch latency.
        _norm_case('one token', 'norm', 1, 1, 4096, 'bf16'),
        # Training the price model: a branch with dropout onto the stream, and the LayerNorm of the next.
        _norm_case('block norm training', 'norm_step', 1024, 65, 128, 'bf16', norm='layer', p=0.1),
        # Training a wide model: norms before and after the branch, a learned gate per channel, an fp32 residual stream.
        _norm_case('wide norm training', 'norm_step', 4, 2048, 4096, 'bf16', stream='fp32', post='rms', gate='vector'),
        # Training a model conditioned by sequence: a gate for each sequence, LayerNorm, a ragged number of tokens, fp16.
        _norm_case('conditioned training', 'norm_step', 16, 1025, 1152, 'fp16', norm='layer', gate='sequence', layout='view'),
        # One token through a gated feed-forward block's projections in 8 bits: the weights' bytes.
        _product_case('gated 8-bit, one token', 'gated_product', 1, 1, 4096, 11008, 'bf16', 'silu', bias=False),
        # A batch of tokens being decoded, through an output projection in 8 bits.
        _product_case('8-bit, a decoding batch', 'product', 48, 1, 4096, 4096, 'fp16', residual=True),
        # A ragged prompt through a gated block in 8 bits.
        _product_case('gated 8-bit, a prompt', 'gated_product', 1, 2051, 2048, 5632, 'bf16', 'silu', layout='view'),
        # A long prompt through the first projection of a wide block in 8 bits.
        _product_case('8-bit, a long prompt', 'product', 1, 8192, 4096, 16384, 'bf16', 'gelu'),
        # Widths that fill no block and no tile, fp32 activations.
        _product_case('8-bit, odd widths', 'product', 3, 173, 1000, 2730, 'fp32', 'gelu_tanh'),
        # A prompt between two layers: the branch onto the stream, its norm, and the next projection in 8 bits.
        _norm_case('norm into 8 bits', 'norm_product', 2, 2048, 4096, 'bf16', width_out=4096),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    most = {k: max(work(c)[k] for c in listed()) for k in ('bytes', 'flops')}
    while True:
        kind = rng.choice(['dropout', 'norm', 'norm', 'norm_step', 'norm_step', 'norm_step', 'product', 'product', 'gated_product',
                           'norm_product'])
        batch, rows = _log_uniform(rng, 1, 1024), _log_uniform(rng, 1, 8192)
        width, width_out = _log_uniform(rng, 16, 8192), _log_uniform(rng, 16, 16384)
        if rng.random() < 0.6:  # model widths: multiples of 16
            width, width_out = -(-width // 16) * 16, -(-width_out // 16) * 16
        dtype, layout = rng.choice(['bf16', 'bf16', 'fp16', 'fp32']), rng.choice(['rows', 'rows', 'view'])
        p = rng.choice([0.0, 0.0, 0.1, rng.uniform(0.01, 0.9)])
        if kind == 'dropout':
            case = _dropout_case('', batch, rows, width, dtype, p or 0.1, layout)
        elif kind in ('product', 'gated_product'):
            gated = kind == 'gated_product'
            activation = rng.choice(['silu', 'gelu', 'gelu_tanh'] + ([] if gated else ['none', 'none', 'relu']))
            case = _product_case('', kind, batch, rows, width, width_out, dtype, activation, rng.random() < 0.6,
                                 not gated and rng.random() < 0.5, layout)
        else:
            case = _norm_case('', kind, batch, rows, width, dtype, stream=rng.choice(['same', 'same', 'fp32']),
                              norm=rng.choice(['rms', 'layer']), post=rng.choice(['none', 'none', 'rms', 'layer']),
                              gate=rng.choice(['none', 'none', 'vector', 'sequence', 'full']), p=p if kind == 'norm_step' else 0.0,
                              scale=rng.choice([1.0, 1.0, 0.5, 2.0]), layout=layout,
                              width_out=width_out if kind == 'norm_product' else 0)
        w = work(case)
        if w['bytes'] <= most['bytes'] and w['flops'] <= most['flops']:
            return case


def _sizes(case):
    """Bytes of an element, of an element of the residual stream."""
    size = 4 if case['dtype'] == 'fp32' else 2
    return size, 4 if case.get('stream') == 'fp32' else size


def work(case):
    m, d = case['batch'] * case['rows'], case['width']
    size, wide = _sizes(case)
    if case['kind'] == 'dropout':  # x and dy in, y and dx out
        return {'bytes': 4 * m * d * size, 'flops': 2 * m * d}
    n = case['width_out']
    if case['kind'] in ('product', 'gated_product'):
        n_w = 2 * n if case['kind'] == 'gated_product' else n
        values = m * d + n_w * case['bias'] + m * n * (1 + case['residual'])
        return {'bytes': values * size + n_w * d + -(-n_w // BLOCK) * -(-d // BLOCK), 'flops': 2 * m * n_w * d}
    gate = {'none': 0, 'vector': d, 'sequence': case['batch'] * d, 'full': m * d}[case['gate']]
    small = (gate + d * ((1 + (case['norm'] == 'layer')) + {'none': 0, 'rms': 1, 'layer': 2}[case['post']])) * wide
    if case['kind'] == 'norm':
        return {'bytes': 2 * m * d * (size + wide) + small, 'flops': 16 * m * d}
    if case['kind'] == 'norm_step':  # x, r and the gradients of h and n in; h, n and the gradients of x and r out
        return {'bytes': 4 * m * d * (size + wide) + 2 * small, 'flops': 48 * m * d}
    return {'bytes': m * d * (size + 2 * wide) + small + n * d + -(-n // BLOCK) * -(-d // BLOCK) + m * n * size,
            'flops': 2 * m * n * d + 16 * m * d}


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    dtype = DTYPES[case['dtype']]
    wide = torch.float32 if case.get('stream') == 'fp32' else dtype
    shape, d = (case['batch'], case['rows'], case['width']), case['width']

    def normal(*sizes, scale=1.0, offset=0.0, to=dtype):
        return torch.randn(*sizes, generator=gen, device='cuda').mul_(scale).add_(offset).to(to)

    def rows(scale, to):
        """Hidden rows, a few of their features large."""
        width = d if case['layout'] == 'rows' else d + 2 * (-(-d // 16) * 8)
        x = torch.randn(*shape[:2], width, generator=gen, device='cuda').mul_(scale)
        x = x.mul_(1.0 + 7.0 * (torch.rand(width, generator=gen, device='cuda') < 0.01)).to(to)
        return x if case['layout'] == 'rows' else x[..., (width - d) // 2:(width - d) // 2 + d]

    state = {'case': dict(case), 'x': rows(1.0, dtype)}
    step = case['kind'] in ('dropout', 'norm_step')
    if case.get('p'):
        state['rng'] = torch.randint(1 << 62, (2,), generator=gen, device='cuda')  # the seed, the step's number
    if case['kind'] == 'dropout':
        state['grad'] = normal(*shape)
        state['x'].requires_grad_()
        return state
    if 'norm' in case['kind']:
        state['residual'] = normal(*shape, scale=2.0, to=wide)
        state['weight'] = normal(d, scale=0.1, offset=1.0, to=wide)
        state['bias'] = normal(d, scale=0.1, to=wide) if case['norm'] == 'layer' else None
        state['post_weight'] = normal(d, scale=0.1, offset=0.5, to=wide) if case['post'] != 'none' else None
        state['post_bias'] = normal(d, scale=0.1, to=wide) if case['post'] == 'layer' else None
        gate = {'none': None, 'vector': (d,), 'sequence': (case['batch'], 1, d), 'full': shape}[case['gate']]
        state['gate'] = None if gate is None else normal(*gate, scale=0.5, offset=0.2, to=wide)
        if step:
            state['grad_h'], state['grad_n'] = normal(*shape, scale=0.1, to=wide), normal(*shape, scale=0.1)
            for name in LEAVES:
                if state[name] is not None:
                    state[name].requires_grad_()
    if 'product' in case['kind']:
        n = case['width_out']
        n_w = 2 * n if case['kind'] == 'gated_product' else n
        weight = torch.randn(n_w, d, generator=gen, device='cuda').mul_(d ** -0.5)
        state['codes'], state['scales'] = _eight_bit(weight, BLOCK)
        state['layer_bias'] = normal(n_w, scale=0.1) if case.get('bias') else None
        state['layer_residual'] = normal(*shape[:2], n) if case.get('residual') else None
    return state


# ------------------------------------------------------------------ the 8-bit form


def _eight_bit(x, high):
    """Codes and scales of an fp32 matrix whose blocks of `high` rows of 128 share a power of two."""
    rows, width = x.shape
    padded = torch.nn.functional.pad(x, (0, -width % BLOCK, 0, -rows % high))
    blocks = padded.reshape(padded.shape[0] // high, high, -1, BLOCK)
    mantissa, exponent = torch.frexp(blocks.abs().amax((1, 3)))  # the largest = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = exponent - 9 + (mantissa > CODE_MAX / 512).to(torch.int32)  # 448 * 2^e >= the largest
    e = torch.where(mantissa > 0, e, LOWEST_EXPONENT).clamp_min(LOWEST_EXPONENT)
    codes = torch.ldexp(blocks, -e[:, None, :, None]).reshape(padded.shape)[:rows].to(torch.float8_e4m3fn)
    scales = torch.zeros(e.shape[0], -(-e.shape[1] // 4) * 4, dtype=torch.uint8, device=x.device)
    scales[:, :e.shape[1]] = (e + 127).to(torch.uint8)
    return codes, scales.view(torch.float8_e8m0fnu)


def _values(codes, scales, high, width):
    """What codes and scales stand for, in fp32."""
    e = scales.view(torch.uint8).to(torch.int32)[:, :codes.shape[1] // BLOCK] - 127
    e = e.repeat_interleave(high, 0)[:codes.shape[0]].repeat_interleave(BLOCK, 1)
    return torch.ldexp(codes.float(), e)[:, :width]


# ------------------------------------------------------------------ plain form


def _philox_round(state, _):
    (a, b, c, d), (k0, k1) = state
    low, high = 0xD2511F53 * a, 0xCD9E8D57 * c  # (64-bit integers wrap)
    mask = 0xFFFFFFFF
    counter = ((high >> 32 & mask) ^ b ^ k0, high & mask, (low >> 32 & mask) ^ d ^ k1, low & mask)
    return counter, (k0 + 0x9E3779B9 & mask, k1 + 0xBB67AE85 & mask)


def _kept(state):
    """The factor of every element: 0 or 65536 / (65536 - t)."""
    case, rng = state['case'], state['rng']
    rows, width = case['batch'] * case['rows'], case['width']
    groups = -(-width // 8)
    at = torch.arange(rows * groups, device=rng.device)
    mask = 0xFFFFFFFF
    counter = (at & mask, at >> 32, torch.full_like(at, STREAM), torch.ones_like(at) * (rng[1] & mask))
    words, _ = functools.reduce(_philox_round, range(10), (counter, (rng[0] & mask, rng[0] >> 32 & mask)))
    words = torch.stack(words, -1)
    bits = torch.stack([words & 0xFFFF, words >> 16], -1).reshape(rows, groups * 8)[:, :width]
    t = round(65536 * case['p'])
    return torch.where(bits >= t, 65536.0 / (65536 - t), 0.0).float().reshape(case['batch'], case['rows'], width)


def _normalised(x, kind):
    """(x - mean) / deviation and 1 / deviation."""
    x = x - x.mean(-1, keepdim=True) if kind == 'layer' else x
    r = ((x * x).mean(-1, keepdim=True) + EPS) ** -0.5
    return x * r, r


def _affine(x, weight, bias):
    x = x * weight
    return x if bias is None else x + bias


def _norm_gradient(g, hat, r, weight, kind):
    g = g * weight
    g_hat = g - hat * (g * hat).mean(-1, keepdim=True)
    return (g_hat - g.mean(-1, keepdim=True) if kind == 'layer' else g_hat) * r


def _stream(state, at_least):
    """The forward pass in at least that type: all that the backward pass needs of it."""
    case = state['case']
    x, residual, weight, bias, gate, post_weight, post_bias = (None if state[k] is None else state[k].to(at_least) for k in LEAVES)
    kept = _kept(state).to(at_least) if case['p'] else None
    post_hat = post_r = None
    u = x
    if case['post'] != 'none':
        post_hat, post_r = _normalised(x, case['post'])
        u = _affine(post_hat, post_weight, post_bias)
    v = u if kept is None else u * kept
    h = case['residual_scale'] * residual + (v if gate is None else gate * v)
    hat, r = _normalised(h, case['norm'])
    return h, _affine(hat, weight, bias), (weight, gate, post_weight, kept, post_hat, post_r, v, hat, r)


def _norm_plain(state):
    case = state['case']
    h, n, (weight, gate, post_weight, kept, post_hat, post_r, v, hat, r) = _stream(state, torch.float32)
    to = {k: state[k].dtype for k in LEAVES if state[k] is not None}
    out = {'h': h.to(to['residual']), 'n': n.to(to['x'])}
    if case['kind'] == 'norm':
        return out
    g_n = state['grad_n'].float()
    g_h = state['grad_h'].float() + _norm_gradient(g_n, hat, r, weight, case['norm'])
    out['d_weight'] = (g_n * hat).sum((0, 1))
    out['d_bias'] = g_n.sum((0, 1))
    out['d_residual'] = case['residual_scale'] * g_h
    g_v = g_h
    if gate is not None:
        out['d_gate'] = (g_h * v).sum_to_size(gate.shape)
        g_v = g_h * gate
    g_u = g_v if kept is None else g_v * kept
    out['d_x'] = g_u
    if case['post'] != 'none':
        out['d_post_weight'] = (g_u * post_hat).sum((0, 1))
        out['d_post_bias'] = g_u.sum((0, 1))
        out['d_x'] = _norm_gradient(g_u, post_hat, post_r, post_weight, case['post'])
    return {k: v.to(to.get(k[2:], v.dtype)) for k, v in out.items() if not k.startswith('d_') or k[2:] in to}


def _activation(z, name):
    if name == 'none':
        return z
    if name == 'relu':
        return z.clamp_min(0.0)
    if name == 'silu':
        return z / (1.0 + torch.exp(-z))
    if name == 'gelu':
        return z * 0.5 * torch.erfc(z * -math.sqrt(0.5))
    return z / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))  # gelu_tanh


def _layer_plain(state, rows):
    """The layer on fp32 rows, brought into 8 bits first."""
    case = state['case']
    codes, scales = _eight_bit(rows.reshape(-1, rows.shape[-1]), 1)
    x = _values(codes, scales, 1, rows.shape[-1])
    z = x @ _values(state['codes'], state['scales'], BLOCK, rows.shape[-1]).t()
    z = z.reshape(*rows.shape[:-1], -1)
    if state['layer_bias'] is not None:
        z = z + state['layer_bias'].float()
    activation, n = case.get('activation', 'none'), case['width_out']
    y = _activation(z[..., :n], activation)
    if case['kind'] == 'gated_product':
        y = y * z[..., n:]
    if state['layer_residual'] is not None:
        y = y + state['layer_residual'].float()
    return y.to(state['x'].dtype)


def _plain(state):
    case = state['case']
    if case['kind'] == 'dropout':
        kept = _kept(state)
        return {'y': (state['x'].float() * kept).to(state['x'].dtype), 'd_x': (state['grad'].float() * kept).to(state['x'].dtype)}
    if case['kind'] in ('norm', 'norm_step'):
        return _norm_plain(state)
    if case['kind'] == 'norm_product':
        h, n, _ = _stream(state, torch.float64)  # (n is rounded to few bits: what lies next to a border goes by 64)
        return {'h': h.to(state['residual'].dtype), 'y': _layer_plain(state, n.float())}
    return _layer_plain(state, state['x'].float())


# ---------------------------------------------------------- the framework's own


def _own(state):
    import vectra_amd.kernels  # noqa: F401  (registers the operators)

    ops, case, x = torch.ops.vectra, state['case'], state['x']
    if case['kind'] == 'dropout':
        y = ops.dropout(x, case['p'], state['rng'], STREAM)
        return {'y': y, 'd_x': torch.autograd.grad(y, x, state['grad'])[0]}
    if case['kind'] == 'product':
        return ops.linear_8bit(x, state['codes'], state['scales'], state['layer_bias'], state['layer_residual'], case['activation'])
    if case['kind'] == 'gated_product':
        return ops.gated_linear_8bit(x, state['codes'], state['scales'], state['layer_bias'], case['activation'])
    stream = ops.residual_norm_8bit if case['kind'] == 'norm_product' else ops.residual_norm
    h, *n = stream(*(state[k] for k in LEAVES), norm=case['norm'], post=case['post'], eps=EPS, residual_scale=case['residual_scale'],
                   p=case['p'], rng=state.get('rng'), stream=STREAM)
    if case['kind'] == 'norm_product':
        codes, scales = n
        return {'h': h, 'y': ops.linear_8bit(codes, state['codes'], state['scales'], scales=scales, dtype=x.dtype)}
    out = {'h': h, 'n': n[0]}
    if case['kind'] == 'norm_step':
        leaves = {k: state[k] for k in LEAVES if state[k] is not None}
        gradients = torch.autograd.grad((h, n[0]), tuple(leaves.values()), (state['grad_h'], state['grad_n']))
        out.update({'d_' + k: g for k, g in zip(leaves, gradients)})
    return out


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


# ---------------------------------------------------------------------- 64 bits


def _kept_exact(case, rng):
    """The factors of the elements, by 64-bit unsigned integers in numpy."""
    seed, step = (int(v) for v in rng.tolist())
    low = np.uint64(0xFFFFFFFF)
    shift = np.uint64(32)
    rows, width = case['batch'] * case['rows'], case['width']
    groups = -(-width // 8)
    at = np.arange(rows * groups, dtype=np.uint64)
    x = [at & low, at >> shift, np.full_like(at, STREAM), np.full_like(at, step & 0xFFFFFFFF)]
    key = [seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF]
    for _ in range(10):
        p, q = np.uint64(0xD2511F53) * x[0], np.uint64(0xCD9E8D57) * x[2]
        x = [(q >> shift) ^ x[1] ^ np.uint64(key[0]), q & low, (p >> shift) ^ x[3] ^ np.uint64(key[1]), p & low]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    bits = np.empty((rows * groups, 8), np.int64)
    for word in range(4):
        bits[:, 2 * word] = x[word] & np.uint64(0xFFFF)
        bits[:, 2 * word + 1] = x[word] >> np.uint64(16)
    t = round(65536 * case['p'])
    kept = np.where(bits.reshape(rows, -1)[:, :width] < t, 0.0, 65536.0 / (65536 - t))
    return torch.from_numpy(kept.reshape(case['batch'], case['rows'], width)).cuda()


def _rows_exact(x):
    """What the 8-bit form of 64-bit rows stands for, from the table of e4m3's values."""
    table = torch.tensor([m * 2.0 ** -9 if p == 0 else (8 + m) * 2.0 ** (p - 10) for p in range(16) for m in range(8)][:127],
                         dtype=torch.float64, device='cuda')
    rows, width = x.shape
    out = torch.empty_like(x)
    for first in range(0, width, BLOCK):
        block = x[:, first:first + BLOCK]
        largest = block.abs().amax(1, keepdim=True)
        e = torch.full_like(largest, LOWEST_EXPONENT)
        guess = torch.ceil(torch.log2(largest / CODE_MAX))
        for near in (1, 0, -1):  # the smallest of three that fits (the logarithm may be off by a rounding)
            fits = (largest > 0) & (CODE_MAX * torch.exp2(guess + near) >= largest) & (guess + near >= LOWEST_EXPONENT)
            e = torch.where(fits, guess + near, e)
        y = block.abs() / torch.exp2(e)
        above = torch.searchsorted(table, y.contiguous()).clamp_max(126)
        below = (above - 1).clamp_min(0)
        to_above, to_below = table[above] - y, y - table[below]
        code = torch.where((to_above < to_below) | ((to_above == to_below) & (above % 2 == 0)), above, below)
        out[:, first:first + BLOCK] = torch.copysign(table[code] * torch.exp2(e), block)
    return out


def exact(case, seed):
    functional = torch.nn.functional
    state = prepare(case, seed)
    kept = _kept_exact(case, state['rng']) if case.get('p') else 1.0
    if case['kind'] == 'dropout':
        return {'y': state['x'].detach().double() * kept, 'd_x': state['grad'].double() * kept}
    d = case['width']
    out, rows = {}, state['x'].detach().double()
    if 'norm' in case['kind']:
        leaves = {k: state[k].detach().double().requires_grad_() for k in LEAVES if state[k] is not None}

        def norm(x, kind, weight, bias):
            if kind == 'layer':
                return functional.layer_norm(x, (d,), weight, bias, EPS)
            x = x / torch.sqrt(torch.mean(torch.square(x), -1, keepdim=True) + EPS) * weight
            return x if bias is None else x + bias

        u = leaves['x']
        if case['post'] != 'none':
            u = norm(u, case['post'], leaves['post_weight'], leaves.get('post_bias'))
        h = leaves['residual'] * case['residual_scale'] + u * kept * leaves.get('gate', 1.0)
        n = norm(h, case['norm'], leaves['weight'], leaves.get('bias'))
        out = {'h': h.detach()}
        if case['kind'] == 'norm_product':
            rows = n.detach()
        else:
            out['n'] = n.detach()
        if case['kind'] == 'norm_step':
            gradients = torch.autograd.grad((h, n), tuple(leaves.values()), (state['grad_h'].double(), state['grad_n'].double()))
            out.update({'d_' + k: g for k, g in zip(leaves, gradients)})
        if case['kind'] != 'norm_product':
            return out
    codes, scales = state['codes'].double(), state['scales'].view(torch.uint8)
    weight = torch.cat([codes[:, k:k + BLOCK] * torch.exp2(scales[:, k // BLOCK].double() - 127.0).repeat_interleave(BLOCK)[:len(codes), None]
                        for k in range(0, codes.shape[1], BLOCK)], 1)[:, :d]
    z = _rows_exact(rows.reshape(-1, d)) @ weight.t()
    if state['layer_bias'] is not None:
        z = z + state['layer_bias'].double()
    act = {'none': lambda t: t, 'relu': torch.relu, 'silu': functional.silu, 'gelu': functional.gelu,
           'gelu_tanh': lambda t: functional.gelu(t, approximate='tanh')}[case.get('activation', 'none')]
    if case['kind'] == 'gated_product':
        gate, up = z.chunk(2, dim=-1)
        y = act(gate) * up
    else:
        y = act(z)
    y = y.reshape(*rows.shape[:-1], -1)
    if state['layer_residual'] is not None:
        y = y + state['layer_residual'].double()
    return {**out, 'y': y} if out else y
