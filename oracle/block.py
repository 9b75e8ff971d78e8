"""Oracle of the operators between a block's dense products: dropout and the
residual stream with its norms, forward and backward, from their definitions in
64 bits, with bounds on how far a computation in fp32 with stated roundings may be.

Bounds: running error analysis to first order.  A `Bounded` is a float64 value
with the largest absolute error that fp32 arithmetic in any order may have left
in it (u = 2^-24, a rounding to fp32, relative):

  a + b    e_a + e_b + u |a + b|
  a b      |a| e_b + |b| e_a + u |a b|
  sum      sum e + depth u sum |v|; a term passes through at most `depth`
           additions

The kernels add at most 32 elements in a lane (four chunks of eight), 6 times
across a wave, and at most 8 waves: 46; torch's row sums pass through fewer than 64
up to the widths of the tests.  Sums over rows pass through at most rows + 80 additions.
"""

import dataclasses

import numpy as np
import torch

from oracle import dense

U = dense.U
ROW_DEPTH = 64
rounding = dense.rounding
assert_within = dense.assert_within


@dataclasses.dataclass
class Bounded:
    v: torch.Tensor
    e: torch.Tensor

    @classmethod
    def exact(cls, v):
        v = torch.as_tensor(v, dtype=torch.float64)
        return cls(v, torch.zeros_like(v))

    def __add__(self, other):
        v = self.v + other.v
        return Bounded(v, self.e + other.e + U * v.abs())

    def __sub__(self, other):
        return self + Bounded(-other.v, other.e)

    def __mul__(self, other):
        v = self.v * other.v
        return Bounded(v, self.v.abs() * other.e + other.v.abs() * self.e + self.e * other.e + U * v.abs())

    def sum(self, dims, depth, keepdim=False):
        return Bounded(self.v.sum(dims, keepdim), (self.e + depth * U * (self.v.abs() + self.e)).sum(dims, keepdim))

    def mean(self, depth=ROW_DEPTH):
        n = self.v.shape[-1]
        s = self.sum((-1,), depth, True)  # times 1 / n, itself rounded
        return Bounded(s.v / n, s.e / n + 2 * U * s.v.abs() / n)

    def inverse_root(self):
        """v^-1/2 of a positive value, the hardware's good to 2 u.  Past a relative error of a half
        the first order says nothing: such rows are not compared."""
        relative = torch.where(self.v > 0, self.e / self.v, torch.zeros_like(self.v))
        v = self.v ** -0.5
        e = v * (relative / 2 * (1 + relative) + 4 * U)
        return Bounded(v, torch.where(relative > 0.5, torch.full_like(e, float('inf')), e))

    def result(self, dtype):
        """(value, bound) of the value rounded once to `dtype`."""
        return self.v, self.e * 1.01 + rounding(self.v, self.e, dtype)


def philox(counter, key):
    """Philox 4x32 with ten rounds, on Python integers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        p, q = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(q >> 32) ^ c[1] ^ k[0], q & 0xFFFFFFFF, (p >> 32) ^ c[3] ^ k[1], p & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def factors(rows, width, p, rng, stream):
    """0 or 65536 / (65536 - t) of every element, float64 [rows, width]."""
    seed, offset = (int(v) for v in rng)
    t = int(np.rint(65536.0 * p))
    key = (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF)
    groups = -(-width // 8)
    at = np.arange(rows * groups, dtype=np.uint64)
    low, half, shift = np.uint64(0xFFFFFFFF), np.uint64(0xFFFF), np.uint64(32)
    c = [at & low, at >> shift, np.full_like(at, stream), np.full_like(at, offset & 0xFFFFFFFF)]
    k = list(key)
    for _ in range(10):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> shift) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> shift) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    bits = np.stack([part for word in c for part in (word & half, word >> np.uint64(16))], -1)
    kept = bits.reshape(rows, groups * 8)[:, :width] >= t
    return torch.from_numpy(np.where(kept, 65536.0 / (65536 - t), 0.0))


def fp32(value):
    return float(np.float32(value))


def normalised(x, kind, eps):
    """((x - mean) / deviation, 1 / deviation)."""
    c = x - x.mean() if kind == 'layer' else x
    r = ((c * c).mean() + Bounded.exact(fp32(eps))).inverse_root()
    return c * r, r


@dataclasses.dataclass
class Stream:
    """One call's arguments; x and residual [rows, width], the gate of any broadcastable shape given as
    [rows, width] with `gate_rows`, the rows that share each of its rows."""

    x: torch.Tensor
    residual: torch.Tensor
    weight: torch.Tensor | None = None
    bias: torch.Tensor | None = None
    gate: torch.Tensor | None = None
    post_weight: torch.Tensor | None = None
    post_bias: torch.Tensor | None = None
    norm: str = 'rms'
    post: str = 'none'
    eps: float = 1e-6
    residual_scale: float = 1.0
    p: float = 0.0
    rng: tuple = (0, 0)
    stream: int = 0

    def __post_init__(self):
        self.sizes = self.x.shape
        self.flat = {}
        rows = self.x.numel() // max(1, self.sizes[-1])
        for name in ('x', 'residual', 'weight', 'bias', 'post_weight', 'post_bias'):
            t = getattr(self, name)
            if t is not None:
                t = t.detach().double().cpu()
                self.flat[name] = Bounded.exact(t.reshape(rows, -1) if name in ('x', 'residual') else t)
        if self.gate is not None:
            g = self.gate.detach().double().cpu()
            self.flat['gate'] = Bounded.exact(g.expand(self.sizes).reshape(rows, -1))
        self.k = None
        if self.p:
            k = factors(rows, self.sizes[-1], self.p, self.rng, self.stream)
            self.k = Bounded(k, (k - k.float().double()).abs())

    def _affine(self, x, weight, bias):
        if weight in self.flat:
            x = x * self.flat[weight]
        return x + self.flat[bias] if bias in self.flat else x

    def _forward(self):
        x, hat, r = self.flat['x'], None, None
        if self.post != 'none':
            hat, r = normalised(x, self.post, self.eps)
            x = self._affine(hat, 'post_weight', 'post_bias')
        v = x * self.k if self.k is not None else x
        s = Bounded.exact(fp32(self.residual_scale))
        h = self.flat['residual'] * s + (v * self.flat['gate'] if self.gate is not None else v)
        return h, v, hat, r

    def forward(self):
        """{'h', 'n'}: (value, bound)."""
        h = self._forward()[0]
        n = self._affine(normalised(h, self.norm, self.eps)[0], 'weight', 'bias')
        return {'h': h.result(self.residual.dtype), 'n': n.result(self.x.dtype)}

    @staticmethod
    def _transpose(g, hat, r, kind):
        d = g - hat * (g * hat).mean()
        return (d - g.mean() if kind == 'layer' else d) * r

    def backward(self, grad_h=None, grad_n=None):
        """{argument's name: (gradient, bound)}."""
        h, v, post_hat, post_r = self._forward()
        if self.gate is None and self.post == 'none' and self.residual.dtype == torch.float32:  # from h as it was rounded
            h = Bounded(h.v, h.e + rounding(h.v, h.e, self.residual.dtype))

        def flat(g):
            return Bounded.exact(torch.zeros_like(h.v) if g is None else g.detach().double().cpu().reshape(h.v.shape))

        gn, gt = flat(grad_n), flat(grad_h)
        out = {}
        rows = h.v.shape[0]
        if grad_n is not None:
            hat, r = normalised(h, self.norm, self.eps)
            d = gn * self.flat['weight'] if self.weight is not None else gn
            gt = gt + self._transpose(d, hat, r, self.norm)
            if self.weight is not None:
                out['weight'] = (gn * hat).sum((0,), rows + 80).result(self.weight.dtype)
        elif self.weight is not None:
            out['weight'] = torch.zeros(h.v.shape[1]).double(), torch.zeros(h.v.shape[1]).double()
        if self.bias is not None:
            out['bias'] = gn.sum((0,), rows + 80).result(self.bias.dtype)
        out['residual'] = (gt * Bounded.exact(fp32(self.residual_scale))).result(self.residual.dtype)
        gu = gt
        if self.gate is not None:
            own, dims = gt * v, self.gate.shape
            shaped = Bounded(own.v.reshape(self.sizes), own.e.reshape(self.sizes))
            if self.gate.dim() == 1:
                over = tuple(range(len(self.sizes) - 1))
            else:
                over = tuple(d for d in range(len(dims) - 1) if dims[d] == 1 and self.sizes[d] != 1)
            total = shaped.sum(over, rows + 80, True) if over else shaped
            out['gate'] = Bounded(total.v.reshape(dims), total.e.reshape(dims)).result(self.gate.dtype)
            gu = gt * self.flat['gate']
        if self.k is not None:
            gu = gu * self.k
        if self.post != 'none':
            if self.post_weight is not None:
                out['post_weight'] = (gu * post_hat).sum((0,), rows + 80).result(self.post_weight.dtype)
            if self.post_bias is not None:
                out['post_bias'] = gu.sum((0,), rows + 80).result(self.post_bias.dtype)
            d = gu * self.flat['post_weight'] if self.post_weight is not None else gu
            gu = self._transpose(d, post_hat, post_r, self.post)
        out['x'] = gu.result(self.x.dtype)
        return out


# ----------------------------------------------------------------- 8-bit blocks

BLOCK = 128
LOWEST = -117


def quantize(x, high):
    """(code bytes [rows, depth], scale bytes [ceil(rows / high), 4 ceil(width / 512)]) of a matrix whose blocks of
    `high` rows of 128 share a power of two, from the table of e4m3's magnitudes."""
    rows, width = x.shape
    v = x.detach().double().cpu().numpy()
    depth = -(-width // BLOCK) * BLOCK
    codes = np.zeros((rows, depth), np.uint8)
    scales = np.zeros((-(-rows // high), -(-width // (4 * BLOCK)) * 4), np.uint8)
    for i in range(scales.shape[0]):
        for j in range(depth // BLOCK):
            part = v[i * high:(i + 1) * high, j * BLOCK:(j + 1) * BLOCK]
            finite = np.isfinite(part)
            largest = np.where(finite, np.abs(part), 0.0).max()
            e = LOWEST
            while np.ldexp(448.0, e) < largest:
                e += 1
            y = np.abs(np.where(finite, part, 0.0)) * np.ldexp(1.0, -e)
            above = np.minimum(np.searchsorted(dense.MAGNITUDES, y), 126)
            below = np.maximum(above - 1, 0)
            up, down = dense.MAGNITUDES[above] - y, y - dense.MAGNITUDES[below]
            code = np.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
            code = np.where(np.ldexp(dense.MAGNITUDES[code], e) > torch.finfo(torch.float32).max, code - 1, code)
            code = np.where(finite, code, 0x7F) | (np.signbit(np.where(finite, part, 0.0)) * 0x80)
            codes[i * high:(i + 1) * high, j * BLOCK:j * BLOCK + part.shape[1]] = code
            scales[i, j] = e + 127
    return torch.from_numpy(codes), torch.from_numpy(scales)


def values(codes, scales, high, width):
    """What codes and scales stand for, float64 [rows, width]."""
    codes, scales = codes.view(torch.uint8).cpu().numpy(), scales.view(torch.uint8).cpu().numpy()
    value = np.append(dense.MAGNITUDES, np.nan)[codes & 0x7F] * np.where(codes & 0x80, -1.0, 1.0)
    e = scales.astype(np.int64)[:, :codes.shape[1] // BLOCK] - 127
    e = np.repeat(np.repeat(e, high, 0)[:codes.shape[0]], BLOCK, 1)
    return torch.from_numpy(np.where(e == 128, np.nan, np.ldexp(value, e))[:, :width])


# --------------------------------------------------------------- 8-bit products


def layer(x, weight, bias=None, residual=None, activation='none', gated=False, dtype=torch.float32, cores=False):
    """(y, bound) of a layer on float64 values x [rows, width] and weight [n_w, width].

    Exact products in fp32 sums, or with `cores` the 8-bit matrix cores': products p of a group are aligned to
    the largest one's power of two, 2^q, and lose what lies below g = 2^(q - 13).  A product of two e4m3 values
    has at most eight significant bits, so one of at least 2^(q - 6) loses nothing and a smaller one at most
    min(|p|, g); the sums that pass through a group's alignment lose at most g each, four times per block of 128.
    The group is bounded by its block."""
    z = x @ weight.t()
    size = x.abs() @ weight.abs().t()
    err = (x.shape[1] + 2) * U * 1.01 * size
    if cores:
        for k in range(0, x.shape[1], BLOCK):
            p = (x[:, None, k:k + BLOCK] * weight[None, :, k:k + BLOCK]).abs()
            largest = p.amax(-1, keepdim=True)
            q = torch.floor(torch.log2(largest.clamp_min(1e-300)))
            g = torch.exp2(q - 13)
            err = err + (torch.where(p < torch.exp2(q - 6), torch.minimum(p, g), torch.zeros_like(p)).sum(-1) + 4 * g[..., 0])
    if bias is not None:
        z = z + bias
        err = err + U * z.abs() + U * bias.abs()
    steep = dense.MOST_SLOPE[activation]
    if gated:
        n = z.shape[1] // 2
        a, b, da, db = z[:, :n], z[:, n:], err[:, :n], err[:, n:]
        value, _ = dense.activation(a, activation)
        dv = steep * da + dense.ACT_ERROR * (1 + a.abs())
        y = value * b
        e = dv * (b.abs() + db) + value.abs() * db + 2 * U * y.abs()
    else:
        y, _ = dense.activation(z, activation)
        e = steep * err + (dense.ACT_ERROR * (1 + z.abs()) if activation != 'none' else 0)
    if residual is not None:
        y = y + residual
        e = e + 2 * U * (y.abs() + residual.abs())
    return y, e * 1.01 + rounding(y, e, dtype)
