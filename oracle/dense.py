"""Oracle of the dense operators: the layers, their gradients and the 8-bit
rows from their definitions in 64 bits, and bounds on how far a computation in
fp32 sums with stated roundings may be from them.

Bounds.  With u = 2^-24 (a rounding to fp32, relative), a sum of n products
in any order and its n - 1 additions is off by at most (n + 1) u sum|a||b| to
first order; `SLACK` covers the second-order terms.  A result in type t is off
by half a step more: h = finfo(t).eps / 2 relative (or half the smallest
subnormal).  An activation is computed from a z that is off by dz: it moves by
at most max|act'| dz, its slope by max|act''| dz, and its own evaluation in
fp32 adds ACT_ERROR (1 + |z|).
"""

import dataclasses

import numpy as np
import torch

U = 2.0 ** -24
SLACK = 1.01
# The kernels evaluate Phi, the sigmoid and their products in at most 25 fp32
# operations on quantities of at most 1 + |z| (the exponent's argument, up to
# z^2, is off by z^2 u relative to a factor exp(-z^2 / 2) that shrinks faster:
# z^3 exp(-z^2 / 2) <= 1.2); hardware exp2 and reciprocal are good to 2 u.
ACT_ERROR = 32 * U
# max |act'| and max |act''| over all z (gelu: 1.129 and 0.798 = 2 phi(0);
# gelu_tanh likewise to three digits; silu: 1.0998 and 1/2).
MOST_SLOPE = {'none': 1.0, 'relu': 1.0, 'gelu': 1.13, 'gelu_tanh': 1.13, 'silu': 1.1}
MOST_BEND = {'none': 0.0, 'relu': 0.0, 'gelu': 0.8, 'gelu_tanh': 0.81, 'silu': 0.5}


def activation(z, name):
    """act(z) and act'(z) of a float64 tensor."""
    if name == 'none':
        return z, torch.ones_like(z)
    if name == 'relu':
        return z.clamp_min(0), (z > 0).double()
    if name == 'silu':
        s = torch.sigmoid(z)
        return z * s, s + z * s * torch.sigmoid(-z)
    if name == 'gelu':
        cdf = 0.5 * torch.special.erfc(-z / 2 ** 0.5)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
    if name == 'gelu_tanh':
        c = (2 / torch.pi) ** 0.5
        y = 2 * c * (z + 0.044715 * z ** 3)
        s = torch.sigmoid(y)
        return z * s, s + z * s * torch.sigmoid(-y) * 2 * c * (1 + 3 * 0.044715 * z * z)
    raise ValueError(name)


@dataclasses.dataclass
class Layer:
    """A layer's inputs as float64 matrices on the CPU."""

    x: torch.Tensor
    weight: torch.Tensor
    bias: torch.Tensor | None
    residual: torch.Tensor | None
    activation: str
    gated: bool

    @classmethod
    def of(cls, x, weight, bias=None, residual=None, act='none', gated=False):
        flat = [None if t is None else t.detach().double().cpu() for t in (x, weight, bias, residual)]
        return cls(flat[0].reshape(-1, x.shape[-1]), flat[1], flat[2],
                   None if residual is None else flat[3].reshape(-1, residual.shape[-1]), act, gated)

    def _z(self):
        z = self.x @ self.weight.t()
        return z if self.bias is None else z + self.bias

    def _z_error(self):
        size = self.x.abs() @ self.weight.abs().t()
        if self.bias is not None:
            size = size + self.bias.abs()
        return (self.x.shape[1] + 2) * U * SLACK * size

    def _halves(self, z):
        n = z.shape[1] // 2
        return z[:, :n], z[:, n:]

    def forward(self, dtype):
        """(y, bound on |computed - y|) for a result in `dtype`."""
        z, dz = self._z(), self._z_error()
        if self.gated:
            (a, b), (da, db) = self._halves(z), self._halves(dz)
            value, _ = activation(a, self.activation)
            dv = MOST_SLOPE[self.activation] * da + ACT_ERROR * (1 + a.abs())
            y = value * b
            err = dv * (b.abs() + db) + value.abs() * db + 2 * U * y.abs()
        else:
            value, _ = activation(z, self.activation)
            y = value
            err = MOST_SLOPE[self.activation] * dz
            if self.activation != 'none':
                err = err + ACT_ERROR * (1 + z.abs())
        if self.residual is not None:
            y = y + self.residual
            err = err + 2 * U * (value.abs() + self.residual.abs())
        return y, err * SLACK + rounding(y, err, dtype)

    def backward(self, grad, dtype, bias_dtype):
        """{'x', 'weight', 'bias'}: (gradient, bound)."""
        g = grad.detach().double().cpu().reshape(-1, grad.shape[-1])
        z, dz_err = self._z(), self._z_error()
        bend, steep = MOST_BEND[self.activation], MOST_SLOPE[self.activation]
        if self.gated:
            (a, b), (da, db) = self._halves(z), self._halves(dz_err)
            value, slope = activation(a, self.activation)
            dv, ds = steep * da + ACT_ERROR * (1 + a.abs()), bend * da + ACT_ERROR * (1 + a.abs())
            if self.activation == 'relu':  # as below: within its error of 0 the gate's slope is 0 or 1
                ds = torch.where(a.abs() <= da, torch.ones_like(ds), ds)
            first, second = g * b * slope, g * value
            err = torch.cat([g.abs() * (ds * (b.abs() + db) + slope.abs() * db) + 3 * U * first.abs(),
                             g.abs() * dv + 2 * U * second.abs()], 1)
            dz = torch.cat([first, second], 1)
        elif self.activation == 'none':
            dz, err = g, torch.zeros_like(g)
        elif self.activation == 'relu':
            # The slope jumps at 0: where z is within its own error of 0, either side's is right.
            dz = g * (z > 0)
            err = torch.where(z.abs() <= dz_err, g.abs(), torch.zeros_like(g))
        else:
            _, slope = activation(z, self.activation)
            dz = g * slope
            err = g.abs() * (bend * dz_err + ACT_ERROR * (1 + z.abs())) + 2 * U * dz.abs()
        kept = err if self.activation == 'none' and not self.gated else err + rounding(dz, err, dtype)
        size = dz.abs() + kept
        m, n = dz.shape

        def product(value, left, left_err, right):
            e = left_err @ right.abs() + (left.shape[1] + 1) * U * SLACK * ((left.abs() + left_err) @ right.abs())
            return value, e + rounding(value, e, dtype)

        bias = dz.sum(0)
        bias_err = kept.sum(0) + (m + 1) * U * SLACK * size.sum(0)
        return {
            'x': product(dz @ self.weight, dz, kept, self.weight),
            'weight': product(dz.t() @ self.x, dz.t(), kept.t(), self.x),
            'bias': (bias, bias_err + rounding(bias, bias_err, bias_dtype)),
        }


def rounding(value, err, dtype):
    """Half a step of `dtype` at value +- err."""
    info = torch.finfo(dtype)
    return (value.abs() + err) * (info.eps / 2) + info.smallest_normal * info.eps


def assert_within(got, want, bound):
    """Every element of `got` within `bound` of `want`; inf where `want` is past the type's largest."""
    got = got.detach().double().cpu().reshape(want.shape)
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), (
        f'{int(bad.sum())} of {bad.numel()} outside; worst {float((off / bound).nan_to_num(float("inf")).max()):.3g} '
        f'times the bound, first at {torch.nonzero(bad)[0].tolist()}: got {got[bad][0]}, want {want[bad][0]}')


# ------------------------------------------------------------------ 8-bit rows

BLOCK = 32
LOWEST = {torch.float32: -117, torch.bfloat16: -117, torch.float16: -15}
# e4m3's 127 finite magnitudes, in order of their codes.
MAGNITUDES = np.array([m * 2.0 ** -9 if p == 0 else (8 + m) * 2.0 ** (p - 10) for p in range(16) for m in range(8)][:127])


def quantize(x):
    """(code bytes [rows, width], scale bytes [rows, blocks]) of a matrix."""
    dtype, width = x.dtype, x.shape[1]
    v = x.detach().double().cpu().numpy()
    rows = v.shape[0]
    codes = np.zeros((rows, width), np.uint8)
    scales = np.zeros((rows, -(-width // BLOCK)), np.uint8)
    for b in range(scales.shape[1]):
        part = v[:, b * BLOCK:(b + 1) * BLOCK]
        finite = np.isfinite(part)
        largest = np.where(finite, np.abs(part), 0.0).max(1)
        e = np.full(rows, LOWEST[dtype])
        while True:
            short = np.ldexp(448.0, e) < largest
            if not short.any():
                break
            e = e + short
        y = np.abs(np.where(finite, part, 0.0)) * np.ldexp(1.0, -e)[:, None]
        above = np.minimum(np.searchsorted(MAGNITUDES, y), 126)
        below = np.maximum(above - 1, 0)
        up, down = MAGNITUDES[above] - y, y - MAGNITUDES[below]
        code = np.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
        code = np.where(np.ldexp(MAGNITUDES[code], e[:, None]) > torch.finfo(dtype).max, code - 1, code)
        code = np.where(finite, code, 0x7F)
        codes[:, b * BLOCK:(b + 1) * BLOCK] = code | (np.signbit(np.where(finite, part, 0.0)) * 0x80)
        scales[:, b] = e + 127
    return codes, scales


def dequantize(codes, scales):
    """Their values, float64 [rows, width]."""
    value = np.append(MAGNITUDES, np.nan)[codes & 0x7F] * np.where(codes & 0x80, -1.0, 1.0)
    e = np.repeat(scales.astype(np.int64) - 127, BLOCK, axis=1)[:, :codes.shape[1]]
    return np.where(e == 128, np.nan, np.ldexp(value, e))
