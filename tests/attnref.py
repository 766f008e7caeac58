"""Plain numpy (64-bit) forms of the attention-side operators, and device-side helpers for their tests."""
import math

import numpy as np

import moe_rocm as M

HALF = {M.F32: 2.0 ** -24, M.F16: 2.0 ** -11, M.BF16: 2.0 ** -8}  # half a step, relative
SIZE = {M.F32: 4, M.F16: 2, M.BF16: 2}


def to_bits(x, dtype):
    """float array -> the stored elements of `dtype`, rounded to nearest even."""
    x = np.asarray(x, np.float32)
    if dtype == M.F32:
        return x
    if dtype == M.F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    b = x.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bits(b, dtype):
    if dtype == M.BF16:
        return (b.astype(np.uint32) << 16).view(np.float32)
    return b.astype(np.float32)


def rounded(x, dtype):
    return from_bits(to_bits(x, dtype), dtype)


class Rows:
    """Rows [T, H, D] on the device inside a buffer [T, pad heads], filled with a mark around them."""

    def __init__(self, ctx, x, dtype, T=None, H=None, D=None, pad=0, first=0):
        T, H, D = x.shape if x is not None else (T, H, D)
        self.ctx, self.dtype, self.shape, self.first = ctx, dtype, (T, H, D), first
        self.width = (H + pad) * D
        kind = np.float32 if dtype == M.F32 else np.float16 if dtype == M.F16 else np.uint16
        self.mark = to_bits(np.float32(-7.5), dtype).astype(kind)
        host = np.full((max(T, 1), H + pad, D), self.mark, kind)
        if x is not None:
            host[:T, first:first + H] = to_bits(x, dtype)
        self.buf = ctx.to_device(host)
        self.heads = M.Heads(self.buf.ptr + first * D * SIZE[dtype], H, dtype, self.width if pad else 0, D if pad else 0)

    def all(self):
        kind = np.float32 if self.dtype == M.F32 else np.float16 if self.dtype == M.F16 else np.uint16
        return self.buf.download(kind, max(self.shape[0], 1) * self.width)

    def get(self):
        T, H, D = self.shape
        a = self.all().reshape(-1, self.width // D, D)
        outside = np.concatenate([a[:, :self.first].ravel(), a[:, self.first + H:].ravel()])
        assert (outside == self.mark).all(), "written outside the rows"
        return from_bits(a[:T, self.first:self.first + H], self.dtype)

    def free(self):
        self.buf.free()


def i32(ctx, a):
    return ctx.to_device(np.asarray(a, np.int32))


# ---- rotary positions ------------------------------------------------------------------------
def rope_freqs(n, base, scaling="plain", factor=1.0, orig=0):
    f = [base ** (-2.0 * i / n) for i in range(n // 2)]
    if scaling == "linear":
        return np.array(f) / factor, 1.0
    if scaling.startswith("yarn"):
        low, high = (n * math.log(orig / (b * 2 * math.pi)) / (2 * math.log(base)) for b in (32.0, 1.0))
        if scaling == "yarn":
            low, high = math.floor(low), math.ceil(high)
        low = max(low, 0)
        high = max(low, min(high, n - 1))
        if low == high:
            high += 0.001
        r = np.clip((np.arange(n // 2) - low) / (high - low), 0, 1)
        return np.array(f) / factor * r + np.array(f) * (1 - r), 0.1 * math.log(factor) + 1
    return np.array(f), 1.0


def rope(x, pos, freqs, mul, interleaved, w=None, eps=0.0):
    """-> (values, magnitude of each value's pair, what its rounding errors are relative to)."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    n = 2 * len(freqs)
    t = np.asarray(pos, np.float64)[:, None, None] * freqs
    c, s = np.cos(t) * mul, np.sin(t) * mul
    ia, ib = (np.arange(0, n, 2), np.arange(1, n, 2)) if interleaved else (np.arange(n // 2), np.arange(n // 2, n))
    a, b = x[..., ia], x[..., ib]
    y, size = x.copy(), np.abs(x)
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    size[..., ia] = size[..., ib] = np.hypot(a, b) * mul
    return y, size


# ---- the cache's formats ------------------------------------------------------------------------
FP4 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def stored(x, fmt):
    """The values a cache of `fmt` holds for x: the grid value nearest to x / 2^e, by distance."""
    x = np.where(np.isnan(x), 0, x).astype(np.float64)
    if fmt == M.KV_F16:
        return np.clip(x, -65504, 65504).astype(np.float32).astype(np.float16).astype(np.float64)
    hi = 13 if fmt == M.KV_MXFP4 else 9
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = np.abs(b).max(-1)
    e = np.full(top.shape, -16)
    for k in range(-16, hi):
        over = top > 7.0 * 2.0 ** k if fmt == M.KV_MXFP4 else top >= 127.5 * 2.0 ** k
        e = np.where(over, k + 1, e)
    s = 2.0 ** e[..., None]
    a = np.abs(b) / s
    if fmt == M.KV_MXINT8:
        return (np.minimum(np.rint(a), 127) * np.sign(b) * s).reshape(x.shape)
    d = np.abs(np.minimum(a, 6)[..., None] - FP4)
    code = d.argmin(-1)  # the lower of two nearest codes
    tie = np.take_along_axis(d, np.minimum(code + 1, 7)[..., None], -1)[..., 0] == d.min(-1)
    code = np.where(tie & (code % 2 == 1) & (code < 7), code + 1, code)
    return (FP4[code] * np.sign(b) * s).reshape(x.shape)


# ---- attention ------------------------------------------------------------------------------------
def attend(q, k, v, scale, first, last, sink=None):
    """One query row over keys first..last of k, v [n, D] -> (out, sum p |v|, largest |score| sum, keys seen)."""
    D = len(q)
    if last < first:
        return np.zeros(D), np.zeros(D), 0.0, 0
    q, k, v = q.astype(np.float64), k[first:last + 1].astype(np.float64), v[first:last + 1].astype(np.float64)
    s = k @ q * scale
    size = float((np.abs(k) @ np.abs(q)).max() * abs(scale))
    m = max(s.max(), -np.inf if sink is None else float(sink))
    p = np.exp(s - m)
    z = p.sum() + (0.0 if sink is None else math.exp(float(sink) - m))
    return p @ v / z, p @ np.abs(v) / z, size, len(s)


def attention_bound(y, size_v, size_s, n, D, out_type, p_half):
    """How far a result may be off. The output's own rounding. The weights': each p is off by p_half of it at most (and
    half of the smallest f16 step, 2^-25, for each of n keys, whose weights sum to 1 or more before the division), in
    the sum of values and in the divisor alike, so the quotient by p_half (sum p |v| + |y| sum p) / sum p. The scores',
    D products summed in 32 bits and two more roundings before the exponential (whose own error is a few steps of 32
    bits), each an error of p relative to p, in sum and quotient."""
    ds = (D + 4) * 2.0 ** -24 * size_s + 8 * 2.0 ** -24
    return HALF[out_type] * np.abs(y) * 1.01 + p_half * np.abs(y) + (p_half + 2 * ds + n ** 0.5 * 2.0 ** -23) * size_v + n * 2.0 ** -25 * np.max(size_v, initial=0) + 2.0 ** -25
