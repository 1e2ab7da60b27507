"""Rotary positions and the paged 4-bit key / value cache on the CPU: the rules of the entry points in
include/fopt_b200.h, restated with numpy. Angles and attention are in 64 bits or more; what the rules fix to
f32 (the rotation's products, the quantiser) is f32 with one rounding per operation, so that stored codes
can be compared bit for bit."""
from __future__ import annotations

import numpy as np

GROUP = 32
_F = np.float32


def bf16_round(x):
    """f32 -> the nearest bf16 as f32 (half to even, subnormals to signed zero, NaN kept)."""
    x = np.asarray(x, _F)
    u = x.view(np.uint32).astype(np.uint64)
    r = (((u + 0x7FFF + ((u >> 16) & 1)) >> 16) << 16).astype(np.uint32).view(_F)
    tiny = (u >> 23) & 0xFF == 0
    return np.where(np.isnan(x), x, np.where(tiny, np.copysign(_F(0), x), r)).astype(_F)


def turns(positions, inv_freq, magnitude=1.0):
    """(cos, sin) f32 [T, pairs] of positions * inv_freq, the angle in extended precision."""
    a = np.asarray(positions, np.longdouble)[:, None] * np.asarray(inv_freq, np.longdouble)
    m = np.float64(magnitude)
    return (np.cos(a).astype(np.float64) * m).astype(_F), (np.sin(a).astype(np.float64) * m).astype(_F)


def rotate(x, positions, inv_freq, layout="half", magnitude=1.0):
    """x f32 [T, H, D] -> rotated f32, products and sums rounded one by one."""
    x = np.asarray(x, _F)
    c, s = (t[:, None, :] for t in turns(positions, inv_freq, magnitude))
    n = c.shape[-1]
    first, second = (slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    y = x.copy()
    with np.errstate(invalid="ignore", over="ignore"):
        y[..., first] = x[..., first] * c - x[..., second] * s
        y[..., second] = x[..., second] * c + x[..., first] * s
    return y


def quantise(x):
    """x f32 [..., D] -> (codes int8 [..., D], steps f32, offsets f32 [..., D / 32])."""
    x = np.asarray(x, _F)
    x = np.where(np.isnan(x), _F(0), np.clip(x, -_F(2.0 ** 100), _F(2.0 ** 100))).astype(_F)
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    lo, hi = g.min(-1), g.max(-1)
    step = bf16_round((hi - lo) / _F(15))
    offset = bf16_round(lo + _F(8) * step)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        c = np.where(step[..., None] > 0, np.rint((g - offset[..., None]) / step[..., None]), _F(0))
    return np.clip(c, -8, 7).astype(np.int8).reshape(x.shape), step, offset


def values(codes, step, offset):
    """code * step + offset, f64."""
    g = codes.reshape(*codes.shape[:-1], -1, GROUP).astype(np.float64)
    return (g * step[..., None].astype(np.float64) + offset[..., None]).reshape(codes.shape)


class Cache:
    """Plain pages: codes int8 [P, H, S, D], steps and offsets f32 [P, H, S, D / 32], for k and for v."""

    def __init__(self, pages, page_size, heads, dim):
        self.page_size, self.heads, self.dim = page_size, heads, dim
        self.codes = {n: np.zeros((pages, heads, page_size, dim), np.int8) for n in "kv"}
        self.step = {n: np.zeros((pages, heads, page_size, dim // GROUP), _F) for n in "kv"}
        self.offset = {n: np.zeros((pages, heads, page_size, dim // GROUP), _F) for n in "kv"}

    def append(self, k, v, slots):
        """k (rotated already) and v f32 [T, H, D] into the slots; negative slots are no tokens."""
        slots = np.asarray(slots)
        live = slots >= 0
        p, s = slots[live] // self.page_size, slots[live] % self.page_size
        for n, x in (("k", k), ("v", v)):
            c, st, of = quantise(np.asarray(x, _F)[live])
            self.codes[n][p, :, s], self.step[n][p, :, s], self.offset[n][p, :, s] = c, st, of

    def values(self, n):
        return values(self.codes[n], self.step[n], self.offset[n])

    def parts(self, n):
        """(code + 8) step + |offset - 8 step|: the size of what sums to a value, which may cancel in it."""
        c, st, of = (a[n].astype(np.float64) for a in (self.codes, self.step, self.offset))
        return values(c + 8, st, np.abs(of - 8 * st))

    def image(self, n):
        """The codes in the order of the cache's image (flat)."""
        w = 8 if n == "k" else 4
        c = self.codes[n].reshape(*self.codes[n].shape[:-1], -1, GROUP // w, w)  # [.., G, 32 / w, w]
        return np.ascontiguousarray(np.swapaxes(c, -3, -2)).reshape(-1)

    def scale_image(self, n):
        return np.stack([self.step[n], self.offset[n]], -1).reshape(-1)


def attention(q, cache, table, q_start, kv_len, scale, causal=True):
    """q f32 [T, Hq, D]; table [B, W]. Returns (o, a): the output in f64 and, for every output element,
    sum_i p_i ((code_i + 8) step_i + |offset_i - 8 step_i|), which a rounding of probabilities is relative to:
    the products may run on codes from 0 to 15 and offsets apart. Rows of no sequence are NaN."""
    T, Hq, D = q.shape
    group = Hq // cache.heads
    o, a = np.full((T, Hq, D), np.nan), np.zeros((T, Hq, D))
    K, V, A = cache.values("k"), cache.values("v"), cache.parts("v")
    for b, n in enumerate(kv_len):
        q0, q1 = q_start[b], q_start[b + 1]
        pages = np.asarray(table[b][:-(-int(n) // cache.page_size)], np.int64)
        for h in range(cache.heads):
            k = K[pages, h].reshape(-1, D)[:n]
            v, va = V[pages, h].reshape(-1, D)[:n], A[pages, h].reshape(-1, D)[:n]
            for t in range(q0, q1):
                seen = max(0, n - (q1 - q0) + (t - q0) + 1) if causal else n
                rows = slice(h * group, (h + 1) * group)
                if not seen:
                    o[t, rows] = 0
                    continue
                x = (q[t, rows].astype(np.float64) @ k[:seen].T) * scale
                with np.errstate(invalid="ignore", over="ignore"):
                    p = np.exp(x - x.max(-1, keepdims=True))
                    p /= p.sum(-1, keepdims=True)
                    o[t, rows] = p @ v[:seen]
                    a[t, rows] = p @ va[:seen]
    return o, a
