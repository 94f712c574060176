"""Shared by the tests of the 4-bit cache and of linear attention: their definitions in 64 bits and error bounds.

Linear attention's bounds count every rounding. With w_tj the decays, A = |scale| (sum_j w_tj sum_c |q_tc k_jc| |v_j| +
w |q| |S_0|), B the same sum of |k| |v| and |S_0| that a state is:
  products take states and weights as two 16-bit numbers at least (2^-16 each, bf16's two roundings), a decay is off
  by 2^-21 (fp32 exponent and exp2) and passes n / 64 + 2 steps, n + hd + 64 terms are added in fp32 (2^-24 each):
    |o - exact| <= A (2^-14 + (n / 64 + 2) 2^-21 + (n + hd + 64) 2^-24) + u |o| + smallest
  the next state's products take 21 bits or more of a decayed value:
    |S - exact| <= B (2^-20 + (n / 64 + 2) 2^-21 + (n + hd + 64) 2^-24)
"""
import numpy as np

import prism_amd as P
from seqlib import HALF_STEP, SMALLEST, to_bits, values

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
POWERS = {"fp16": (-23, 13), "bf16": (-125, 125)}


def block_of(hd):
    return min(hd, 32)


def quantise(x, dtype):
    """x [..., hd] fp32 -> (codes uint8 [..., hd / 2], bytes of the blocks' powers uint8 [..., blocks]), by the
    definition: the smallest e with max <= 7 * 2^e, the nearest magnitude, ties to the even number."""
    x = np.asarray(x, np.float32).astype(np.float64)
    hd = x.shape[-1]
    b = x.reshape(x.shape[:-1] + (hd // block_of(hd), block_of(hd)))
    fine = np.isfinite(b).all(-1, keepdims=True)
    top = np.where(fine, np.abs(np.where(fine, b, 0)).max(-1, keepdims=True), 0)
    low, high = POWERS[dtype]
    grid = 7.0 * 2.0 ** np.arange(low, high)  # e = low + how many of them are below the largest
    e = low + np.searchsorted(grid, top, side="left")
    a = np.abs(np.where(fine, b, 0)) / 2.0 ** e
    far = np.abs(a[..., None] - MAGNITUDES)
    # the nearest; of two as near, the even one: odd numbers a hair further off
    code = np.argmin(np.where(far == far.min(-1, keepdims=True), np.arange(8) % 2, 9), -1)
    code = np.where(fine, code + 8 * np.signbit(b), 0).astype(np.uint8).reshape(x.shape)
    return code[..., 0::2] | code[..., 1::2] << 4, np.where(fine, e + 127, 255).astype(np.uint8)[..., 0]


def dequantise(codes, scales):
    """-> fp64 [..., hd]."""
    c = np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[:-1] + (2 * codes.shape[-1],))
    v = np.where(c & 8, -1.0, 1.0) * MAGNITUDES[c & 7]
    b = scales.astype(np.float64)
    s = np.where(b == 255, np.nan, 2.0 ** (b - 127))
    return (v.reshape(scales.shape + (v.shape[-1] // scales.shape[-1],)) * s[..., None]).reshape(v.shape)


def turned(x, pos, pairs, layout, ladder, base, bits=64):
    """x [tokens][heads][hd], pos [axes][tokens] -> (turned, bound without the rounding to a type). Angle: 2^-51 of its
    size here and there; sin, cos, products in 64 bits: 2^-50; the result in fp32: 2^-24. In 32 bits (queries, keys that
    stay 16-bit) cos and sin are rounded by 2^-25 at most, the first product by 2^-24 of it: (|u| + |w|) 2^-23 more."""
    more = 2.0 ** -23 if bits == 32 else 0.0
    n, y, bound = sum(pairs), x.copy(), np.zeros_like(x)
    i = 0
    for axis, count in enumerate(pairs):
        for j in range(count):
            f = base ** -(i / n if ladder == P.ROPE_ONE_LADDER else j / count)
            phi = pos[axis][:len(x)].astype(np.float64)[:, None] * f
            a, b = (i, i + n) if layout == P.ROPE_HALVES else (2 * i, 2 * i + 1)
            u, w = x[..., a], x[..., b]
            y[..., a], y[..., b] = u * np.cos(phi) - w * np.sin(phi), w * np.cos(phi) + u * np.sin(phi)
            for c in (a, b):
                bound[..., c] = (np.abs(u) + np.abs(w)) * (np.abs(phi) * 2.0 ** -50 + 2.0 ** -49 + more) + 2.0 ** -24 * np.abs(y[..., c])
            i += 1
    return y, bound


def linear(q, k, v, rate, start, scale, dtype):
    """One head along one sequence: q [n][hd], k, v [n][hd], start [hd][hd] -> (out, bound, state, bound)."""
    n, hd = q.shape
    keep = np.exp(-max(rate, 0.0)) if rate == rate else 1.0
    S, B = start.copy(), np.abs(start)
    out, bound = np.zeros((n, hd)), np.zeros((n, hd))
    for t in range(n):
        S, B = S * keep + np.outer(k[t], v[t]), B * keep + np.outer(np.abs(k[t]), np.abs(v[t]))
        out[t] = scale * (q[t] @ S)
        off = 2.0 ** -14 + (n / 64 + 2) * 2.0 ** -21 + (n + hd + 64) * 2.0 ** -24
        bound[t] = abs(scale) * (np.abs(q[t]) @ B) * off + HALF_STEP[dtype] * np.abs(out[t]) + SMALLEST[dtype]
    return out, bound, S, B * (2.0 ** -20 + (n / 64 + 2) * 2.0 ** -21 + (n + hd + 64) * 2.0 ** -24)


class Cache:
    """A 4-bit or 16-bit cache on the host: pools whose slots hold what must not be used, pages in mixed order."""

    def __init__(self, rng, lengths, kv, hd, page, dtype, four, spare=3):
        need = [-(-n // page) for n in lengths]
        pool = sum(need) + spare
        order = iter(rng.permutation(pool))
        self.table = np.full((len(lengths), max(need + [0]) + 1), -1, np.int32)
        self.table[:, -1] = 2 ** 31 - 1
        for s, n in enumerate(need):
            for j in range(n):
                self.table[s, j] = next(order)
        self.four, self.page, self.kv, self.hd, self.dtype = four, page, kv, hd, dtype
        shape = (pool, kv, page)
        if four:
            self.k, self.v = (rng.integers(0, 256, shape + (hd // 2,), np.uint8) for _ in "kv")
            self.ks, self.vs = (np.full(shape + (hd // block_of(hd),), 255, np.uint8) for _ in "kv")
        else:
            self.k, self.v = (np.full(shape + (hd,), 0x7FFF, np.uint16) for _ in "kv")  # NaN in both types
            self.ks = self.vs = np.zeros(16, np.uint8)

    def desc(self):
        t = {"fp16": P.F16, "bf16": P.BF16}[self.dtype]
        return P.CacheDesc(dtype=t, n_kv_heads=self.kv, head_dim=self.hd, page_size=self.page, n_pages=self.k.shape[0],
                           n_seqs=len(self.table), table_pages=self.table.shape[1])

    def put(self, dev):
        self.there = [dev.put(a) for a in (self.k, self.v, self.ks, self.vs)]
        return P.CachePages(k=self.there[0], v=self.there[1], k_scales=self.there[2], v_scales=self.there[3])

    def got(self, dev):
        """The pools as the device has them now."""
        return [dev.get(p, a.shape, a.dtype) for p, a in zip(self.there, (self.k, self.v, self.ks, self.vs))]

    def place(self, s, j):
        """(page, slot) of token j of sequence s, None if it has none."""
        if not (0 <= s < len(self.table) and 0 <= j < self.table.shape[1] * self.page):
            return None
        p = self.table[s, j // self.page]
        return (p, j % self.page) if 0 <= p < self.k.shape[0] else None

    def write(self, s, j, k, v):
        """fp32 rows [kv][hd] into token j of sequence s."""
        at = self.place(s, j)
        if at is None:
            return
        p, slot = at
        if self.four:
            self.k[p, :, slot], self.ks[p, :, slot] = quantise(k, self.dtype)
            self.v[p, :, slot], self.vs[p, :, slot] = quantise(v, self.dtype)
        else:
            self.k[p, :, slot], self.v[p, :, slot] = to_bits(k, self.dtype), to_bits(v, self.dtype)

    def fill(self, s, js, k, v):
        """fp32 rows [len(js)][kv][hd] into tokens js of sequence s, all of which have places; 4 bits."""
        p, slot = self.table[s, js // self.page], js % self.page
        self.k[p, :, slot], self.ks[p, :, slot] = quantise(k, self.dtype)
        self.v[p, :, slot], self.vs[p, :, slot] = quantise(v, self.dtype)

    def rows(self, s, js):
        """(k, v) [len(js)][kv][hd] in 64 bits; 4 bits."""
        p, slot = self.table[s, js // self.page], js % self.page
        return dequantise(self.k[p, :, slot], self.ks[p, :, slot]), dequantise(self.v[p, :, slot], self.vs[p, :, slot])

    def read(self, s, j):
        """(k, v) [kv][hd] in 64 bits."""
        p, slot = self.place(s, j)
        if self.four:
            return (dequantise(self.k[p, :, slot], self.ks[p, :, slot]), dequantise(self.v[p, :, slot], self.vs[p, :, slot]))
        return values(self.k[p, :, slot], self.dtype), values(self.v[p, :, slot], self.dtype)
