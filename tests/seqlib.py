"""Shared by the tests of the sequence operators: 16-bit types, definitions in 64 bits, error bounds.

Bounds count every rounding of the kernels. u = half a step of the type (fp16 2^-11, bf16 2^-8).
Attention: the scores are sums of hd products in fp32, so a weight is off by a factor 1 + d with
d <= (hd + 8) 2^-24 scale max_j sum_i |q_i k_ij| (the products' sum, the scaling and the
exponent's argument; the maximum is subtracted from numbers of that size), and as much again in the
sum of the weights; 2^-20 for exp2 and the division; the weights may be rounded to the type before
they meet v (u, and 2^-25 absolute where fp16 weights are subnormal, the largest weight being at least 1);
the n terms are added in fp32 (n 2^-24); the output is rounded once (u |o|, and half the type's smallest
step). Each but the last acts on A = sum_j p_j |v_j|.
"""
import numpy as np

import prism_amd as P

TYPES = {"fp16": P.F16, "bf16": P.BF16}
HALF_STEP = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}
SMALLEST = {"fp16": 2.0 ** -25, "bf16": 2.0 ** -134}
NAN = {"fp16": 0x7E00, "bf16": 0x7FC0}


def to_bits(x, dtype):
    """fp64 -> 16-bit patterns, to nearest, ties to even."""
    x = np.asarray(x, np.float32)
    if dtype == "fp16":
        return x.astype(np.float16).view(np.uint16)
    b = x.view(np.uint32)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def values(bits, dtype):
    bits = np.ascontiguousarray(bits, np.uint16)
    if dtype == "fp16":
        return bits.view(np.float16).astype(np.float64)
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def normal(rng, shape, dtype):
    return to_bits(rng.standard_normal(shape), dtype)


def visible(p, n, left, right, sinks):
    """Which of n keys the query at p sees."""
    j = np.arange(n)
    near = np.ones(n, bool) if left < 0 else j >= p - left
    after = np.ones(n, bool) if right < 0 else j <= p + right
    return after & (near | (j < sinks))


def attention_row(q, k, v, seen, scale, dtype):
    """One query over keys k, v [n][hd] where seen: (output, bound)."""
    hd = q.shape[0]
    if not seen.any():
        return np.zeros(hd), np.zeros(hd)
    k, v = k[seen], v[seen]
    z = scale * (k @ q)
    w = np.exp(z - z.max())
    total = w.sum()
    o = w @ v / total
    size = w @ np.abs(v) / total
    d = (hd + 8) * 2.0 ** -24 * scale * (np.abs(k) @ np.abs(q)).max()
    u, n = HALF_STEP[dtype], len(k)
    sub = 2.0 ** -25 * np.abs(v).sum(0) if dtype == "fp16" else 0.0
    return o, size * (2 * d + 2.0 ** -20 + u + n * 2.0 ** -23) + sub + u * np.abs(o) + SMALLEST[dtype]


class Device:
    """Device copies of host arrays, freed together."""

    def __init__(self, hip, make):
        self.hip, self.make = hip, make

    def put(self, a):
        a = np.ascontiguousarray(a)
        d = self.make(max(a.nbytes, 16), zero=False)
        if a.nbytes:
            self.hip.upload(d.ptr, a)
        return d.ptr

    def get(self, ptr, shape, dtype=np.uint16):
        self.hip.sync()
        return self.hip.download(np.empty(shape, dtype), ptr)
