"""The sequence operators at the ends of their range on the GPU: scores, scales and weights of any size, against
definitions in 64 bits."""
import numpy as np
import pytest

import prism_amd as P
from seqlib import HALF_STEP, NAN, SMALLEST, TYPES, Device, normal, to_bits, values, visible

pytestmark = pytest.mark.gpu
KINDS = ["few", "some", "many"]  # workgroups: the three kernels of the sequence attention


@pytest.fixture
def dev(hip, device_arena):
    return Device(hip, device_arena)


def spare(fill):
    """(empty sequences, key rows for each sequence) that lead to the kernels for few, some and many workgroups."""
    return {"few": (0, 400), "some": (165, 400), "many": (1025, 0)}[fill]


def run_seq(engine, dev, dtype, q, k, v, left, right, sinks, scale, fill):
    """One sequence of q [nq][heads][hd] over k, v [nk][kv][hd], and empty ones behind it."""
    nq, heads, hd = q.shape
    nk, kv = k.shape[:2]
    empty, rows = spare(fill)
    seqs = 1 + empty
    more = max(nk, rows * seqs) - nk  # rows of no sequence
    k, v = (np.concatenate([x, np.full((more, kv, hd), NAN[dtype], np.uint16)]) for x in (k, v))
    cu = [dev.put(np.array([0] + [n] * seqs, np.int32)) for n in (nq, nk)]
    out = dev.put(np.full(q.shape, NAN[dtype], np.uint16))
    print(f"[seq] {dtype} {nq} x {nk}, {heads}/{kv} x {hd}, {fill}", flush=True)
    engine.seq_attn(P.SeqAttnPush(
        dtype=TYPES[dtype], n_seqs=seqs, n_q=nq, n_k=len(k), n_heads=heads, n_kv_heads=kv, head_dim=hd, left=left, right=right,
        sinks=sinks, scale=scale, q_token_stride=heads * hd, q_head_stride=hd, k_token_stride=kv * hd, k_head_stride=hd,
        v_token_stride=kv * hd, v_head_stride=hd, out_token_stride=heads * hd, out_head_stride=hd),
        dev.put(q), dev.put(k), dev.put(v), cu[0], cu[1], out)
    return values(dev.get(out, q.shape), dtype)


def run_paged(engine, dev, dtype, q, k, v, scale, max_len, page=16):
    """One sequence: q [heads][hd] over k, v [n][kv][hd] in pages in order."""
    heads, hd = q.shape
    n, kv = k.shape[:2]
    pages = -(-n // page)
    pool = [np.full((pages * page, kv, hd), NAN[dtype], np.uint16) for _ in "kv"]
    pool[0][:n], pool[1][:n] = k, v
    kp, vp = (dev.put(x.reshape(pages, page, kv, hd).transpose(0, 2, 1, 3)) for x in pool)
    out = dev.put(np.full(q.shape, NAN[dtype], np.uint16))
    push = P.PagedAttnPush(
        cache=P.CacheDesc(dtype=TYPES[dtype], n_kv_heads=kv, head_dim=hd, page_size=page, n_pages=pages, n_seqs=1,
                          table_pages=pages), n_heads=heads, left=-1, sinks=0, max_len=max_len, scale=scale,
        q_seq_stride=heads * hd, q_head_stride=hd, out_seq_stride=heads * hd, out_head_stride=hd)
    need = engine.paged_attn_workspace(push)
    ws = dev.put(np.full(need // 2, NAN["fp16"], np.uint16))
    print(f"[paged] {dtype} {heads}/{kv} x {hd}, {n} keys, announced {max_len}", flush=True)
    engine.paged_attn(push, dev.put(q), kp, vp, dev.put(np.arange(pages, dtype=np.int32)), dev.put(np.array([n], np.int32)), out,
                      ws, need)
    return values(dev.get(out, q.shape), dtype)


# --------------------------------------------------------------- huge scores

# q and k have one channel each that is not zero, a power of two and 2^e (128 .. 255), so every score is exact in fp32, and
# so is its product with 1; two unlike scores differ by at least 2^22 (fp16) or 2^32 (bf16), hundreds of steps of fp32 at that
# size, so all the weight is on the keys of the largest score, equally: the output is the mean of their values.
HUGE = {"fp16": (2.0 ** 15, 2.0 ** 7), "bf16": (2.0 ** 20, 2.0 ** 12)}


def huge(rng, dtype, n, heads, kv, hd, queries):
    a, b = HUGE[dtype]
    rank = rng.integers(128, 256, (n, kv))
    sign = np.where(rng.random((queries, heads)) < 0.5, -1, 1)
    q, k = np.zeros((queries, heads, hd)), rng.standard_normal((n, kv, hd))
    q[..., 3] = a * sign
    k[..., 3] = b * rank
    return rank, sign, to_bits(q, dtype), to_bits(k, dtype), normal(rng, (n, kv, hd), dtype)


def largest(rank, sign, v, seen, dtype):
    """The mean of the values of the largest score, and its bound: weights rounded, one sum, one rounding of the output."""
    r = np.where(seen, rank * sign, -1000)
    top = v[r == r.max()]
    o, size = top.mean(0), np.abs(top).mean(0)
    return o, size * (2 * HALF_STEP[dtype] + 2.0 ** -20) + SMALLEST[dtype]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 128])
@pytest.mark.parametrize("kv,group", [(2, 1), (1, 2), (2, 3), (1, 17)])
@pytest.mark.parametrize("n,max_len", [(1, 1), (50, 16), (300, 300), (5000, 5000)])
def test_paged_huge_scores(engine, dev, dtype, hd, kv, group, n, max_len):
    """Scores of 2^30 (fp16) and 2^40 (bf16), where a step of fp32 is many powers of two: the largest takes all."""
    rng = np.random.default_rng(hd + group + n)
    rank, sign, q, k, v = huge(rng, dtype, n, kv * group, kv, hd, 1)
    got = run_paged(engine, dev, dtype, q[0], k, v, 1.0, max_len)
    for h in range(kv * group):
        want, bound = largest(rank[:, h // group], sign[0, h], values(v[:, h // group], dtype), np.ones(n, bool), dtype)
        assert (np.abs(got[h] - want) <= bound).all(), h


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("kv,group,left", [(2, 1, -1), (1, 3, 60)])
@pytest.mark.parametrize("fill", KINDS)
def test_seq_huge_scores(engine, dev, dtype, hd, kv, group, left, fill):
    rng = np.random.default_rng(hd + group)
    n, sinks = 300, 3
    rank, sign, q, k, v = huge(rng, dtype, n, kv * group, kv, hd, n)
    got = run_seq(engine, dev, dtype, q, k, v, left, 0, sinks, 1.0, fill)
    for h in range(kv * group):
        vv = values(v[:, h // group], dtype)
        for i in range(n):
            want, bound = largest(rank[:, h // group], sign[i, h], vv, visible(i, n, left, 0, sinks), dtype)
            assert (np.abs(got[i, h] - want) <= bound).all(), (i, h)


# ----------------------------------------------- one key before many weak ones

# Scores are exact: q is 1 in one channel, the strong key's is `ahead`, every other key's 0, scale = log(2); so the strong key
# weighs 1 and each other 2^-ahead, off by what ahead log2(e) ln(2) is rounded by (2^-24 of it, three times) and exp2's 2^-20.
# The strong key's value is 0, the others' are between 1 and 2: what is lost of the weak weights is not hidden by anything.

def behind_one_key(dtype, ahead, n, hd, at, rng):
    k, v = np.zeros((n, 1, hd)), 1 + rng.random((n, 1, hd))
    k[at, 0, 5], v[at] = ahead, 0
    v = to_bits(v, dtype)
    x = values(v[:, 0], dtype)
    w = 2.0 ** -float(ahead)
    total = 1 + (n - 1) * w
    mean = w * x.sum(0) / total
    # every weight: 2^-20 for exp2, 3 ahead 2^-24 for its argument; n 2^-23 for the sums of weights and products
    bound = mean * (2 * (2.0 ** -20 + 3 * ahead * 2.0 ** -24) + n * 2.0 ** -23 + HALF_STEP[dtype]) + SMALLEST[dtype]
    return to_bits(k, dtype), v, mean, bound, x.sum(0) / total


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 128])
@pytest.mark.parametrize("group", [1, 3, 17])
@pytest.mark.parametrize("n,ahead,max_len", [(131_075, 25.5, 131_075), (20_001, 26, 16), (131_075, 30, 300)])
@pytest.mark.parametrize("last", [False, True])
def test_paged_many_weak_keys_behind_one(engine, dev, dtype, hd, group, n, ahead, max_len, last):
    """The weak keys together weigh as the sum says, however many heads share a key head."""
    k, v, mean, bound, weak = behind_one_key(dtype, ahead, n, hd, n - 1 if last else 0, np.random.default_rng(hd))
    q = np.zeros((group, hd))
    q[:, 5] = 1
    got = run_paged(engine, dev, dtype, to_bits(q, dtype), k, v, np.log(2.0), max_len, page=64)
    # weights meet the values as the sum of two 16-bit numbers: a step of one step at most, (2 u)^2, and fp16's
    # smallest step 2^-24 of numbers of which the largest is 2^14 at least
    two = 4 * mean * HALF_STEP[dtype] ** 2 + (2.0 ** -38 * weak if dtype == "fp16" else 0)
    for h in range(group):
        assert (np.abs(got[h] - mean) <= bound + two).all(), (h, np.abs(got[h] - mean).max(), mean.max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [1, 2, 3, 17])
@pytest.mark.parametrize("pairs,max_len", [(20, 16), (300, 600), (2000, 4000)])
def test_paged_weights_are_not_rounded_to_16_bits(engine, dev, dtype, group, pairs, max_len):
    """Two kinds of keys, one of weight 2^-a (another a for every head), whose values cancel but for the rounding of that
    weight to 16 bits: the output is that rounding, and a kernel that rounds the weight gives 0."""
    rng = np.random.default_rng(group)
    hd, n = 32, 2 * pairs
    a = values(to_bits(np.linspace(0.03, 0.97, group), dtype), dtype)
    k, v, q = np.zeros((n, 1, hd)), np.ones((n, 1, hd)), np.zeros((group, hd))
    other = rng.permutation(n) < pairs
    k[other, 0, 0] = -1
    q[:, 0] = a
    v[~other, 0, :group] = -values(to_bits(2.0 ** -a, dtype), dtype)  # head h's in channel h
    got = run_paged(engine, dev, dtype, to_bits(q, dtype), to_bits(k, dtype), to_bits(v, dtype), np.log(2.0), max_len)
    v = values(to_bits(v, dtype), dtype)[:, 0]
    for h in range(group):
        w = np.where(other, 2.0 ** -a[h], 1.0)
        want, size = w @ v / w.sum(), w @ np.abs(v) / w.sum()
        # 2^-20 for exp2 and 3 2^-24 for its argument, twice; the sums; the weight as two 16-bit numbers, a step of one
        # step at most; one rounding of the output
        bound = size * (2 * (2.0 ** -20 + 3 * 2.0 ** -24) + n * 2.0 ** -23 + 4 * HALF_STEP[dtype] ** 2) + \
            HALF_STEP[dtype] * np.abs(want) + SMALLEST[dtype]
        assert (np.abs(got[h] - want) <= bound).all(), (h, np.abs(got[h] - want).max())


@pytest.mark.parametrize("dtype,bits", [("fp16", 0x7C00), ("bf16", 0x7F80)])
@pytest.mark.parametrize("group", [1, 3])
@pytest.mark.parametrize("n,max_len", [(1, 1), (1, 40), (40, 16), (700, 700), (3000, 3000)])
def test_paged_infinite_values(engine, dev, dtype, bits, group, n, max_len):
    """An infinite value makes its channel infinite and no other."""
    rng = np.random.default_rng(n)
    hd = 64
    q, k, v = normal(rng, (group, hd), dtype), normal(rng, (n, 1, hd), dtype), normal(rng, (n, 1, hd), dtype)
    clean = run_paged(engine, dev, dtype, q, k, v, 0.125, max_len)
    v[n // 2, 0, 7], v[n - 1, 0, 8] = bits, bits | 0x8000
    got = run_paged(engine, dev, dtype, q, k, v, 0.125, max_len)
    assert np.isposinf(got[:, 7]).all() and np.isneginf(got[:, 8]).all()
    rest = np.delete(np.arange(hd), [7, 8])
    assert (got[:, rest] == clean[:, rest]).all()


@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("n,ahead", [(131_075, 25.5), (100_000, 27)])
@pytest.mark.parametrize("last", [False, True])
@pytest.mark.parametrize("fill", ["few", "some", "many"])
def test_seq_many_weak_keys_behind_one(engine, dev, hd, n, ahead, last, fill):
    """fp16: weights below 2^-25 of the largest are not lost."""
    dtype = "fp16"
    k, v, mean, bound, weak = behind_one_key(dtype, ahead, n, hd, n - 1 if last else 0, np.random.default_rng(hd))
    q = np.zeros((3, 1, hd))
    q[..., 5] = 1
    got = run_seq(engine, dev, dtype, to_bits(q, dtype), k, v, -1, -1, 0, np.log(2.0), fill)
    # weights are rounded to half a step, and to fp16's smallest half step 2^-25 of numbers of which the largest is 2^7 at least;
    # their sum may be that of the rounded ones
    one = mean * HALF_STEP[dtype] + 2.0 ** -32 * weak
    for i in range(3):
        assert (np.abs(got[i, 0] - mean) <= bound + 2 * one).all(), (i, np.abs(got[i, 0] - mean).max(), mean.max())


# --------------------------------------------------------------- tiny scales

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [1e-38, 1e-40, 2e-38])
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("left,right,sinks", [(40, 0, 2), (9, -1, 0), (9, 400, 0)])
@pytest.mark.parametrize("fill", KINDS)
def test_seq_tiny_scale(engine, dev, dtype, scale, hd, left, right, sinks, fill):
    """Any positive scale: at 1e-38 all weights are alike, and the output is the mean of the values seen. (With a window of 9,
    rows of one wave begin to see keys in different steps.)"""
    rng = np.random.default_rng(hd)
    n = 330
    q, k, v = (normal(rng, (n, 1, hd), dtype) for _ in "qkv")
    got = run_seq(engine, dev, dtype, q, k, v, left, right, sinks, scale, fill)
    x = values(v[:, 0], dtype)
    for i in range(n):
        seen = x[visible(i, n, left, right, sinks)]
        want, size, u = seen.mean(0), np.abs(seen).mean(0), HALF_STEP[dtype]
        # scores below 2^-110; sums; the weights' rounding; one of the output
        bound = size * (2.0 ** -20 + n * 2.0 ** -23 + 2 * u) + u * np.abs(want) + SMALLEST[dtype]
        assert (np.abs(got[i, 0] - want) <= bound).all(), i


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [1, 3])
@pytest.mark.parametrize("n,max_len", [(30, 30), (700, 700), (3000, 3000)])
def test_paged_tiny_scale(engine, dev, dtype, group, n, max_len):
    rng = np.random.default_rng(n)
    q, k, v = normal(rng, (group, 64), dtype), normal(rng, (n, 1, 64), dtype), normal(rng, (n, 1, 64), dtype)
    got = run_paged(engine, dev, dtype, q, k, v, 1e-40, max_len)
    x, u = values(v[:, 0], dtype), HALF_STEP[dtype]
    bound = np.abs(x).mean(0) * (2.0 ** -20 + n * 2.0 ** -23 + 2 * u) + u * np.abs(x.mean(0)) + SMALLEST[dtype]
    assert (np.abs(got - x.mean(0)) <= bound).all()


# ----------------------------------------------- weights of zero, large values

@pytest.mark.parametrize("dtype,small,large,ahead", [("fp16", 2.0 ** -12, 60_000.0, 70), ("bf16", 1.0, 2.0 ** 100, 240)])
@pytest.mark.parametrize("group", [1, 3])
@pytest.mark.parametrize("n,max_len", [(40, 16), (700, 700), (70_000, 70_000)])
def test_paged_large_values_without_weight(engine, dev, dtype, small, large, ahead, group, n, max_len):
    """Keys `ahead` powers of two behind one: their values, however large, add nothing (n 2^-ahead large < small 2^-20). Their
    sum stays in fp32's range, which a part of the keys without the strong one needs."""
    hd, at = 64, n // 3
    q, k, v = np.zeros((group, hd)), np.zeros((n, 1, hd)), np.full((n, 1, hd), large)
    q[:, 5], k[at, 0, 5], v[at] = 1, ahead, small
    got = run_paged(engine, dev, dtype, to_bits(q, dtype), to_bits(k, dtype), to_bits(v, dtype), np.log(2.0), max_len)
    assert n * 2.0 ** -ahead * large < small * 2.0 ** -20
    assert (np.abs(got - small) <= small * (2.0 ** -19 + HALF_STEP[dtype])).all(), np.abs(got - small).max()


@pytest.mark.parametrize("dtype,small,large,ahead", [("fp16", 2.0 ** -12, 60_000.0, 70), ("bf16", 1.0, 2.0 ** 100, 240)])
@pytest.mark.parametrize("hd", [16, 64, 128])
@pytest.mark.parametrize("fill", KINDS)
def test_seq_large_values_without_weight(engine, dev, dtype, small, large, ahead, hd, fill):
    n, at = 20_000, 7
    q, k, v = np.zeros((3, 1, hd)), np.zeros((n, 1, hd)), np.full((n, 1, hd), large)
    q[..., 5], k[at, 0, 5], v[at] = 1, ahead, small
    got = run_seq(engine, dev, dtype, to_bits(q, dtype), to_bits(k, dtype), to_bits(v, dtype), -1, -1, 0, np.log(2.0), fill)
    assert (np.abs(got - small) <= small * (2.0 ** -19 + 2 * HALF_STEP[dtype])).all(), np.abs(got - small).max()
