"""The 4-bit cache and linear attention on the GPU, through the C ABI, against their definitions in 64 bits (memlib.py).
Outputs start as NaN, so every value has to be written; what must not be used is NaN as well."""
import math

import numpy as np
import pytest

import prism_amd as P
from memlib import Cache, linear, quantise, turned
from seqlib import HALF_STEP, NAN, SMALLEST, TYPES, Device, attention_row, normal, to_bits, values, visible

pytestmark = pytest.mark.gpu
MAX = 2 ** 31 - 1


@pytest.fixture
def dev(hip, device_arena):
    return Device(hip, device_arena)


def outside(got, want, bound):
    """The worst excess over the bound, for a message."""
    off = np.abs(got - want)
    bad = ~(off <= bound)
    return "" if not bad.any() else f"{bad.sum()} values off, worst {np.nanmax(np.where(bad, off, 0)):.3g}, first at {np.argwhere(bad)[0]}"


# ---------------------------------------------------- turned into the cache

def append(engine, dev, cache, rows, heads, seq, at, pos, pairs, layout, ladder, base=10000.0, in_place=False):
    """rows [n][heads + 2 kv][hd] 16 bits; returns q_out (the whole rows if in place) and the call's pages."""
    n, hd, kv = len(rows), cache.hd, cache.kv
    row = rows.shape[1] * hd
    x, pages = dev.put(rows), cache.put(dev)
    q_out = x if in_place else dev.put(np.full((n, max(heads, 1), hd), NAN[cache.dtype], np.uint16))
    push = P.RopeAppendPush(
        cache=cache.desc(), format=P.CACHE_4 if cache.four else P.CACHE_16, n_new=n, n_heads=heads, n_axes=len(pairs),
        pairs=pairs + (0,) * (4 - len(pairs)), layout=layout, ladder=ladder, base=base, q_token_stride=row, q_head_stride=hd,
        k_token_stride=row, k_head_stride=hd, v_token_stride=row, v_head_stride=hd,
        out_token_stride=row if in_place else heads * hd, out_head_stride=hd, pos_stride=pos.shape[1])
    engine.rope_append(push, x if heads else None, x + 2 * heads * hd, x + 2 * (heads + kv) * hd,
                       dev.put(pos) if len(pairs) else None, q_out if heads else None, dev.put(seq), dev.put(at),
                       dev.put(cache.table), pages)
    return dev.get(q_out, rows.shape if in_place else (n, max(heads, 1), hd)), pages


def same_blocks(codes, scales, x, bound, dtype):
    """Whether 4-bit rows are those of x, or of values as far off as bound allows."""
    ok = np.zeros(scales.shape, bool)
    for shift in (0.0, -1.0, 1.0):
        c, s = quantise((x + shift * bound).astype(np.float32), dtype)
        one = c.reshape(s.shape + (-1,)) == codes.reshape(s.shape + (-1,))
        ok |= (s == scales) & one.all(-1)
    return ok.all()


SHAPES = [  # tokens of each sequence, query heads, key heads, hd, pairs, page
    ([1], 8, 8, 32, (4, 6, 6), 16), ([0, 3, 1, 17], 1, 1, 16, (1, 0, 2), 1), ([5, 33, 2], 6, 3, 64, (9, 11, 12), 4),
    ([70, 9], 8, 2, 128, (12, 18, 18), 64), ([21, 4], 0, 5, 32, (3, 4, 2), 16), ([300, 1], 3, 3, 128, (11, 13, 31), 128),
    ([40, 40], 2, 1, 16, (8,), 16), ([9], 40, 40, 64, (8, 8, 8, 8), 2), ([130], 1, 1, 64, (), 32),
]


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", [P.ROPE_HALVES, P.ROPE_ADJACENT])
@pytest.mark.parametrize("lens,heads,kv,hd,pairs,page", SHAPES)
def test_rope_append_and_read(engine, dev, four, dtype, layout, lens, heads, kv, hd, pairs, page):
    rng = np.random.default_rng(sum(lens) + hd + heads)
    cache = Cache(rng, [n + 2 for n in lens], kv, hd, page, dtype, four)
    n = len(lens)
    cache.table[-1, -2] = cache.k.shape[0]  # the last sequence's last page is not in the pool
    seq = np.repeat(np.arange(n), lens)
    at = np.concatenate([np.arange(x) for x in lens])
    seq = np.concatenate([seq, [-1, n, MAX, 0, 0, 0, -2 ** 31]]).astype(np.int32)
    at = np.concatenate([at, [0, 0, 0, -1, cache.table.shape[1] * page, MAX, 0]]).astype(np.int32)
    mix = rng.permutation(len(seq))
    seq, at = seq[mix], at[mix]
    ladder = hd // 16 % 2
    rows = normal(rng, (len(seq), heads + 2 * kv, hd), dtype)
    pos = rng.integers(-50, 200_000, (max(len(pairs), 1), len(seq) + 3)).astype(np.int32)
    pos[0, 0], pos[-1, -4] = -2 ** 31, MAX
    print(f"[rope append] {dtype} 4 bits {four} layout {layout} {len(seq)} x {heads} + 2 x {kv} x {hd} {pairs}", flush=True)
    got, pages = append(engine, dev, cache, rows, heads, seq, at, pos, pairs, layout, ladder)
    x = values(rows, dtype)
    y, bound = turned(x[:, :heads + kv], pos, pairs, layout, ladder, 10000.0, 64 if four else 32)
    if heads:
        b = turned(x[:, :heads + kv], pos, pairs, layout, ladder, 10000.0, 32)[1] + HALF_STEP[dtype] * np.abs(y) + SMALLEST[dtype]
        assert not outside(values(got, dtype), y[:, :heads], b[:, :heads])
        assert (got[..., 2 * sum(pairs):] == rows[:, :heads, 2 * sum(pairs):]).all()  # copied bits
    pools = cache.got(dev)
    seen = 0
    for i in range(len(seq)):
        place = cache.place(seq[i], at[i])
        if place is None:
            continue
        p, slot = place
        seen += 1
        k, kb = y[i, heads:], bound[i, heads:]
        cache.write(seq[i], at[i], k, x[i, heads + kv:])  # values and the other slots exactly, keys within a rounding
        if four:
            assert same_blocks(pools[0][p, :, slot], pools[2][p, :, slot], k, kb, dtype)
            cache.k[p, :, slot], cache.ks[p, :, slot] = pools[0][p, :, slot], pools[2][p, :, slot]
        else:
            assert not outside(values(pools[0][p, :, slot], dtype), k, kb + HALF_STEP[dtype] * np.abs(k) + SMALLEST[dtype])
            cache.k[p, :, slot] = pools[0][p, :, slot]
    assert (seen > 0 or n == 1) and all((a == b).all() for a, b in zip(pools, (cache.k, cache.v, cache.ks, cache.vs)))

    # read back, in another order, into wider rows; zeros where there is nothing
    mix = rng.permutation(len(seq))
    wide = dev.put(np.full((len(seq), 2 * kv + 1, hd), NAN[dtype], np.uint16))
    row = (2 * kv + 1) * hd
    engine.cache_read(P.CacheReadPush(cache=cache.desc(), format=P.CACHE_4 if four else P.CACHE_16, n_rows=len(seq),
                                      k_token_stride=row, k_head_stride=hd, v_token_stride=row, v_head_stride=hd),
                      pages, dev.put(seq[mix]), dev.put(at[mix]), dev.put(cache.table), wide, wide + 2 * kv * hd)
    back = dev.get(wide, (len(seq), 2 * kv + 1, hd))
    assert (back[:, 2 * kv] == NAN[dtype]).all()
    for i, j in enumerate(mix):
        if cache.place(seq[j], at[j]) is None:
            assert (back[i, :2 * kv] == 0).all()
        else:
            k, v = cache.read(seq[j], at[j])
            assert (values(back[i, :kv], dtype) == k).all() and (values(back[i, kv:2 * kv], dtype) == v).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 64])
def test_blocks_at_their_borders(engine, dev, dtype, hd):
    """Values on and beside every border between 4-bit values and between powers, the type's ends, blocks of zeros, with
    infinities and with NaN: the bytes of the definition."""
    rng = np.random.default_rng(hd)
    marks = np.array([0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7])
    marks = np.concatenate([marks, -marks])
    rows = []
    for power in (-30, -24, -23, -16, -14, -3, 0, 4, 12, 13) if dtype == "fp16" else (-133, -126, -125, -124, -3, 0, 90, 124, 125):
        with np.errstate(over="ignore"):
            base = to_bits(marks * 2.0 ** power, dtype)
        for step in (-1, 0, 1):  # the neighbours of each in the type
            bits = np.where(base & 0x7FFF, base.astype(np.int32) + step, base).astype(np.uint16)
            bits = bits[np.isfinite(values(bits, dtype))]
            rows += [rng.choice(bits, hd) for _ in range(4)]
    for top in (0x7BFF, 0x0001, 0x0400) if dtype == "fp16" else (0x7F7F, 0x0001, 0x0080):
        rows += [np.where(rng.random(hd) < 0.3, top, 0x8000).astype(np.uint16)]
    rows += [np.zeros(hd, np.uint16), np.full(hd, 0x8000, np.uint16)]
    inf = 0x7C00 if dtype == "fp16" else 0x7F80
    for bad in (inf, inf | 0x8000, NAN[dtype]):
        row = to_bits(rng.standard_normal(hd), dtype)
        row[hd // 2 + 3] = bad
        rows.append(row)
    v = np.stack(rows)[:, None]
    n = len(v)
    cache = Cache(rng, [n], 1, hd, 8, dtype, True)
    both = np.concatenate([v[::-1], v], 1)
    got, pages = append(engine, dev, cache, both, 0, np.zeros(n, np.int32), np.arange(n, dtype=np.int32),
                        np.zeros((1, n), np.int32), (), 0, 0)
    for i in range(n):
        cache.write(0, i, values(both[i, :1], dtype), values(both[i, 1:], dtype))
    for name, a, b in zip(("k", "v", "k scales", "v scales"), cache.got(dev), (cache.k, cache.v, cache.ks, cache.vs)):
        assert (a == b).all(), name
    out = dev.put(np.zeros((n, 2, hd), np.uint16))
    engine.cache_read(P.CacheReadPush(cache=cache.desc(), format=P.CACHE_4, n_rows=n, k_token_stride=2 * hd, k_head_stride=hd,
                                      v_token_stride=2 * hd, v_head_stride=hd), pages, dev.put(np.zeros(n, np.int32)),
                      dev.put(np.arange(n, dtype=np.int32)), dev.put(cache.table), out, out + 2 * hd)
    back = values(dev.get(out, (n, 2, hd)), dtype)
    for i in range(n):
        for a, b in zip(back[i], cache.read(0, i)):
            assert np.array_equal(a, b[0], equal_nan=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", [P.ROPE_HALVES, P.ROPE_ADJACENT])
@pytest.mark.parametrize("heads,kv,hd,pairs", [(8, 2, 128, (20, 23)), (3, 1, 32, (5,)), (5, 5, 16, (4, 4)), (2, 1, 64, (16, 16))])
def test_rope_append_in_place_is_prism_rope(engine, dev, dtype, layout, heads, kv, hd, pairs):
    """Queries in place, and keys in a 16-bit cache, are prism_rope's within its fp32 angles; the rest of the rows stays."""
    rng = np.random.default_rng(hd)
    n = 37
    cache = Cache(rng, [n], kv, hd, 16, dtype, False)
    rows = normal(rng, (n, heads + 2 * kv, hd), dtype)
    pos = rng.integers(0, 5000, (len(pairs), n)).astype(np.int32)
    got, _ = append(engine, dev, cache, rows, heads, np.zeros(n, np.int32), np.arange(n, dtype=np.int32), pos, pairs, layout, 1,
                    in_place=True)
    assert (got[:, heads:] == rows[:, heads:]).all()
    row = (heads + 2 * kv) * hd
    x, y = dev.put(rows), dev.put(np.full((n, heads + kv, hd), NAN[dtype], np.uint16))
    engine.rope(P.RopePush(dtype=TYPES[dtype], n_tokens=n, n_heads=heads + kv, head_dim=hd, n_axes=len(pairs),
                           pairs=pairs + (0,) * (4 - len(pairs)), layout=layout, ladder=1, inverse=0, base=10000.0,
                           in_token_stride=row, in_head_stride=hd, out_token_stride=(heads + kv) * hd, out_head_stride=hd,
                           pos_stride=n), x, dev.put(pos), y)
    want = values(dev.get(y, (n, heads + kv, hd)), dtype)
    k, slots = cache.got(dev)[0], [cache.place(0, j) for j in range(n)]
    mine = np.concatenate([values(got[:, :heads], dtype), np.stack([values(k[p, :, s], dtype) for p, s in slots])], 1)
    # angles in fp32: 2 pi 2^-25 + 2^-21 of the pair, then a rounding each
    size = np.abs(values(rows[:, :heads + kv], dtype)).max(-1, keepdims=True) * 2
    assert not outside(mine, want, size * (2 * np.pi * 2.0 ** -25 + 2.0 ** -21) + 2 * HALF_STEP[dtype] * np.abs(want) + SMALLEST[dtype])


# ------------------------------------------- a token against a cache of 4 bits

def run_paged4(engine, dev, cache, q, lengths, left, sinks, scale, max_len, guard=2):
    n, heads, hd = q.shape
    out = dev.put(np.full((n + guard, heads, hd), NAN[cache.dtype], np.uint16))
    push = P.PagedAttnPush(cache=cache.desc(), n_heads=heads, left=left, sinks=sinks, max_len=max_len, scale=scale,
                           q_seq_stride=heads * hd, q_head_stride=hd, out_seq_stride=heads * hd, out_head_stride=hd)
    need = engine.paged_attn4_workspace(push)
    ws = dev.put(np.full(max(need, 16) // 2, NAN["fp16"], np.uint16))
    engine.paged_attn4(push, dev.put(q), cache.put(dev), dev.put(cache.table), dev.put(np.array(lengths, np.int32)), out, ws, need)
    got = dev.get(out, (n + guard, heads, hd))
    assert (got[n:] == NAN[cache.dtype]).all()  # rows behind the last sequence
    return values(got[:n], cache.dtype)


def check_paged4(engine, dev, rng, dtype, hd, kv, group, page, lengths, left, sinks, max_len=None, q=None, big=1.0, lost=()):
    """lost: (sequence, page of it) that are not in the pool."""
    cache = Cache(rng, lengths, kv, hd, page, dtype, True)
    heads, scale = kv * group, 1 / math.sqrt(hd)
    q = normal(rng, (len(lengths), heads, hd), dtype) if q is None else q
    sees = []
    for s, n in enumerate(lengths):
        seen = visible(n - 1, n, left, 0, sinks)
        js = np.flatnonzero(seen)  # the others' blocks stay NaN
        cache.fill(s, js, rng.standard_normal((len(js), kv, hd)) * big, rng.standard_normal((len(js), kv, hd)))
        for j in range(-(-n // page)):
            if not seen[j * page:(j + 1) * page].any():
                cache.table[s, j] = -1
        sees.append(seen)
    want, bound = np.zeros(q.shape), np.zeros(q.shape)
    qv = values(q, dtype)
    for s, seen in enumerate(sees):
        for a, j in lost:
            if a == s:
                seen[j * page:(j + 1) * page] = False
        js = np.flatnonzero(seen)
        k, v = cache.rows(s, js)
        for h in range(heads):
            want[s, h], bound[s, h] = attention_row(qv[s, h], k[:, h // group], v[:, h // group], np.ones(len(js), bool), scale, dtype)
    for s, j in lost:
        cache.table[s, j] = cache.k.shape[0] + 5
    print(f"[paged4] {dtype} {heads}/{kv} x {hd} pages of {page} lengths {lengths} left {left} sinks {sinks}", flush=True)
    got = run_paged4(engine, dev, cache, q, lengths, left, sinks, scale, max(lengths) if max_len is None else max_len)
    assert not outside(got, want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,kv,group", [(16, 8, 1), (16, 1, 40), (32, 8, 1), (32, 3, 2), (32, 2, 5), (64, 3, 1), (64, 2, 4),
                                         (64, 1, 17), (128, 2, 1), (128, 1, 2), (128, 2, 4), (128, 1, 33)])
def test_paged4_shapes(engine, dev, dtype, hd, kv, group):
    rng = np.random.default_rng(hd + group)
    check_paged4(engine, dev, rng, dtype, hd, kv, group, 16, [1, 2, 15, 16, 17, 31, 33, 64, 65, 100, 0], -1, 0)


@pytest.mark.parametrize("group", [1, 2, 4])
@pytest.mark.parametrize("page,left,sinks", [(1, 5, 3), (16, 0, 0), (4, 20, 0), (64, 31, 40), (32, 17, 1), (16, MAX, MAX), (2, 200, 7)])
def test_paged4_windows(engine, dev, page, left, sinks, group):
    rng = np.random.default_rng(page)
    check_paged4(engine, dev, rng, "fp16", 32, 2, group, page, [1, 3, 22, 64, 90, 131], left, sinks)


@pytest.mark.parametrize("dtype,hd,kv,group,lengths,max_len", [
    ("fp16", 128, 1, 1, [3001, 5], 3001), ("bf16", 128, 1, 4, [2500, 700, 1], 0), ("bf16", 64, 1, 2, [4099], 4099),
    ("fp16", 32, 2, 1, [3333, 100], 3333), ("fp16", 64, 1, 8, [2100, 2099], 2100), ("bf16", 16, 1, 3, [3000], 3000),
    ("fp16", 128, 1, 2, [1500, 40], 30),
])
def test_paged4_long(engine, dev, dtype, hd, kv, group, lengths, max_len):
    rng = np.random.default_rng(hd)
    check_paged4(engine, dev, rng, dtype, hd, kv, group, 64, lengths, -1, 0, max_len)


def test_paged4_long_window_and_sinks(engine, dev):
    check_paged4(engine, dev, np.random.default_rng(4), "fp16", 128, 1, 4, 32, [3000, 1200], 1100, 33)


@pytest.mark.parametrize("group", [1, 4])
def test_paged4_sharp_scores(engine, dev, group):
    check_paged4(engine, dev, np.random.default_rng(5), "bf16", 64, 2, group, 16, [200, 77], -1, 0, big=40.0)


@pytest.mark.parametrize("hd", [16, 128])
@pytest.mark.parametrize("group", [1, 2, 3])
def test_paged4_pages_out_of_the_pool(engine, dev, hd, group):
    check_paged4(engine, dev, np.random.default_rng(6), "fp16", hd, 2, group, 16, [100, 33, 16], -1, 0, lost=[(0, 2), (0, 6), (2, 0)])


@pytest.mark.parametrize("group", [1, 2, 4])
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
def test_paged4_many_short(engine, dev, hd, group):
    """Waves that work alone: more items than a launch of four waves each takes."""
    rng = np.random.default_rng(7)
    lengths = [int(x) for x in rng.integers(0, 40, 520)]
    check_paged4(engine, dev, rng, "bf16", hd, 8, group, 16, lengths, 30, 2)


@pytest.mark.parametrize("group", [1, 4])
def test_paged4_a_block_of_nan_reaches_its_stream_alone(engine, dev, group):
    rng = np.random.default_rng(8)
    dtype, hd, kv, page, lengths = "fp16", 64, 2, 16, [50, 50, 50]
    cache = Cache(rng, lengths, kv, hd, page, dtype, True)
    for s, n in enumerate(lengths):
        for j in range(n):
            cache.write(s, j, rng.standard_normal((kv, hd)), rng.standard_normal((kv, hd)))
    p, slot = cache.place(1, 20)
    cache.vs[p, 0, slot, 1] = 255  # channels 32.. of key head 0
    q = normal(rng, (3, kv * group, hd), dtype)
    got = run_paged4(engine, dev, cache, q, lengths, -1, 0, 0.125, 50)
    bad = np.zeros(got.shape, bool)
    bad[1, :group, 32:] = True
    assert (np.isnan(got) == bad).all()


# -------------------------------------------------------- linear attention

RATES = np.array([0.0, 0.003, 0.7, np.inf, 0.05, -1.0, 20.0, np.nan], np.float32)


def linear_push(dtype, n, tokens, heads, kv, hd, states, scale, row):
    return P.LinearAttnPush(dtype=TYPES[dtype], n_seqs=n, n_tokens=tokens, n_heads=heads, n_kv_heads=kv, head_dim=hd,
                            n_states=states, scale=scale, q_token_stride=row, q_head_stride=hd, k_token_stride=row,
                            k_head_stride=hd, v_token_stride=row, v_head_stride=hd, out_token_stride=heads * hd,
                            out_head_stride=hd)


def run_linear(engine, dev, dtype, rows, heads, kv, lens, rates, state_of=None, state_in=None, states=0, scale=None, guard=3,
               equal=False, keep_state=True, stream=None):
    """rows [guard + tokens + guard][heads + 2 kv][hd]; returns (out of all rows, states)."""
    total, width, hd = rows.shape
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32) + (0 if equal else guard)
    x, out = dev.put(rows), dev.put(np.full((total, heads, hd), NAN[dtype], np.uint16))
    push = linear_push(dtype, len(lens), total, heads, kv, hd, states, hd ** -0.5 if scale is None else scale, width * hd)
    need = engine.linear_attn_workspace(push)
    ws = dev.put(np.full(max(need, 16) // 4, np.nan, np.float32))
    new = dev.put(np.full((max(states, 1), heads, hd, hd), np.nan, np.float32))
    engine.linear_attn(push, x, x + 2 * heads * hd, x + 2 * (heads + kv) * hd, dev.put(rates), None if equal else dev.put(cu),
                       None if state_of is None else dev.put(state_of), None if state_in is None else dev.put(state_in), out,
                       new if keep_state else None, ws if need else None, need, stream)
    return dev.get(out, (total, heads, hd)), dev.get(new, (max(states, 1), heads, hd, hd), np.float32)


def check_linear(engine, dev, rng, dtype, hd, kv, group, lens, start="all", scale=None, equal=False, big=1.0, rates=RATES):
    heads, n, guard = kv * group, len(lens), 0 if equal else 3
    total = sum(lens) + 2 * guard
    rows = to_bits(rng.standard_normal((total, heads + 2 * kv, hd)) * big, dtype)
    if guard:
        rows[:guard], rows[-guard:] = NAN[dtype], NAN[dtype]
    rates = np.resize(rates, heads)
    states = n + 2
    state_of = rng.permutation(states)[:n].astype(np.int32)
    if n > 2:
        state_of[1], state_of[2] = -1, states
    s0 = (rng.standard_normal((states, heads, hd, hd)) * 3).astype(np.float32) if start == "all" else None
    print(f"[linear] {dtype} {heads}/{kv} x {hd} lengths {lens} start {start}", flush=True)
    got, new = run_linear(engine, dev, dtype, rows, heads, kv, lens, rates, state_of, s0, states, scale, guard, equal)
    x, at = values(rows, dtype), guard
    assert (got[:guard] == NAN[dtype]).all() and (got[total - guard:] == NAN[dtype]).all()
    untouched = np.ones(states, bool)
    for s, ln in enumerate(lens):
        num = state_of[s] if 0 <= state_of[s] < states else None
        for h in range(heads):
            first = np.zeros((hd, hd)) if num is None or s0 is None else s0[num, h].astype(np.float64)
            part = x[at:at + ln]
            o, b, S, B = linear(part[:, h], part[:, heads + h // group], part[:, heads + kv + h // group], float(rates[h]), first,
                                hd ** -0.5 if scale is None else scale, dtype)
            assert not outside(values(got[at:at + ln, h], dtype), o, b), (s, h, rates[h])
            if num is not None:
                untouched[num] = False
                assert not outside(new[num, h].astype(np.float64), S, B), (s, h, rates[h])
                if ln == 0:
                    assert (new[num, h] == (0 if s0 is None else s0[num, h])).all()
        at += ln
    assert np.isnan(new[untouched]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,kv,group", [(16, 8, 1), (16, 3, 1), (16, 1, 5), (32, 8, 1), (32, 2, 3), (64, 5, 1), (64, 2, 4),
                                         (128, 4, 1), (128, 1, 8)])
def test_linear_shapes(engine, dev, dtype, hd, kv, group):
    check_linear(engine, dev, np.random.default_rng(hd + kv), dtype, hd, kv, group, [5, 64, 1, 0, 63, 65, 130, 2])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("start", ["all", "none"])
def test_linear_long(engine, dev, dtype, hd, start):
    """Few long sequences: split over their length, where that is done."""
    check_linear(engine, dev, np.random.default_rng(hd), dtype, hd, 2, 1, [1500, 777], start)


@pytest.mark.parametrize("hd", [16, 128])
@pytest.mark.parametrize("rate", [0.0, 0.002])
def test_linear_one_very_long(engine, dev, hd, rate):
    check_linear(engine, dev, np.random.default_rng(3), "bf16", hd, 1, 1, [6001], rates=np.array([rate], np.float32))


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_equal_lengths_and_scales(engine, dev, dtype):
    check_linear(engine, dev, np.random.default_rng(2), dtype, 32, 4, 2, [70, 70, 70], scale=-2.5, equal=True)
    check_linear(engine, dev, np.random.default_rng(2), dtype, 64, 1, 1, [33], scale=0.0, equal=True)


@pytest.mark.parametrize("dtype,big", [("fp16", 2.0 ** -12), ("fp16", 200.0), ("bf16", 2.0 ** -30), ("bf16", 2.0 ** 30)])
def test_linear_small_and_large_values(engine, dev, dtype, big):
    """Products past fp16's range on the way (200^3 sqrt(64) = 2^26; the scale brings outputs back), and values whose
    products are small."""
    check_linear(engine, dev, np.random.default_rng(9), dtype, 64, 2, 1, [200, 65], "none", scale=1 / (big * big * 64), big=big)


def test_linear_many_sequences(engine, dev):
    rng = np.random.default_rng(4)
    check_linear(engine, dev, rng, "fp16", 16, 2, 1, [int(x) for x in rng.integers(0, 9, 300)])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("what,which", [(math.nan, "q"), (math.inf, "k"), (math.nan, "k"), (-math.inf, "v"), (math.nan, "v")])
def test_linear_bad_values_reach_only_what_follows(engine, dev, dtype, hd, what, which):
    rng = np.random.default_rng(hd)
    heads, lens, guard = 2, [100, 140, 90], 3
    total = sum(lens) + 2 * guard
    rows = normal(rng, (total, 3 * heads, hd), dtype)
    rates = np.array([0.01, 0.0], np.float32)
    clean, cs = run_linear(engine, dev, dtype, rows, heads, heads, lens, rates, states=3)
    t, c, h = guard + lens[0] + 75, hd - 3, 1
    rows[t, {"q": h, "k": heads + h, "v": 2 * heads + h}[which], c] = to_bits(np.array(what), dtype)
    got, gs = run_linear(engine, dev, dtype, rows, heads, heads, lens, rates, states=3)
    bad, bad_state = np.zeros(got.shape, bool), np.zeros(gs.shape, bool)
    end = guard + lens[0] + lens[1]
    if which == "q":
        bad[t, h] = True
    elif which == "k":
        bad[t:end, h] = True
        bad_state[1, h, c] = True
    else:
        bad[t:end, h, c] = True
        bad_state[1, h, :, c] = True
    g = values(got, dtype)
    inside = slice(guard, total - guard)
    assert (~np.isfinite(g[inside]) == bad[inside]).all()
    assert (got[~bad] == clean[~bad]).all()
    assert not np.isfinite(gs[bad_state]).any() and (gs[~bad_state] == cs[~bad_state]).all()


# -------------------------------------------------------- a token at a time

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,kv,group,n", [(16, 8, 1, 33), (16, 1, 3, 1), (32, 8, 1, 50), (32, 1, 5, 2), (64, 4, 2, 7), (128, 1, 4, 3),
                                           (128, 3, 1, 1), (64, 1, 1, 300)])
def test_linear_step(engine, dev, dtype, hd, kv, group, n):
    rng = np.random.default_rng(hd + n)
    heads, states = kv * group, n + 3
    rows = normal(rng, (n, heads + 2 * kv, hd), dtype)
    rates, scale = np.resize(RATES, heads), 0.3
    state_of = rng.permutation(states)[:n].astype(np.int32)
    if n > 2:
        state_of[0], state_of[1] = -1, states
    s0 = (rng.standard_normal((states, heads, hd, hd)) * 2).astype(np.float32)
    x, out = dev.put(rows), dev.put(np.full((n + 2, heads, hd), NAN[dtype], np.uint16))
    old, new = dev.put(s0), dev.put(np.full(s0.shape, np.nan, np.float32))
    push = linear_push(dtype, n, n, heads, kv, hd, states, scale, (heads + 2 * kv) * hd)
    args = (x, x + 2 * heads * hd, x + 2 * (heads + kv) * hd, dev.put(rates), dev.put(state_of))
    print(f"[step] {dtype} {n} x {heads}/{kv} x {hd}", flush=True)
    engine.linear_step(push, *args, old, out, new)
    got, gs = dev.get(out, (n + 2, heads, hd)), dev.get(new, s0.shape, np.float32)
    assert (got[n:] == NAN[dtype]).all() and (dev.get(old, s0.shape, np.float32) == s0).all()
    v, touched = values(rows, dtype), np.zeros(states, bool)
    for s in range(n):
        if not 0 <= state_of[s] < states:
            assert (got[s] == 0).all()
            continue
        touched[state_of[s]] = True
        for h in range(heads):
            o, b, S, B = linear(v[s:s + 1, h], v[s:s + 1, heads + h // group], v[s:s + 1, heads + kv + h // group], float(rates[h]),
                                s0[state_of[s], h].astype(np.float64), scale, dtype)
            assert not outside(values(got[s:s + 1, h], dtype), o, b) and not outside(gs[state_of[s], h].astype(np.float64), S, B)
    assert np.isnan(gs[~touched]).all()
    engine.linear_step(push, *args, old, out, old)  # in place: the same bits, and the other states as they were
    assert (dev.get(out, got.shape) == got).all()
    there = dev.get(old, s0.shape, np.float32)
    assert (there[touched] == gs[touched]).all() and (there[~touched] == s0[~touched]).all()


# ------------------------------------------------------- as they are used

@pytest.mark.parametrize("dtype,four,heads,kv,hd", [("fp16", True, 8, 8, 32), ("bf16", True, 8, 2, 128), ("fp16", False, 4, 4, 16)])
def test_streamed_frames_and_the_clip_at_once(engine, dev, dtype, four, heads, kv, hd):
    """rope_append -> one token per stream, frame by frame, against rope_append of the whole clip -> cache_read ->
    attention along the sequences. Cache and queries have the same bits; the attentions differ by their roundings."""
    rng = np.random.default_rng(hd)
    frames, places, page, group, scale = 21, 6, 4, heads // kv, hd ** -0.5
    pairs = (hd // 8, hd // 8, hd // 8)
    rows = normal(rng, (places, frames, heads + 2 * kv, hd), dtype)
    clip, row = rows.reshape(places * frames, -1, hd), (heads + 2 * kv) * hd
    pos = np.stack([np.tile(np.arange(frames), places), np.repeat(np.arange(places) // 3, frames),
                    np.repeat(np.arange(places) % 3, frames)]).astype(np.int32)
    seq, at = np.repeat(np.arange(places), frames).astype(np.int32), np.tile(np.arange(frames), places).astype(np.int32)
    whole = Cache(np.random.default_rng(1), [frames] * places, kv, hd, page, dtype, four)
    turned_q, pages = append(engine, dev, whole, clip, heads, seq, at, pos, pairs, 0, 0)
    fmt = P.CACHE_4 if four else P.CACHE_16
    kv_rows = dev.put(np.full((places * frames, 2 * kv, hd), NAN[dtype], np.uint16))
    engine.cache_read(P.CacheReadPush(cache=whole.desc(), format=fmt, n_rows=len(seq), k_token_stride=2 * kv * hd, k_head_stride=hd,
                                      v_token_stride=2 * kv * hd, v_head_stride=hd), pages, dev.put(seq), dev.put(at),
                      dev.put(whole.table), kv_rows, kv_rows + 2 * kv * hd)
    out = dev.put(np.zeros((places * frames, heads, hd), np.uint16))
    engine.seq_attn(P.SeqAttnPush(
        dtype=TYPES[dtype], n_seqs=places, n_q=len(seq), n_k=len(seq), n_heads=heads, n_kv_heads=kv, head_dim=hd, left=-1, right=0,
        sinks=0, scale=scale, q_token_stride=heads * hd, q_head_stride=hd, k_token_stride=2 * kv * hd, k_head_stride=hd,
        v_token_stride=2 * kv * hd, v_head_stride=hd, out_token_stride=heads * hd, out_head_stride=hd),
        dev.put(turned_q), kv_rows, kv_rows + 2 * kv * hd, None, None, out)
    at_once = values(dev.get(out, (places, frames, heads, hd)), dtype)
    kvr = values(dev.get(kv_rows, (places, frames, 2 * kv, hd)), dtype)
    tq = values(turned_q.reshape(places, frames, heads, hd), dtype)

    stepped = Cache(np.random.default_rng(1), [frames] * places, kv, hd, page, dtype, four)
    for f in range(frames):
        x = np.ascontiguousarray(rows[:, f])
        p = np.ascontiguousarray(pos.reshape(3, places, frames)[:, :, f])
        q, step_pages = append(engine, dev, stepped, x, heads, np.arange(places, dtype=np.int32), np.full(places, f, np.int32), p,
                               pairs, 0, 0)
        assert (q == turned_q.reshape(places, frames, heads, hd)[:, f]).all()
        for a, b in zip(("k", "v", "ks", "vs"), stepped.got(dev)):
            setattr(stepped, a, b)
        push = P.PagedAttnPush(cache=stepped.desc(), n_heads=heads, left=-1, sinks=0, max_len=frames, scale=scale,
                               q_seq_stride=heads * hd, q_head_stride=hd, out_seq_stride=heads * hd, out_head_stride=hd)
        o, lens, table = dev.put(np.zeros((places, heads, hd), np.uint16)), dev.put(np.full(places, f + 1, np.int32)), dev.put(stepped.table)
        if four:
            assert engine.paged_attn4_workspace(push) == 0
            engine.paged_attn4(push, dev.put(q), step_pages, table, lens, o, None, 0)
        else:
            engine.paged_attn(push, dev.put(q), step_pages.k, step_pages.v, table, lens, o, None, 0)
        got = values(dev.get(o, (places, heads, hd)), dtype)
        for s in range(places):
            for h in range(heads):
                want, bound = attention_row(tq[s, f, h], kvr[s, :f + 1, h // group], kvr[s, :f + 1, kv + h // group],
                                            np.ones(f + 1, bool), scale, dtype)
                assert not outside(got[s, h], want, bound) and not outside(at_once[s, f, h], want, bound)
    assert all((a == b).all() for a, b in zip(stepped.got(dev), whole.got(dev)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 128])
def test_a_prompt_then_tokens_one_at_a_time(engine, dev, dtype, hd):
    """linear_attn over a prompt, its states on in linear_step, against linear_attn over all of it."""
    rng = np.random.default_rng(hd)
    n, prompt, more, heads = 3, 70, 5, 2
    rows = normal(rng, (n, prompt + more, 3 * heads, hd), dtype)
    rates = np.array([0.02, 0.3], np.float32)
    head = np.ascontiguousarray(rows[:, :prompt]).reshape(n * prompt, 3 * heads, hd)
    all_rows = rows.reshape(n * (prompt + more), 3 * heads, hd)
    _, state = run_linear(engine, dev, dtype, head, heads, heads, [prompt] * n, rates, states=n, equal=True, guard=0)
    whole, last = run_linear(engine, dev, dtype, all_rows, heads, heads, [prompt + more] * n, rates, states=n, equal=True, guard=0)
    states, out = dev.put(state), dev.put(np.zeros((n, heads, hd), np.uint16))
    push = linear_push(dtype, n, n, heads, heads, hd, n, hd ** -0.5, 3 * heads * hd)
    r = dev.put(rates)
    whole = values(whole.reshape(n, prompt + more, heads, hd), dtype)
    for i in range(more):
        x = dev.put(np.ascontiguousarray(rows[:, prompt + i]))
        engine.linear_step(push, x, x + 2 * heads * hd, x + 4 * heads * hd, r, None, states, out, states)
        got = values(dev.get(out, (n, heads, hd)), dtype)
        for s in range(n):
            for h in range(heads):
                part = values(rows[s, :prompt + i + 1], dtype)
                o, b, S, B = linear(part[:, h], part[:, heads + h], part[:, 2 * heads + h], float(rates[h]), np.zeros((hd, hd)),
                                    hd ** -0.5, dtype)
                assert not outside(got[s, h], o[-1], b[-1]) and not outside(whole[s, prompt + i, h], o[-1], b[-1])
    end = dev.get(states, state.shape, np.float32)
    for s in range(n):
        for h in range(heads):
            part = values(rows[s], dtype)
            S, B = linear(part[:, h], part[:, heads + h], part[:, 2 * heads + h], float(rates[h]), np.zeros((hd, hd)), 1.0, dtype)[2:]
            assert not outside(end[s, h].astype(np.float64), S, B) and not outside(last[s, h].astype(np.float64), S, B)


def test_captured_and_replayed(hip, engine, dev):
    """One graph of the five calls on a stream of its own, replayed on new inputs in the same buffers with eager calls
    in between: the same bits."""
    rng = np.random.default_rng(12)
    n, heads, kv, hd, page, length = 5, 8, 2, 64, 16, 2000
    width, row = -(-length // page), (heads + 2 * kv) * hd
    cache = P.CacheDesc(dtype=P.F16, n_kv_heads=kv, head_dim=hd, page_size=page, n_pages=n * width, n_seqs=n, table_pages=width)
    add = P.RopeAppendPush(cache=cache, format=P.CACHE_4, n_new=n, n_heads=heads, n_axes=2, pairs=(16, 16, 0, 0), layout=0, ladder=0,
                           base=1000.0, q_token_stride=row, q_head_stride=hd, k_token_stride=row, k_head_stride=hd,
                           v_token_stride=row, v_head_stride=hd, out_token_stride=heads * hd, out_head_stride=hd, pos_stride=n)
    one = P.PagedAttnPush(cache=cache, n_heads=heads, left=-1, sinks=0, max_len=length, scale=0.125, q_seq_stride=heads * hd,
                          q_head_stride=hd, out_seq_stride=heads * hd, out_head_stride=hd)
    rows = n * 100
    read = P.CacheReadPush(cache=cache, format=P.CACHE_4, n_rows=rows, k_token_stride=kv * hd, k_head_stride=hd,
                           v_token_stride=kv * hd, v_head_stride=hd)
    lin = linear_push("fp16", 2, rows, kv, kv, hd, 2, 0.125, kv * hd)  # along what was read: queries = keys
    step = linear_push("fp16", n, n, heads, kv, hd, n, 0.125, row)
    need, need2 = engine.paged_attn4_workspace(one), engine.linear_attn_workspace(lin)
    blocks = (n * width, kv, page, hd // 32)
    pool, scales = rng.integers(0, 256, (n * width, kv, page, hd // 2), np.uint8), rng.integers(124, 130, blocks).astype(np.uint8)
    table = dev.put(rng.permutation(n * width).astype(np.int32))
    seq, at, lens = dev.put(np.arange(n, dtype=np.int32)), dev.put(np.full(n, length - 1, np.int32)), dev.put(np.full(n, length, np.int32))
    rseq, rat = dev.put(np.repeat(np.arange(n, dtype=np.int32), 100)), dev.put(np.tile(np.arange(length - 100, length, dtype=np.int32), n))
    cu, rates = dev.put(np.array([0, 177, rows], np.int32)), dev.put(np.resize(np.array([0.01, 0.1], np.float32), heads))

    def buffers():
        return dict(x=dev.put(np.zeros((n, row), np.uint16)), pos=dev.put(np.arange(2 * n, dtype=np.int32)), q=dev.put(np.zeros((n, heads, hd), np.uint16)),
                    pages=P.CachePages(k=dev.put(pool), v=dev.put(pool), k_scales=dev.put(scales), v_scales=dev.put(scales)),
                    a=dev.put(np.zeros((n, heads, hd), np.uint16)), k=dev.put(np.zeros((rows, kv, hd), np.uint16)),
                    v=dev.put(np.zeros((rows, kv, hd), np.uint16)), b=dev.put(np.zeros((rows, kv, hd), np.uint16)),
                    s=dev.put(np.zeros((2, kv, hd, hd), np.float32)), c=dev.put(np.zeros((n, heads, hd), np.uint16)),
                    t=dev.put(np.zeros((n, heads, hd, hd), np.float32)), ws=dev.put(np.zeros(max(need, 16), np.uint8)),
                    ws2=dev.put(np.zeros(max(need2, 16), np.uint8)))

    def calls(d, s):
        k, v = d["x"] + 2 * heads * hd, d["x"] + 2 * (heads + kv) * hd
        engine.rope_append(add, d["x"], k, v, d["pos"], d["q"], seq, at, table, d["pages"], s)
        engine.paged_attn4(one, d["q"], d["pages"], table, lens, d["a"], d["ws"], need, s)
        engine.cache_read(read, d["pages"], rseq, rat, table, d["k"], d["v"], s)
        engine.linear_attn(lin, d["k"], d["k"], d["v"], rates, cu, None, d["s"], d["b"], d["s"], d["ws2"], need2, s)
        engine.linear_step(step, d["x"], k, v, rates, None, d["t"], d["c"], d["t"], s)

    caught, eager, s = buffers(), buffers(), hip.stream()
    hip.sync()
    hip.begin_capture(s)
    calls(caught, s)
    graph = hip.end_capture(s)
    ready = hip.graph_instantiate(graph)
    for _ in range(4):
        x = normal(rng, (n, row), "fp16")
        hip.upload(caught["x"], x)
        hip.upload(eager["x"], x)
        hip.graph_launch(ready, s)
        calls(eager, None)
        hip.stream_sync(s)
        for name, shape, t in (("q", (n, heads, hd), np.uint16), ("a", (n, heads, hd), np.uint16), ("k", (rows, kv, hd), np.uint16),
                               ("b", (rows, kv, hd), np.uint16), ("c", (n, heads, hd), np.uint16), ("s", (2, kv, hd, hd), np.float32),
                               ("t", (n, heads, hd, hd), np.float32)):
            got = dev.get(caught[name], shape, t)
            assert (got == dev.get(eager[name], shape, t)).all() and got.any()
    hip.graph_destroy(graph, ready)


def test_refused_calls(hip, engine, dev):
    """Refusals that need a context; nothing runs."""
    import test_memory_rules as R
    import test_seq_rules as S
    a = dev.put(np.zeros(4096, np.uint16))
    g = P.CachePages(k=a, v=a, k_scales=a, v_scales=a)

    def refused(call, *args):
        with pytest.raises(P.PrismError) as e:
            call(*args)
        assert e.value.code in (P.ERR_INVALID, P.ERR_UNSUPPORTED) and engine.error()

    add = R.rope_append
    refused(engine.rope_append, add(), None, a, a, a, a, a, a, a, g)
    refused(engine.rope_append, add(), a, a, a, None, a, a, a, a, g)
    refused(engine.rope_append, add(), a, a, a, a, a, a, a, None, g)
    refused(engine.rope_append, add(), a, a + 2, a, a, a, a, a, a, g)
    refused(engine.rope_append, add(), a, a, a, a, a, a, a, a, g)  # in place with unequal strides
    refused(engine.rope_append, add(), a, a, a, a, a + 16, a, a, a, P.CachePages(k=a, v=a))
    refused(engine.rope_append, add(), a, a, a, a, a + 16, a, a, a, P.CachePages(k=a, v=a, k_scales=a + 4, v_scales=a))
    refused(engine.rope_append, add(format=P.CACHE_16), a, a, a, a, a + 16, a, a, a, P.CachePages(k=a))
    refused(engine.rope_append, add(format=7), a, a, a, a, a + 16, a, a, a, g)
    refused(engine.cache_read, R.cache_read(), g, a, a, None, a, a)
    refused(engine.cache_read, R.cache_read(), g, a, a, a, a, a + 8)
    refused(engine.cache_read, R.cache_read(), P.CachePages(), a, a, a, a, a)
    refused(engine.paged_attn4, S.paged(), a, P.CachePages(k=a, v=a), a, a, a, a, 1 << 20)
    refused(engine.paged_attn4, S.paged(), None, g, a, a, a, a, 1 << 20)
    refused(engine.paged_attn4, S.paged(), a, P.CachePages(k=a, v=a, k_scales=a, v_scales=a + 8), a, a, a, a, 1 << 20)
    long = S.paged(cache=S.cache(n_seqs=1, table_pages=1000), max_len=16000)
    need = engine.paged_attn4_workspace(long)
    assert need > 0
    refused(engine.paged_attn4, long, a, g, a, a, a, a, need - 1)
    refused(engine.paged_attn4, long, a, g, a, a, a, None, need)
    lin = R.linear
    refused(engine.linear_attn, lin(), a, a, a, None, a, None, None, a, None, None, 0)
    refused(engine.linear_attn, lin(), a, None, a, a, a, None, None, a, None, None, 0)
    refused(engine.linear_attn, lin(), a, a, a, a, a, None, a + 4, a, None, None, 0)
    refused(engine.linear_attn, lin(n_tokens=7), a, a, a, a, None, None, None, a, None, None, 0)  # equal lengths do not fill
    refused(engine.linear_attn, lin(scale=math.nan), a, a, a, a, a, None, None, a, None, None, 0)
    refused(engine.linear_step, lin(), a, a, a, a, None, None, a, a)
    refused(engine.linear_step, lin(), a, a, a, a, None, a, a, None)
    refused(engine.linear_step, lin(n_tokens=10), a, a, a, a, None, a, a, a)


def test_calls_without_rows(engine, dev):
    """Nothing to do is no error, whatever the pointers; without a place in the cache queries still turn, rows read are zeros."""
    import test_memory_rules as R
    none = P.CachePages()
    engine.rope_append(R.rope_append(n_new=0), None, None, None, None, None, None, None, None, none)
    engine.cache_read(R.cache_read(n_rows=0), none, None, None, None, None, None)
    engine.linear_attn(R.linear(n_seqs=0, n_tokens=0), None, None, None, None, None, None, None, None, None, None, 0)
    engine.linear_step(R.linear(n_seqs=0, n_tokens=0), None, None, None, None, None, None, None, None)
    rng = np.random.default_rng(0)
    x, pos, y = normal(rng, (5, 8, 32), "fp16"), np.zeros((3, 5), np.int32), dev.put(np.full((5, 4, 32), NAN["fp16"], np.uint16))
    d = dev.put(x)
    engine.rope_append(R.rope_append(cache=R.cache(n_pages=0)), d, d, d, dev.put(pos), y, None, None, None, none)
    assert (dev.get(y, (5, 4, 32)) == x[:, :4]).all()
    engine.cache_read(R.cache_read(cache=R.cache(n_seqs=0)), none, None, None, None, d, d + 64 * 5 * 2)
    assert (dev.get(d, (5, 4, 32)) == 0).all()
    # sequences of no tokens at all: states come from where they were
    s0 = rng.standard_normal((6, 4, 64, 64)).astype(np.float32)
    new = dev.put(np.full(s0.shape, np.nan, np.float32))
    engine.linear_attn(R.linear(n_tokens=0), None, None, None, dev.put(np.zeros(4, np.float32)), None, None, dev.put(s0), None, new,
                       None, 0)
    got = dev.get(new, s0.shape, np.float32)
    assert (got[:5] == s0[:5]).all() and np.isnan(got[5:]).all()


# ------------------------------------------- calls that the documentation allows

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,lens", [(16, [1500, 777, 0, 3]), (32, [2300, 64]), (64, [777, 1500]), (128, [1900, 300]), (128, [63, 65])])
def test_linear_state_in_place(engine, dev, dtype, hd, lens):
    """state_out = state_in: the same bits, whether a sequence is split or not."""
    rng, heads, n = np.random.default_rng(hd), 3, len(lens)
    rows = normal(rng, (sum(lens), 3 * heads, hd), dtype)
    s0 = rng.standard_normal((n, heads, hd, hd)).astype(np.float32)
    push = linear_push(dtype, n, sum(lens), heads, heads, hd, n, 0.1, 3 * heads * hd)
    need = engine.linear_attn_workspace(push)
    assert (need > 0) == (max(lens) > 256)
    x, rates = dev.put(rows), dev.put(np.array([0.0, 0.001, 0.3], np.float32))
    cu = dev.put(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))

    def run(old, new):
        out, ws = dev.put(np.full((sum(lens), heads, hd), NAN[dtype], np.uint16)), dev.put(np.full(max(need, 16) // 4, np.nan, np.float32))
        engine.linear_attn(push, x, x + 2 * heads * hd, x + 4 * heads * hd, rates, cu, None, old, out, new, ws, need)
        return dev.get(out, (sum(lens), heads, hd)), dev.get(new, s0.shape, np.float32)

    apart, same = dev.put(s0), dev.put(s0)
    want, state = run(apart, dev.put(np.full(s0.shape, np.nan, np.float32)))
    got, left = run(same, same)
    assert (got == want).all() and (left == state).all() and not np.isnan(state).any()
    assert (dev.get(apart, s0.shape, np.float32) == s0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
def test_linear_strides(engine, dev, dtype, hd):
    """Heads that read the same queries and the same values (head strides of 0), rows with room in them, outputs head by
    head: the same bits as from dense rows; along a sequence and a token at a time."""
    rng, heads, n, room = np.random.default_rng(hd), 4, 70, 24
    q, k, v = (normal(rng, (n, h, hd), dtype) for h in (1, heads, 1))
    dense = [dev.put(np.ascontiguousarray(np.broadcast_to(a, (n, heads, hd)))) for a in (q, k, v)]
    odd = np.full((n, heads * (hd + 8) + room), NAN[dtype], np.uint16)
    odd[:, :heads * (hd + 8)].reshape(n, heads, hd + 8)[..., :hd] = k
    s0 = dev.put(rng.standard_normal((n, heads, hd, hd)).astype(np.float32))
    rates = dev.put(np.array([0.0, 0.01, 0.3, 3.0], np.float32))

    def push(seqs, **kw):
        p = linear_push(dtype, seqs, n, heads, heads, hd, n, 0.25, heads * hd)
        for name, value in kw.items():
            setattr(p, name, value)
        return p

    strides = dict(q_token_stride=hd, q_head_stride=0, k_token_stride=odd.shape[1], k_head_stride=hd + 8, v_token_stride=hd,
                   v_head_stride=0, out_token_stride=hd + 8, out_head_stride=n * (hd + 8))
    for seqs in (1, n):
        for step in (False, True)[:1 if seqs == 1 else 2]:
            outs, states = [], []
            for x, p in ((dense, push(seqs)), ([dev.put(q), dev.put(odd), dev.put(v)], push(seqs, **strides))):
                new = dev.put(np.full((n, heads, hd, hd), np.nan, np.float32))
                out = dev.put(np.full((heads, n, hd + 8), NAN[dtype], np.uint16))
                if step:
                    engine.linear_step(p, *x, rates, None, s0, out, new)
                else:
                    assert engine.linear_attn_workspace(p) == 0
                    engine.linear_attn(p, *x, rates, None, None, s0, out, new, None, 0)
                outs.append(dev.get(out, (heads, n, hd + 8)))
                states.append(dev.get(new, (seqs, heads, hd, hd), np.float32))
            plain = outs[0].reshape(-1)[:n * heads * hd].reshape(n, heads, hd).transpose(1, 0, 2)
            assert (outs[1][..., :hd] == plain).all() and (outs[1][..., hd:] == NAN[dtype]).all()
            assert (states[0] == states[1]).all() and not np.isnan(states[0]).any()


def test_linear_thousands_of_sequences(engine, dev):
    """More than the 64 x 64 that two looks at the starts find."""
    rng = np.random.default_rng(14)
    check_linear(engine, dev, rng, "bf16", 16, 1, 1, [int(x) for x in rng.integers(0, 4, 4500)])


def test_linear_starts_that_are_not_in_order(engine, dev):
    """What they give is not specified; rows and states that are not the call's stay as they were."""
    rng, heads, hd, n = np.random.default_rng(15), 2, 32, 3
    for cu in ([700, 100, 900, 50], [0, 2000, -5, 1000], [1000, 0, 0, 0]):
        x, out = dev.put(normal(rng, (1000, 3 * heads, hd), "fp16")), dev.put(np.full((1002, heads, hd), NAN["fp16"], np.uint16))
        push = linear_push("fp16", n, 1000, heads, heads, hd, n, 0.1, 3 * heads * hd)
        need = engine.linear_attn_workspace(push)
        ws, new = dev.put(np.zeros(need // 4 + 64, np.float32)), dev.put(np.full((n + 1, heads, hd, hd), 7.0, np.float32))
        assert need > 0
        engine.linear_attn(push, x, x + 2 * heads * hd, x + 4 * heads * hd, dev.put(np.zeros(heads, np.float32)), dev.put(np.array(cu, np.int32)),
                           None, None, out, new, ws, need)
        assert (dev.get(out, (1002, heads, hd))[1000:] == NAN["fp16"]).all()
        assert (dev.get(new, (n + 1, heads, hd, hd), np.float32)[n] == 7.0).all()
        assert (dev.get(ws, need // 4 + 64, np.float32)[need // 4:] == 0).all()


@pytest.mark.parametrize("four", [False, True])
def test_a_pool_past_32_bits(engine, dev, device_arena, four):
    """Pages whose offsets, in elements and in bytes, pass 2^32: written, read back and attended to as in a small pool."""
    rng, dtype, hd, kv, heads, page, n = np.random.default_rng(16), "bf16", 128, 8, 16, 128, 300
    pages = 2 ** 32 // (kv * page * hd) * (2 if four else 1) + 300  # elements, and in 4 bits also bytes
    big = [device_arena(pages * kv * page * b, zero=False).ptr for b in ([hd // 2] * 2 + [hd // 32] * 2 if four else [2 * hd] * 2)]
    big = P.CachePages(**dict(zip(("k", "v", "k_scales", "v_scales"), big)))
    small = P.CachePages(**{name: device_arena(300 * kv * page * (hd // 32 if name[1:] else hd // 2 if four else 2 * hd)).ptr
                            for name in (("k", "v", "k_scales", "v_scales") if four else ("k", "v"))})
    rows = normal(rng, (n, heads + 2 * kv, hd), dtype)
    x, row = dev.put(rows), (heads + 2 * kv) * hd
    seq, at = dev.put(np.repeat([0, 1], n // 2).astype(np.int32)), dev.put(np.tile(np.arange(n // 2), 2).astype(np.int32))
    pos, lengths = dev.put(np.arange(n, dtype=np.int32)), dev.put(np.array([n // 2, 140], np.int32))
    print(f"[big pool] {pages} pages, four {four}", flush=True)
    got = []
    for count, pool in ((300, small), (pages, big)):
        table = dev.put((count - 1 - np.array([[0, 7], [200, 3]])).astype(np.int32))
        cache = P.CacheDesc(dtype=TYPES[dtype], n_kv_heads=kv, head_dim=hd, page_size=page, n_pages=count, n_seqs=2, table_pages=2)
        push = P.RopeAppendPush(cache=cache, format=P.CACHE_4 if four else P.CACHE_16, n_new=n, n_heads=heads, n_axes=1,
                                pairs=(64, 0, 0, 0), layout=0, ladder=0, base=10000.0, q_token_stride=row, q_head_stride=hd,
                                k_token_stride=row, k_head_stride=hd, v_token_stride=row, v_head_stride=hd,
                                out_token_stride=heads * hd, out_head_stride=hd, pos_stride=n)
        q, k, v, o = (dev.put(np.full((n, heads, hd), NAN[dtype], np.uint16)) for _ in range(4))
        engine.rope_append(push, x, x + 2 * heads * hd, x + 2 * (heads + kv) * hd, pos, q, seq, at, table, pool)
        read = P.CacheReadPush(cache=cache, format=push.format, n_rows=n, k_token_stride=heads * hd, k_head_stride=hd,
                               v_token_stride=heads * hd, v_head_stride=hd)
        engine.cache_read(read, pool, seq, at, table, k, v)
        parts = [dev.get(a, (n, heads, hd)) for a in (q, k, v)]
        if four:
            for group in (2, 1):
                one = P.PagedAttnPush(cache=cache, n_heads=kv * group, left=-1, sinks=0, max_len=n // 2, scale=0.1,
                                      q_seq_stride=heads * hd, q_head_stride=hd, out_seq_stride=heads * hd, out_head_stride=hd)
                assert engine.paged_attn4_workspace(one) == 0
                engine.paged_attn4(one, q, pool, table, lengths, o, None, 0)
                parts.append(dev.get(o, (2, heads, hd))[:, :kv * group])
        got.append(parts)
    for a, b in zip(*got):
        assert (a == b).all()
    assert (got[0][1][:, :kv] != NAN[dtype]).any() and (got[0][1][:, kv:] == NAN[dtype]).all()


def test_two_streams_at_once(hip, engine, dev):
    """Calls on two streams, each with a workspace and outputs of its own: the bits of either alone."""
    rng, dtype, hd, heads, n = np.random.default_rng(17), "bf16", 64, 4, 1200
    rows = normal(rng, (n, 3 * heads, hd), dtype)
    x, rates, cu = dev.put(rows), dev.put(np.array([0.0, 0.01, 0.1, 1.0], np.float32)), dev.put(np.array([0, 900, n], np.int32))
    push = linear_push(dtype, 2, n, heads, heads, hd, 2, 0.125, 3 * heads * hd)
    need = engine.linear_attn_workspace(push)
    cache = Cache(rng, [2500, 60], 2, hd, 64, dtype, True)
    for s, ln in enumerate((2500, 60)):
        cache.fill(s, np.arange(ln), rng.standard_normal((ln, 2, hd)), rng.standard_normal((ln, 2, hd)))
    pages, table, lengths, q = cache.put(dev), dev.put(cache.table), dev.put(np.array([2500, 60], np.int32)), dev.put(normal(rng, (2, 8, hd), dtype))
    one = P.PagedAttnPush(cache=cache.desc(), n_heads=8, left=-1, sinks=0, max_len=2500, scale=0.125, q_seq_stride=8 * hd,
                          q_head_stride=hd, out_seq_stride=8 * hd, out_head_stride=hd)
    need4 = engine.paged_attn4_workspace(one)
    assert need > 0 and need4 > 0
    streams = [hip.stream(), hip.stream()]
    mine = [dict(out=dev.put(np.zeros((n, heads, hd), np.uint16)), state=dev.put(np.zeros((2, heads, hd, hd), np.float32)), a=dev.put(np.zeros((2, 8, hd), np.uint16)),
                 ws=dev.put(np.full(need // 4, np.nan, np.float32)), ws4=dev.put(np.full(need4 // 4, np.nan, np.float32))) for _ in range(3)]
    hip.sync()

    def calls(d, s):
        engine.linear_attn(push, x, x + 2 * heads * hd, x + 4 * heads * hd, rates, cu, None, None, d["out"], d["state"], d["ws"], need, s)
        engine.paged_attn4(one, q, pages, table, lengths, d["a"], d["ws4"], need4, s)

    calls(mine[2], None)
    hip.sync()
    for _ in range(5):
        for d, s in zip(mine, streams):
            calls(d, s)
    hip.sync()
    for name, shape, t in (("out", (n, heads, hd), np.uint16), ("state", (2, heads, hd, hd), np.float32), ("a", (2, 8, hd), np.uint16)):
        want = dev.get(mine[2][name], shape, t)
        assert want.any() and all((dev.get(d[name], shape, t) == want).all() for d in mine[:2])


def test_a_page_of_two_streams(engine, dev):
    """A prompt's pages in two streams' tables: each attends as if they were its own."""
    rng, dtype, hd, kv, page = np.random.default_rng(18), "fp16", 32, 2, 16
    cache = Cache(rng, [48, 48], kv, hd, page, dtype, True)
    for j in range(48):
        k, v = rng.standard_normal((2, kv, hd))
        cache.write(0, j, k, v)
        cache.write(1, j, k, v)
    q = np.repeat(normal(rng, (1, 4, hd), dtype), 2, 0)
    apart = run_paged4(engine, dev, cache, q, [48, 48], -1, 0, 0.2, 48)
    cache.table[1, :2] = cache.table[0, :2]
    together = run_paged4(engine, dev, cache, q, [48, 48], -1, 0, 0.2, 48)
    assert (apart == together).all() and (apart[0] == apart[1]).all() and np.isfinite(apart).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,group", [(16, 1), (16, 2), (32, 1), (32, 2), (64, 1), (128, 4)])
@pytest.mark.parametrize("at", [0, 20, 69, 70])
def test_paged4_a_key_of_nan_reaches_its_head_alone(engine, dev, dtype, hd, group, at):
    """A key of NaN makes NaN of the heads that share it, in the stream that sees it (70 keys); one behind the last is not seen."""
    rng = np.random.default_rng(19)
    kv, page, lengths = 2, 16, [71, 70, 71]
    cache = Cache(rng, lengths, kv, hd, page, dtype, True)
    for s, n in enumerate(lengths):
        cache.fill(s, np.arange(n), rng.standard_normal((n, kv, hd)), rng.standard_normal((n, kv, hd)))
    p, slot = cache.place(1, at)
    cache.ks[p, 0, slot, 0] = 255
    got = run_paged4(engine, dev, cache, normal(rng, (3, kv * group, hd), dtype), lengths, -1, 0, 0.2, 71)
    bad = np.zeros(got.shape, bool)
    bad[1, :group] = at < 70
    assert (np.isnan(got) == bad).all()
