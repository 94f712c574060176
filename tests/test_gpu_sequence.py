"""The sequence operators on the GPU, through the C ABI, against their definitions in 64 bits (error bounds:
seqlib.py). Outputs start as NaN, so every value has to be written; what must not be used is NaN as well."""
import math

import numpy as np
import pytest

import prism_amd as P
from seqlib import (HALF_STEP, NAN, SMALLEST, TYPES, Device, attention_row, normal, to_bits, values, visible)

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


# ------------------------------------------------------------------- rope

def rope_ref(x, pos, pairs, layout, ladder, inverse, base, dtype):
    """x [tokens][heads][hd] -> (turned, bound)."""
    n, y = sum(pairs), x.copy()
    bound = np.zeros_like(x)
    i = 0
    for axis, count in enumerate(pairs):
        for j in range(count):
            f = base ** -(i / n if ladder == P.ROPE_ONE_LADDER else j / count) * (-1 if inverse else 1)
            phi = pos[axis][:len(x)].astype(np.float64)[:, None] * f
            a, b = (i, i + n) if layout == P.ROPE_HALVES else (2 * i, 2 * i + 1)
            u, w = x[..., a], x[..., b]
            y[..., a], y[..., b] = u * np.cos(phi) - w * np.sin(phi), w * np.cos(phi) + u * np.sin(phi)
            # angle: 2^-25 turns for its fp32 form, 2^-51 of its size for the 64-bit products (here and there);
            # sin, cos and the two products: 2^-21
            off = 2 * np.pi * 2.0 ** -25 + np.abs(phi) * 2.0 ** -51 + 2.0 ** -21
            for c in (a, b):
                bound[..., c] = (np.abs(u) + np.abs(w)) * off + HALF_STEP[dtype] * np.abs(y[..., c]) + SMALLEST[dtype]
            i += 1
    return y, bound


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", [P.ROPE_HALVES, P.ROPE_ADJACENT])
@pytest.mark.parametrize("tokens,heads,hd,pairs,ladder,inverse", [
    (1, 1, 8, (1, 0, 2, 0), 0, 0), (3, 16, 16, (2, 3, 3), 0, 1), (257, 5, 32, (4, 6, 6), 0, 0), (64, 3, 32, (3, 4, 2), 1, 1),
    (33, 7, 64, (8, 8, 8, 8), 1, 0), (130, 40, 128, (12, 18, 18), 1, 1), (19, 2, 256, (128,), 0, 0), (9, 3, 72, (11, 0, 14), 0, 0),
    (1000, 1, 24, (1,), 0, 1), (5, 300, 16, (4, 4), 1, 0), (61, 11, 128, (24, 20, 20), 0, 0),
])
def test_rope(engine, dev, dtype, layout, tokens, heads, hd, pairs, ladder, inverse):
    rng = np.random.default_rng(tokens + hd + heads)
    extra = heads // 2
    rows = normal(rng, (tokens, heads + extra, hd), dtype)
    pos = rng.integers(-50, 2000, (len(pairs), tokens + 3)).astype(np.int32)
    pos[0, 0], pos[-1, -4] = -2 ** 31, MAX
    x, p, y = dev.put(rows), dev.put(pos), dev.put(np.full((tokens, heads, hd), NAN[dtype], np.uint16))
    push = P.RopePush(dtype=TYPES[dtype], n_tokens=tokens, n_heads=heads, head_dim=hd, n_axes=len(pairs),
                      pairs=pairs + (0,) * (4 - len(pairs)), layout=layout, ladder=ladder, inverse=inverse, base=10000.0,
                      in_token_stride=(heads + extra) * hd, in_head_stride=hd, out_token_stride=heads * hd, out_head_stride=hd,
                      pos_stride=tokens + 3)
    print(f"[rope] {dtype} layout {layout} {tokens} x {heads} x {hd}", flush=True)
    engine.rope(push, x, p, y)
    got = dev.get(y, (tokens, heads, hd))
    want, bound = rope_ref(values(rows[:, :heads], dtype), pos, pairs, layout, ladder, inverse, 10000.0, dtype)
    assert not outside(values(got, dtype), want, bound)
    assert (got[..., 2 * sum(pairs):] == rows[:, :heads, 2 * sum(pairs):]).all()  # copied bits
    # in place, inside the wider rows: the same bits, and the other heads untouched
    push.out_token_stride = push.in_token_stride
    engine.rope(push, x, p, x)
    there = dev.get(x, rows.shape)
    assert (there[:, :heads] == got).all() and (there[:, heads:] == rows[:, heads:]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_rope_heads_outermost_and_repeated_input(engine, dev, dtype):
    """Output [head][token][hd] from one input head for all (head stride 0)."""
    rng = np.random.default_rng(3)
    tokens, heads, hd, pairs = 21, 6, 32, (5, 5, 6)
    rows, pos = normal(rng, (tokens, hd), dtype), rng.integers(0, 99, (3, tokens)).astype(np.int32)
    x, p, y = dev.put(rows), dev.put(pos), dev.put(np.full((heads, tokens, hd), NAN[dtype], np.uint16))
    engine.rope(P.RopePush(dtype=TYPES[dtype], n_tokens=tokens, n_heads=heads, head_dim=hd, n_axes=3, pairs=pairs + (0,),
                           layout=0, ladder=0, inverse=0, base=100.0, in_token_stride=hd, in_head_stride=0,
                           out_token_stride=hd, out_head_stride=tokens * hd, pos_stride=tokens), x, p, y)
    got = values(dev.get(y, (heads, tokens, hd)), dtype).transpose(1, 0, 2)
    want, bound = rope_ref(np.repeat(values(rows, dtype)[:, None], heads, 1), pos, pairs, 0, 0, 0, 100.0, dtype)
    assert not outside(got, want, bound)


def test_rope_gradient(engine, dev):
    """The inverse is the gradient's way back: <g, R x> = <R^-1 g, x>, and it agrees with differences of R."""
    rng = np.random.default_rng(5)
    tokens, heads, hd, pairs, dtype = 12, 3, 32, (4, 6, 5), "fp16"
    n = (tokens, heads, hd)
    g, step = normal(rng, n, dtype), normal(rng, n, dtype)
    x0 = normal(rng, n, dtype)
    x1 = to_bits(values(x0, dtype) + values(step, dtype), dtype)
    pos = rng.integers(0, 5000, (3, tokens)).astype(np.int32)
    p = dev.put(pos)

    def turn(bits, inverse):
        x, y = dev.put(bits), dev.put(np.full(n, NAN[dtype], np.uint16))
        engine.rope(P.RopePush(dtype=0, n_tokens=tokens, n_heads=heads, head_dim=hd, n_axes=3, pairs=pairs + (0,), layout=1,
                               ladder=0, inverse=inverse, base=10000.0, in_token_stride=heads * hd, in_head_stride=hd,
                               out_token_stride=heads * hd, out_head_stride=hd, pos_stride=tokens), x, p, y)
        return values(dev.get(y, n), dtype)

    back, y0, y1 = turn(g, 1), turn(x0, 0), turn(x1, 0)
    want, bound = rope_ref(values(g, dtype), pos, pairs, 1, 0, 1, 10000.0, dtype)
    assert not outside(back, want, bound)
    gv, dx, dy = values(g, dtype), values(x1, dtype) - values(x0, dtype), y1 - y0
    # every output is within its bound of the exact linear map
    b0, b1 = (rope_ref(values(b, dtype), pos, pairs, 1, 0, 0, 10000.0, dtype)[1] for b in (x0, x1))
    assert abs((gv * dy).sum() - (back * dx).sum()) <= (np.abs(gv) * (b0 + b1)).sum() + (np.abs(dx) * bound).sum()


# ----------------------------------------------------------------- the cache

def paged_cache(rng, lengths, kv, hd, page, dtype, spare=3, width_extra=1):
    """(k_pages, v_pages, table): NaN in every slot, pages in mixed order, unused entries out of the pool."""
    need = [-(-n // page) for n in lengths]
    pool = sum(need) + spare
    order = iter(rng.permutation(pool))
    table = np.full((len(lengths), max(need + [0]) + width_extra), -1, np.int32)
    table[:, -1] = MAX
    for s, n in enumerate(need):
        for j in range(n):
            table[s, j] = next(order)
    shape = (pool, kv, page, hd)
    return np.full(shape, NAN[dtype], np.uint16), np.full(shape, NAN[dtype], np.uint16), table


def fill(pages, table, s, rows):
    page = pages.shape[2]
    for j, row in enumerate(rows):
        pages[table[s, j // page], :, j % page] = row


@pytest.mark.parametrize("hd,kv,page,dtype", [(16, 8, 16, "fp16"), (32, 1, 1, "bf16"), (64, 3, 4, "fp16"), (128, 2, 128, "bf16")])
def test_append(engine, dev, hd, kv, page, dtype):
    rng = np.random.default_rng(hd)
    final = [0, 1, 2 * page, 3 * page + 1, 5]
    kp, vp, table = paged_cache(rng, final, kv, hd, page, dtype)
    table[4, 0] = kp.shape[0]  # this sequence's first page is not in the pool
    seq = np.repeat(np.arange(5), final)
    at = np.concatenate([np.arange(n) for n in final])
    # padding rows and positions out of range, among the others
    seq = np.concatenate([seq, [-1, 5, MAX, 0, 2, 3, -2 ** 31]]).astype(np.int32)
    at = np.concatenate([at, [0, 0, 0, -1, table.shape[1] * page, MAX, 0]]).astype(np.int32)
    mix = rng.permutation(len(seq))
    seq, at = seq[mix], at[mix]
    rows = normal(rng, (len(seq), 2 * kv, hd), dtype)
    k, v, sq, pos, t, dk, dv = (dev.put(a) for a in (rows, rows[:, kv:].copy(), seq, at, table, kp, vp))
    print(f"[append] {len(seq)} rows, {kv} x {hd}, pages of {page}", flush=True)
    engine.cache_append(P.AppendPush(
        cache=P.CacheDesc(dtype=TYPES[dtype], n_kv_heads=kv, head_dim=hd, page_size=page, n_pages=kp.shape[0], n_seqs=5,
                          table_pages=table.shape[1]),
        n_new=len(seq), k_token_stride=2 * kv * hd, k_head_stride=hd, v_token_stride=kv * hd, v_head_stride=hd),
        k, v, sq, pos, t, dk, dv)
    for i in range(len(seq)):
        s, j = seq[i], at[i]
        if 0 <= s < 5 and 0 <= j < table.shape[1] * page and 0 <= table[s, j // page] < kp.shape[0]:
            kp[table[s, j // page], :, j % page] = rows[i, :kv]
            vp[table[s, j // page], :, j % page] = rows[i, kv:]
    assert (dev.get(dk, kp.shape) == kp).all() and (dev.get(dv, vp.shape) == vp).all()


def run_paged(engine, dev, dtype, q, kp, vp, table, lengths, left, sinks, scale, max_len, stream=None, out=None, guard=2):
    n, heads, hd = q.shape
    if out is None:
        out = dev.put(np.full((n + guard, heads, hd), NAN[dtype], np.uint16))
    push = P.PagedAttnPush(
        cache=P.CacheDesc(dtype=TYPES[dtype], n_kv_heads=kp.shape[1], head_dim=hd, page_size=kp.shape[2], n_pages=kp.shape[0],
                          n_seqs=n, table_pages=table.shape[1]),
        n_heads=heads, left=left, sinks=sinks, max_len=max_len, scale=scale, q_seq_stride=heads * hd, q_head_stride=hd,
        out_seq_stride=heads * hd, out_head_stride=hd)
    need = engine.paged_attn_workspace(push)
    ws = dev.put(np.full(need // 2, NAN["fp16"], np.uint16))
    engine.paged_attn(push, dev.put(q), dev.put(kp), dev.put(vp), dev.put(table), dev.put(lengths), out, ws, need, stream)
    got = dev.get(out, (n + guard, heads, hd))
    assert (got[n:] == NAN[dtype]).all()  # rows behind the last sequence
    return values(got[:n], dtype)


def check_paged(engine, dev, rng, dtype, hd, kv, group, page, lengths, left, sinks, max_len=None, q=None, big=1.0):
    kp, vp, table = paged_cache(rng, lengths, kv, hd, page, dtype)
    heads, scale = kv * group, 1 / math.sqrt(hd)
    q = normal(rng, (len(lengths), heads, hd), dtype) if q is None else q
    ks, vs = [], []
    for s, n in enumerate(lengths):
        k, v = normal(rng, (n, kv, hd), dtype), normal(rng, (n, kv, hd), dtype)
        if big != 1.0:
            k = to_bits(values(k, dtype) * big, dtype)
        seen = visible(n - 1, n, left, 0, sinks)
        k[~seen], v[~seen] = NAN[dtype], NAN[dtype]
        fill(kp, table, s, k)
        fill(vp, table, s, v)
        for j in range(-(-n // page)):  # pages out of the window need not exist
            if not seen[j * page:(j + 1) * page].any():
                table[s, j] = -1
        ks.append(values(k, dtype))
        vs.append(values(v, dtype))
    print(f"[paged] {dtype} {heads}/{kv} x {hd} pages of {page} lengths {lengths} left {left} sinks {sinks}", flush=True)
    got = run_paged(engine, dev, dtype, q, kp, vp, table, np.array(lengths, np.int32), left, sinks, scale,
                    max(lengths) if max_len is None else max_len)
    qv = values(q, dtype)
    for s, n in enumerate(lengths):
        seen = visible(n - 1, n, left, 0, sinks)
        for h in range(heads):
            want, bound = attention_row(qv[s, h], ks[s][:, h // group], vs[s][:, h // group], seen, scale, dtype)
            msg = outside(got[s, h], want, bound)
            assert not msg, (s, h, msg)


LENGTHS = [0, 1, 15, 16, 17, 33, 130]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("kv,group", [(8, 1), (2, 2), (1, 3), (2, 4), (1, 8), (1, 17), (3, 5)])
def test_paged_shapes(engine, dev, dtype, hd, kv, group):
    rng = np.random.default_rng(hd + 7 * group)
    check_paged(engine, dev, rng, dtype, hd, kv, group, 16, LENGTHS, -1, 0)


@pytest.mark.parametrize("page", [1, 2, 8, 64, 256])
@pytest.mark.parametrize("left,sinks,group", [(-1, 0, 1), (0, 0, 1), (0, 3, 4), (20, 0, 4), (31, 5, 1), (31, 64, 8), (500, 9, 2), (MAX, MAX, 1)])
def test_paged_windows(engine, dev, page, left, sinks, group):
    rng = np.random.default_rng(page + left % 1000 + sinks % 1000)
    check_paged(engine, dev, rng, "fp16", 32, 2, group, page, [1, 5, 32, 33, 64, 131, 300], left, sinks)


@pytest.mark.parametrize("dtype,hd,kv,group,lengths,max_len", [
    ("fp16", 32, 8, 1, [3000], None), ("bf16", 128, 2, 4, [4097, 10, 2500], None), ("fp16", 128, 1, 1, [5001], None),
    ("bf16", 64, 1, 32, [1025, 2047], None),  # more heads than a tile of 16
    ("fp16", 64, 2, 4, [3000, 7], 16),       # longer than announced
    ("fp16", 64, 2, 1, [40, 7], 100000),     # shorter than announced
    ("bf16", 32, 2, 1, [700, 0], 0),         # not announced
])
def test_paged_long(engine, dev, dtype, hd, kv, group, lengths, max_len):
    rng = np.random.default_rng(hd + group)
    check_paged(engine, dev, rng, dtype, hd, kv, group, 32, lengths, -1, 0, max_len)


@pytest.mark.parametrize("group", [1, 4])
def test_paged_long_window_and_sinks(engine, dev, group):
    rng = np.random.default_rng(8)
    check_paged(engine, dev, rng, "bf16", 64, 2, group, 16, [6000, 2500, 1, 900], 2047, 70)


@pytest.mark.parametrize("group", [1, 8])
def test_paged_sharp_scores(engine, dev, group):
    """Scores of hundreds: one key takes nearly all the weight, wherever it is."""
    rng = np.random.default_rng(9)
    check_paged(engine, dev, rng, "fp16", 64, 1, group, 16, [257, 1000], -1, 0, big=60.0)


@pytest.mark.parametrize("group", [1, 4])
def test_paged_tiny_values(engine, dev, group):
    """fp16 queries below the type's smallest normal number, a scale that makes up for it."""
    rng = np.random.default_rng(14)
    dtype, hd, n, page = "fp16", 64, 50, 16
    q = to_bits(rng.standard_normal((1, group, hd)) * 2e-5, dtype)
    kp, vp, table = paged_cache(rng, [n], 1, hd, page, dtype)
    k, v = normal(rng, (n, 1, hd), dtype), normal(rng, (n, 1, hd), dtype)
    fill(kp, table, 0, k)
    fill(vp, table, 0, v)
    got = run_paged(engine, dev, dtype, q, kp, vp, table, np.array([n], np.int32), -1, 0, 8192.0, n)
    for h in range(group):
        want, bound = attention_row(values(q[0, h], dtype), values(k[:, 0], dtype), values(v[:, 0], dtype), np.ones(n, bool),
                                    8192.0, dtype)
        assert not outside(got[0, h], want, bound), h


@pytest.mark.parametrize("group", [1, 4])
@pytest.mark.parametrize("hd", [16, 128])
def test_paged_bad_tables(engine, dev, hd, group):
    """Keys of entries out of the pool are not seen; lengths out of range are brought into it."""
    rng = np.random.default_rng(10)
    dtype, kv, page = "fp16", 2, 8
    kp, vp, table = paged_cache(rng, [40, 40, 40, 40], kv, hd, page, dtype, width_extra=0)
    rows = [normal(rng, (40, kv, hd), dtype) for _ in range(4)]
    for s in range(4):
        fill(kp, table, s, rows[s])
        fill(vp, table, s, rows[s])
    table[0, 1], table[0, 4] = -5, kp.shape[0]
    table[1, :] = MAX
    lengths = np.array([40, 40, MAX, -3], np.int32)
    q = normal(rng, (4, kv * group, hd), dtype)
    got = run_paged(engine, dev, dtype, q, kp, vp, table, lengths, -1, 0, 0.25, 40)
    seen = np.ones((4, 40), bool)
    seen[0, 8:16] = seen[0, 32:] = seen[1] = seen[3] = False
    for s in range(4):
        for h in range(kv * group):
            k = values(rows[s][:, h // group], dtype)
            want, bound = attention_row(values(q[s, h], dtype), k, k, seen[s], 0.25, dtype)
            assert not outside(got[s, h], want, bound), (s, h)


def test_paged_offsets_past_32_bits(hip, engine, dev, device_arena):
    """Pools of more than 2^31 elements (4 GiB), the pages at both ends used."""
    rng = np.random.default_rng(11)
    page, kv, hd = 128, 8, 128
    per = page * kv * hd
    n_pages = 2 ** 31 // per + 3
    kp, vp = device_arena(n_pages * per * 2, zero=False), device_arena(n_pages * per * 2, zero=False)
    used = [0, n_pages - 1, n_pages - 2, 1]
    table = np.array([[used[0], used[1]], [used[2], used[3]]], np.int32)
    lengths = [page + 3, 2 * page]
    k, v = normal(rng, (sum(lengths), kv, hd), "bf16"), normal(rng, (sum(lengths), kv, hd), "bf16")
    cache = P.CacheDesc(dtype=P.BF16, n_kv_heads=kv, head_dim=hd, page_size=page, n_pages=n_pages, n_seqs=2, table_pages=2)
    seq = np.repeat([0, 1], lengths).astype(np.int32)
    at = np.concatenate([np.arange(n) for n in lengths]).astype(np.int32)
    dt = dev.put(table)
    engine.cache_append(P.AppendPush(cache=cache, n_new=len(seq), k_token_stride=kv * hd, k_head_stride=hd,
                                     v_token_stride=kv * hd, v_head_stride=hd), dev.put(k), dev.put(v), dev.put(seq),
                        dev.put(at), dt, kp.ptr, vp.ptr)
    for group in (1, 4):
        q = normal(rng, (2, kv * group, hd), "bf16")
        out = dev.put(np.full(q.shape, NAN["bf16"], np.uint16))
        push = P.PagedAttnPush(cache=cache, n_heads=kv * group, left=-1, sinks=0, max_len=256, scale=0.1,
                               q_seq_stride=kv * group * hd, q_head_stride=hd, out_seq_stride=kv * group * hd, out_head_stride=hd)
        need = engine.paged_attn_workspace(push)
        ws = device_arena(max(need, 16))
        engine.paged_attn(push, dev.put(q), kp.ptr, vp.ptr, dt, dev.put(np.array(lengths, np.int32)), out, ws.ptr, need)
        got = values(dev.get(out, q.shape), "bf16")
        for s in range(2):
            for h in range(kv * group):
                rows = seq == s
                kk, vv = values(k[rows][:, h // group], "bf16"), values(v[rows][:, h // group], "bf16")
                want, bound = attention_row(values(q[s, h], "bf16"), kk, vv, np.ones(len(kk), bool), 0.1, "bf16")
                assert not outside(got[s, h], want, bound), (group, s, h)


# ---------------------------------------------------------------- sequences

FILL = pytest.mark.parametrize("fill", ["few", "some", "many"])


def spare(fill, groups=1):
    """What leads to the kernels for few, some and many workgroups: (empty sequences, key rows for each sequence)."""
    return {None: (0, 0), "few": (0, 400), "some": (-(-165 // groups), 400), "many": (1025, 0)}[fill]


def check_seq(engine, dev, rng, dtype, hd, kv, group, lens, left, right, sinks, layout="dense", head=0, tail=3, big=1.0, fill=None):
    """lens: (queries, keys) of each sequence; head, tail: rows before the first and behind the last; fill: see spare."""
    empty, rows = spare(fill, kv if group <= 32 else kv * group)
    lens = lens + [(0, 0)] * empty
    heads, scale = kv * group, 1 / math.sqrt(hd)
    cq = (head + np.concatenate([[0], np.cumsum([a for a, _ in lens])])).astype(np.int32)
    ck = (head + np.concatenate([[0], np.cumsum([b for _, b in lens])])).astype(np.int32)
    nq, nk = int(cq[-1]) + tail, max(int(ck[-1]) + tail, rows * len(lens))
    q, k, v = normal(rng, (nq, heads, hd), dtype), normal(rng, (nk, kv, hd), dtype), normal(rng, (nk, kv, hd), dtype)
    if big != 1.0:
        k = to_bits(values(k, dtype) * big, dtype)
    used = np.zeros(nk, bool)
    for s, (a, b) in enumerate(lens):
        for i in range(a):
            used[ck[s]:ck[s + 1]] |= visible(b - a + i, b, left, right, sinks)
    k[~used], v[~used] = NAN[dtype], NAN[dtype]
    if layout == "fused":  # one row of queries, keys and values per token
        assert nq == nk
        rows = np.concatenate([q, k, v], 1)
        base = dev.put(rows)
        w = rows.shape[1] * hd
        dq, dk, dv = base, base + 2 * heads * hd, base + 2 * (heads + kv) * hd
        st = (w, hd) * 3 + (heads * hd, hd)
    elif layout == "heads":  # [head][row][hd], the output too
        dq, dk, dv = (dev.put(a.transpose(1, 0, 2)) for a in (q, k, v))
        st = (hd, nq * hd, hd, nk * hd, hd, nk * hd, hd, nq * hd)
    else:
        dq, dk, dv = dev.put(q), dev.put(k), dev.put(v)
        st = (heads * hd, hd, kv * hd, hd, kv * hd, hd, heads * hd, hd)
    out = dev.put(np.full(nq * heads * hd, NAN[dtype], np.uint16))
    names = ("q_token_stride", "q_head_stride", "k_token_stride", "k_head_stride", "v_token_stride", "v_head_stride",
             "out_token_stride", "out_head_stride")
    push = P.SeqAttnPush(dtype=TYPES[dtype], n_seqs=len(lens), n_q=nq, n_k=nk, n_heads=heads, n_kv_heads=kv, head_dim=hd,
                         left=left, right=right, sinks=sinks, scale=scale, **dict(zip(names, st)))
    print(f"[seq] {dtype} {heads}/{kv} x {hd} {lens[:12]} fill {fill} left {left} right {right} sinks {sinks} {layout}", flush=True)
    engine.seq_attn(push, dq, dk, dv, dev.put(cq), dev.put(ck), out)
    got = dev.get(out, (heads, nq, hd)).transpose(1, 0, 2) if layout == "heads" else dev.get(out, (nq, heads, hd))
    assert (got[:head] == NAN[dtype]).all() and (got[nq - tail:] == NAN[dtype]).all()
    got, qv, kv_, vv = values(got, dtype), values(q, dtype), values(k, dtype), values(v, dtype)
    for s, (a, b) in enumerate(lens):
        for i in range(a):
            seen = visible(b - a + i, b, left, right, sinks)
            for h in range(heads):
                want, bound = attention_row(qv[cq[s] + i, h], kv_[ck[s]:ck[s + 1], h // group], vv[ck[s]:ck[s + 1], h // group],
                                            seen, scale, dtype)
                msg = outside(got[cq[s] + i, h], want, bound)
                assert not msg, (s, i, h, msg)


RAGGED = [(1, 1), (0, 0), (5, 5), (64, 64), (65, 65), (0, 7), (31, 31), (130, 130), (3, 0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("kv,group", [(2, 1), (1, 3)])
@FILL
def test_seq_shapes(engine, dev, dtype, hd, kv, group, fill):
    check_seq(engine, dev, np.random.default_rng(hd), dtype, hd, kv, group, RAGGED, -1, 0, 0, fill=fill)


@pytest.mark.parametrize("left,right,sinks", [
    (-1, -1, 0), (0, 0, 0), (0, 0, 3), (7, 0, 0), (40, 0, 5), (63, 0, 100), (20, 9, 2), (0, 30, 0), (-1, 5, 0), (200, -1, 1),
    (MAX, MAX, MAX), (3, -1, 0), (0, 0, 384), (63, 3, 400), (150, 250, 3), (384, 0, 2), (190, 1, 0),
])
@pytest.mark.parametrize("hd", [32, 128])
@FILL
def test_seq_windows(engine, dev, left, right, sinks, hd, fill):
    rng = np.random.default_rng(abs(left) % 97 + right % 89 + sinks % 83)
    check_seq(engine, dev, rng, "fp16", hd, 1, 2, [(150, 450), (1, 1), (33, 600), (70, 20), (200, 200)], left, right, sinks,
              fill=fill)


@pytest.mark.parametrize("layout", ["fused", "heads"])
@pytest.mark.parametrize("hd", [16, 128])
def test_seq_layouts(engine, dev, layout, hd):
    rng = np.random.default_rng(hd)
    check_seq(engine, dev, rng, "bf16", hd, 2, 2, [(70, 70), (12, 12)], 30, 0, 4, layout, head=5)


@pytest.mark.parametrize("dtype,hd,lens,left,sinks", [
    ("fp16", 32, [(600, 600)], 128, 20), ("bf16", 128, [(300, 900), (257, 257)], 200, 4), ("fp16", 64, [(1, 2000), (4, 700)], 511, 1),
    ("bf16", 16, [(513, 513)], -1, 0),
])
@FILL
def test_seq_long(engine, dev, dtype, hd, lens, left, sinks, fill):
    check_seq(engine, dev, np.random.default_rng(1), dtype, hd, 1, 2, lens, left, 0, sinks, fill=fill)


@pytest.mark.parametrize("hd,kv,group", [(16, 1, 32), (32, 1, 33), (64, 3, 5), (32, 2, 8), (128, 1, 16), (16, 8, 2)])
@FILL
def test_seq_shared_heads(engine, dev, hd, kv, group, fill):
    """Groups that fill a workgroup's rows evenly or not, with a few queries, or not at all."""
    rng = np.random.default_rng(group)
    check_seq(engine, dev, rng, "bf16", hd, kv, group, [(9, 20), (1, 1), (0, 3), (37, 37), (5, 2)], 12, 0, 2, fill=fill)


@FILL
def test_seq_sharp_scores(engine, dev, fill):
    check_seq(engine, dev, np.random.default_rng(2), "fp16", 64, 1, 1, [(300, 300)], 100, 0, 3, big=60.0, fill=fill)


@FILL
def test_seq_rising_scores(engine, dev, fill):
    """The largest score comes last, tile after tile: the running maximum moves every time."""
    rng = np.random.default_rng(4)
    dtype, hd, n = "bf16", 32, 400
    k = rng.standard_normal((n, 1, hd)) * 0.1
    k[..., 0] = np.linspace(-60, 60, n)[:, None]
    q = np.zeros((n, 1, hd))
    q[..., 0] = np.where(np.arange(n) % 2, 4.0, -4.0)[:, None]
    empty, rows = spare(fill)  # one sequence and empty ones, or no starts at all
    seqs, nk = 1 + empty, max(n, rows * (1 + empty))
    q, v = to_bits(q, dtype), normal(rng, (nk, 1, hd), dtype)
    k = np.concatenate([to_bits(k, dtype), normal(rng, (nk - n, 1, hd), dtype)])
    out = dev.put(np.full((n, 1, hd), NAN[dtype], np.uint16))
    cu = dev.put(np.array([0] + [n] * seqs, np.int32)) if seqs > 1 else None
    push = P.SeqAttnPush(dtype=P.BF16, n_seqs=seqs, n_q=n, n_k=nk, n_heads=1, n_kv_heads=1, head_dim=hd, left=-1, right=0, sinks=0,
                         scale=1.0, q_token_stride=hd, q_head_stride=hd, k_token_stride=hd, k_head_stride=hd, v_token_stride=hd,
                         v_head_stride=hd, out_token_stride=hd, out_head_stride=hd)
    engine.seq_attn(push, dev.put(q), dev.put(k), dev.put(v), cu, cu, out)
    got = values(dev.get(out, (n, 1, hd)), dtype)
    for i in range(n):
        want, bound = attention_row(values(q[i, 0], dtype), values(k[:n, 0], dtype), values(v[:n, 0], dtype),
                                    visible(i, n, -1, 0, 0), 1.0, dtype)
        assert not outside(got[i, 0], want, bound), i


@pytest.mark.parametrize("dtype,hd", [("fp16", 16), ("bf16", 32), ("fp16", 64), ("bf16", 128)])
@pytest.mark.parametrize("what", ["v nan", "v inf", "k nan"])
@pytest.mark.parametrize("group", [1, 3])
@FILL
def test_seq_bad_values_reach_only_who_sees_them(engine, dev, dtype, hd, what, group, fill):
    """One key's value is NaN or infinite: the queries that see it get what the formula gives, the others what they
    would get without it."""
    rng = np.random.default_rng(hd)
    left = {"few": 200, "some": 400, "many": 40}[fill]
    empty, rows = spare(fill)
    n, at, sinks, seqs = 220 + 2 * left, 100, 2, 1 + empty
    nk = max(n, rows * seqs)
    q, k, v = normal(rng, (n, group, hd), dtype), normal(rng, (nk, 1, hd), dtype), normal(rng, (nk, 1, hd), dtype)
    inf = 0x7C00 if dtype == "fp16" else 0x7F80
    if what == "k nan":
        k[at, 0, 3] = NAN[dtype]
    else:
        v[at, 0, 5] = inf if what == "v inf" else NAN[dtype]
    out = dev.put(np.full((n, group, hd), NAN[dtype], np.uint16))
    st = {f"{x}_{y}_stride": hd * (group if x in ("q", "out") and y == "token" else 1) for x in ("q", "k", "v", "out")
          for y in ("token", "head")}
    cu = dev.put(np.array([0] + [n] * seqs, np.int32))
    engine.seq_attn(P.SeqAttnPush(dtype=TYPES[dtype], n_seqs=seqs, n_q=n, n_k=nk, n_heads=group,
                                  n_kv_heads=1, head_dim=hd, left=left, right=0, sinks=sinks, scale=0.1, **st), dev.put(q),
                    dev.put(k), dev.put(v), cu, cu, out)
    got_all = values(dev.get(out, (n, group, hd)), dtype)
    kv, vv = values(k[:n, 0], dtype), values(v[:n, 0], dtype)
    for h in range(group):
        got, qv = got_all[:, h], values(q[:, h], dtype)
        for i in range(n):
            seen = visible(i, n, left, 0, sinks)
            if not seen[at]:
                want, bound = attention_row(qv[i], kv, vv, seen, 0.1, dtype)
                assert not outside(got[i], want, bound), i
            elif what == "k nan":
                assert np.isnan(got[i]).all(), i
            else:
                want, bound = attention_row(qv[i], kv, np.where(np.isfinite(vv), vv, 0), seen, 0.1, dtype)
                want, bound, rest = np.delete(want, 5), np.delete(bound, 5), np.delete(got[i], 5)
                assert not outside(rest, want, bound), i
                assert np.isposinf(got[i, 5]) if what == "v inf" else np.isnan(got[i, 5]), i


@pytest.mark.parametrize("n_seqs", [70, 300])
def test_seq_many_short(engine, dev, n_seqs):
    """More sequences than a wave has lanes, empty ones among them."""
    rng = np.random.default_rng(n_seqs)
    lens = [(int(x), int(x)) for x in rng.integers(0, 6, n_seqs)]
    lens[n_seqs // 2] = (260, 261)
    check_seq(engine, dev, rng, "fp16", 16, 1, 1, lens, 3, 0, 1, head=131)


def test_seq_starts_out_of_range(engine, dev):
    """Starts past the rows or out of order: rows inside the buffers at most, and the good sequences right."""
    rng = np.random.default_rng(6)
    dtype, hd, n = "fp16", 32, 40
    q = normal(rng, (n, 1, hd), dtype)
    out = dev.put(np.full((n, 1, hd), NAN[dtype], np.uint16))
    cu = dev.put(np.array([0, 20, 10, MAX], np.int32))  # [0, 20), nothing, [10, 40)
    push = P.SeqAttnPush(dtype=P.F16, n_seqs=3, n_q=n, n_k=n, n_heads=1, n_kv_heads=1, head_dim=hd, left=-1, right=0, sinks=0,
                         scale=0.2, q_token_stride=hd, q_head_stride=hd, k_token_stride=hd, k_head_stride=hd, v_token_stride=hd,
                         v_head_stride=hd, out_token_stride=hd, out_head_stride=hd)
    x = dev.put(q)
    engine.seq_attn(push, x, x, x, cu, cu, out)
    got, xv = values(dev.get(out, (n, hd)), dtype), values(q[:, 0], dtype)
    for i in list(range(10)) + list(range(20, 40)):
        first = 0 if i < 10 else 10
        want, bound = attention_row(xv[i], xv[first:], xv[first:], visible(i - first, n - first, -1, 0, 0), 0.2, dtype)
        assert not outside(got[i], want, bound), i


@pytest.mark.parametrize("stride", [0, 8])
@pytest.mark.parametrize("hd", [16, 128])
@FILL
def test_seq_rows_that_overlap(engine, dev, stride, hd, fill):
    """Keys and values repeated or overlapping, an infinite value among them: each channel meets it or does not."""
    rng = np.random.default_rng(hd + stride)
    left = {"few": 200, "some": 400, "many": 40}[fill]
    empty, rows = spare(fill)
    dtype, n, sinks, seqs = "fp16", 220 + 2 * left, 3, 1 + empty
    nk = max(n, rows * seqs)
    flat = normal(rng, nk * stride + hd, dtype)
    flat[:hd:16] = to_bits(np.inf, dtype)
    q, k = normal(rng, (n, 1, hd), dtype), normal(rng, nk * stride + hd, dtype)
    out = dev.put(np.full((n, hd), NAN[dtype], np.uint16))
    cu = dev.put(np.array([0] + [n] * seqs, np.int32))
    push = P.SeqAttnPush(dtype=P.F16, n_seqs=seqs, n_q=n, n_k=nk, n_heads=1, n_kv_heads=1, head_dim=hd, left=left, right=0,
                         sinks=sinks, scale=0.1, q_token_stride=hd, q_head_stride=hd, k_token_stride=stride, k_head_stride=hd,
                         v_token_stride=stride, v_head_stride=hd, out_token_stride=hd, out_head_stride=hd)
    engine.seq_attn(push, dev.put(q), dev.put(k), dev.put(flat), cu, cu, out)
    got, qv = values(dev.get(out, (n, hd)), dtype), values(q[:, 0], dtype)
    row = lambda x: values(np.stack([x[stride * j:][:hd] for j in range(n)]), dtype)
    kv_, vv = row(k), row(flat)
    for i in range(n):
        seen = visible(i, n, left, 0, sinks)
        high = np.isinf(vv[seen]).any(0)
        want, bound = attention_row(qv[i], kv_, np.where(np.isinf(vv), 0, vv), seen, 0.1, dtype)
        assert np.isposinf(got[i, high]).all(), i
        assert not outside(got[i, ~high], want[~high], bound[~high]), i


@pytest.mark.parametrize("hd,n,sequences", [(32, 260, (1, 1101)), (128, 400, (1, 1101))])
def test_seq_largest_key_stride(hip, engine, dev, device_arena, hd, n, sequences):
    """Rows 8 MiB apart: the last of a tile's lies almost 2^31 bytes behind its first."""
    rng = np.random.default_rng(15)
    dtype, far = "bf16", 2 ** 22
    q, k, v = (normal(rng, (n, hd), dtype) for _ in "qkv")
    big = device_arena(((n - 1) * far + 2 * hd) * 2, zero=False)  # a row's keys, then its values
    for j in range(n):
        hip.upload(big.ptr + 2 * far * j, np.concatenate([k[j], v[j]]))
    for seqs in sequences:
        out = dev.put(np.full((n, hd), NAN[dtype], np.uint16))
        cu = dev.put(np.array([0] + [n] * seqs, np.int32))
        push = P.SeqAttnPush(dtype=P.BF16, n_seqs=seqs, n_q=n, n_k=n, n_heads=1, n_kv_heads=1, head_dim=hd, left=-1, right=0,
                             sinks=0, scale=0.2, q_token_stride=hd, q_head_stride=hd, k_token_stride=far, k_head_stride=hd,
                             v_token_stride=far, v_head_stride=hd, out_token_stride=hd, out_head_stride=hd)
        engine.seq_attn(push, dev.put(q), big.ptr, big.ptr + 2 * hd, cu, cu, out)
        got = values(dev.get(out, (n, hd)), dtype)
        for i in range(n):
            want, bound = attention_row(values(q[i], dtype), values(k, dtype), values(v, dtype), visible(i, n, -1, 0, 0), 0.2, dtype)
            assert not outside(got[i], want, bound), i


@pytest.mark.parametrize("hd", [16, 64])
def test_seq_tiny_values(engine, dev, hd):
    """fp16 queries below the type's smallest normal number, a scale that makes up for it."""
    rng = np.random.default_rng(16)
    dtype, n = "fp16", 100
    q, k, v = to_bits(rng.standard_normal((n, hd)) * 2e-5, dtype), normal(rng, (n, hd), dtype), normal(rng, (n, hd), dtype)
    out = dev.put(np.full((n, hd), NAN[dtype], np.uint16))
    push = P.SeqAttnPush(dtype=P.F16, n_seqs=1, n_q=n, n_k=n, n_heads=1, n_kv_heads=1, head_dim=hd, left=-1, right=-1, sinks=0,
                         scale=8192.0, q_token_stride=hd, q_head_stride=hd, k_token_stride=hd, k_head_stride=hd,
                         v_token_stride=hd, v_head_stride=hd, out_token_stride=hd, out_head_stride=hd)
    engine.seq_attn(push, dev.put(q), dev.put(k), dev.put(v), None, None, out)
    got = values(dev.get(out, (n, hd)), dtype)
    for i in range(n):
        want, bound = attention_row(values(q[i], dtype), values(k, dtype), values(v, dtype), np.ones(n, bool), 8192.0, dtype)
        assert not outside(got[i], want, bound), i


# ------------------------------------------------------------- used together

def stream_of_frames(engine, dev, rng, dtype, frames, places, heads, kv, hd, left, sinks):
    """Every place of a grid is a stream: (step-by-step outputs, outputs of the whole clip at once), [place][frame]."""
    pairs, page = (hd // 4, hd // 8, hd // 8), 4
    rows = normal(rng, (frames, places, heads + 2 * kv, hd), dtype)
    pos = np.stack([np.repeat(np.arange(frames), places), np.tile(np.arange(places) // 3, frames),
                    np.tile(np.arange(places) % 3, frames)]).astype(np.int32).reshape(3, frames, places)
    width = -(-frames // page)
    table = rng.permutation(places * width).astype(np.int32).reshape(places, width)
    cache = P.CacheDesc(dtype=TYPES[dtype], n_kv_heads=kv, head_dim=hd, page_size=page, n_pages=places * width, n_seqs=places,
                        table_pages=width)
    row = (heads + 2 * kv) * hd
    pools = [dev.put(np.full((places * width, kv, page, hd), NAN[dtype], np.uint16)) for _ in "kv"]
    dt, seq = dev.put(table), dev.put(np.arange(places, dtype=np.int32))
    turn = P.RopePush(dtype=TYPES[dtype], n_tokens=places, n_heads=heads + kv, head_dim=hd, n_axes=3, pairs=pairs + (0,), layout=0,
                      ladder=0, inverse=0, base=1000.0, in_token_stride=row, in_head_stride=hd, out_token_stride=row,
                      out_head_stride=hd, pos_stride=places)
    stepped = []
    for f in range(frames):
        x = dev.put(rows[f])
        engine.rope(turn, x, dev.put(pos[:, f]), x)  # queries and keys of the fused rows, in place
        k, v = x + 2 * heads * hd, x + 2 * (heads + kv) * hd
        engine.cache_append(P.AppendPush(cache=cache, n_new=places, k_token_stride=row, k_head_stride=hd, v_token_stride=row,
                                         v_head_stride=hd), k, v, seq, dev.put(np.full(places, f, np.int32)), dt, *pools)
        out = dev.put(np.full((places, heads, hd), NAN[dtype], np.uint16))
        push = P.PagedAttnPush(cache=cache, n_heads=heads, left=left, sinks=sinks, max_len=frames, scale=1 / math.sqrt(hd),
                               q_seq_stride=row, q_head_stride=hd, out_seq_stride=heads * hd, out_head_stride=hd)
        need = engine.paged_attn_workspace(push)
        ws = dev.put(np.zeros(need // 2, np.uint16))
        engine.paged_attn(push, x, *pools, dt, dev.put(np.full(places, f + 1, np.int32)), out, ws, need)
        stepped.append(dev.get(out, (places, heads, hd)))
    # the clip at once, streams one behind the other
    clip = np.ascontiguousarray(rows.transpose(1, 0, 2, 3))
    x, n = dev.put(clip), frames * places
    turn.n_tokens, turn.pos_stride = n, n
    engine.rope(turn, x, dev.put(np.ascontiguousarray(pos.transpose(0, 2, 1))), x)
    out = dev.put(np.full((n, heads, hd), NAN[dtype], np.uint16))
    engine.seq_attn(P.SeqAttnPush(dtype=TYPES[dtype], n_seqs=places, n_q=n, n_k=n, n_heads=heads, n_kv_heads=kv, head_dim=hd,
                                  left=left, right=0, sinks=sinks, scale=1 / math.sqrt(hd), q_token_stride=row, q_head_stride=hd,
                                  k_token_stride=row, k_head_stride=hd, v_token_stride=row, v_head_stride=hd,
                                  out_token_stride=heads * hd, out_head_stride=hd),
                    x, x + 2 * heads * hd, x + 2 * (heads + kv) * hd, None, None, out)
    whole = dev.get(out, (places, frames, heads, hd))
    turned = values(dev.get(x, (places, frames, heads + 2 * kv, hd)), dtype)
    return values(np.stack(stepped, 1), dtype), values(whole, dtype), turned


@pytest.mark.parametrize("dtype,heads,kv,hd,left,sinks", [("fp16", 8, 8, 32, 7, 2), ("fp16", 8, 8, 16, -1, 0), ("bf16", 8, 2, 64, 9, 1)])
def test_streamed_frames_and_the_clip_at_once(engine, dev, dtype, heads, kv, hd, left, sinks):
    """rope -> append -> one token per stream, frame by frame, against rope -> attention along the whole clip:
    both within the bound of the definition on the same turned queries and keys."""
    rng = np.random.default_rng(hd)
    frames, places, g = 21, 13, heads // kv
    stepped, whole, x = stream_of_frames(engine, dev, rng, dtype, frames, places, heads, kv, hd, left, sinks)
    for s in range(places):
        for f in range(frames):
            seen = visible(f, frames, left, 0, sinks)
            for h in range(heads):
                want, bound = attention_row(x[s, f, h], x[s, :, heads + h // g], x[s, :, heads + kv + h // g], seen,
                                            1 / math.sqrt(hd), dtype)
                for got in (stepped, whole):
                    assert not outside(got[s, f, h], want, bound), (s, f, h)


# -------------------------------------------------- streams, graphs, refusals

def test_captured_and_replayed(hip, engine, dev):
    """One graph of the four calls on a stream of its own, replayed on new inputs in the same buffers with eager
    calls between: every replay gives the bits of the eager calls."""
    rng = np.random.default_rng(12)
    heads, kv, hd, page, n, length = 8, 2, 64, 16, 3, 2500
    width = -(-length // page)
    row = (heads + 2 * kv) * hd
    cache = P.CacheDesc(dtype=P.F16, n_kv_heads=kv, head_dim=hd, page_size=page, n_pages=n * width, n_seqs=n, table_pages=width)
    turn = P.RopePush(dtype=0, n_tokens=n, n_heads=heads + kv, head_dim=hd, n_axes=2, pairs=(16, 16, 0, 0), layout=0, ladder=0,
                      inverse=0, base=1000.0, in_token_stride=row, in_head_stride=hd, out_token_stride=row, out_head_stride=hd,
                      pos_stride=n)
    add = P.AppendPush(cache=cache, n_new=n, k_token_stride=row, k_head_stride=hd, v_token_stride=row, v_head_stride=hd)
    one = P.PagedAttnPush(cache=cache, n_heads=heads, left=-1, sinks=0, max_len=length, scale=0.125, q_seq_stride=row,
                          q_head_stride=hd, out_seq_stride=heads * hd, out_head_stride=hd)
    all_ = P.SeqAttnPush(dtype=0, n_seqs=1, n_q=n, n_k=n, n_heads=heads, n_kv_heads=kv, head_dim=hd, left=-1, right=0, sinks=0,
                         scale=0.125, q_token_stride=row, q_head_stride=hd, k_token_stride=row, k_head_stride=hd,
                         v_token_stride=row, v_head_stride=hd, out_token_stride=heads * hd, out_head_stride=hd)
    need = engine.paged_attn_workspace(one)
    pool = normal(rng, (n * width, kv, page, hd), "fp16")
    table = dev.put(rng.permutation(n * width).astype(np.int32))
    seq, at, lens = dev.put(np.arange(n, dtype=np.int32)), dev.put(np.full(n, length - 1, np.int32)), dev.put(np.full(n, length, np.int32))

    def buffers():
        return dict(x=dev.put(np.zeros((n, row), np.uint16)), pos=dev.put(np.arange(2 * n, dtype=np.int32)), k=dev.put(pool),
                    v=dev.put(pool), a=dev.put(np.zeros((n, heads, hd), np.uint16)), b=dev.put(np.zeros((n, heads, hd), np.uint16)),
                    ws=dev.put(np.zeros(need // 2, np.uint16)))

    def calls(d, s):
        engine.rope(turn, d["x"], d["pos"], d["x"], s)
        k, v = d["x"] + 2 * heads * hd, d["x"] + 2 * (heads + kv) * hd
        engine.cache_append(add, k, v, seq, at, table, d["k"], d["v"], s)
        engine.paged_attn(one, d["x"], d["k"], d["v"], table, lens, d["a"], d["ws"], need, s)
        engine.seq_attn(all_, d["x"], k, v, None, None, d["b"], s)

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
        for name in "ab":
            assert (dev.get(caught[name], (n, heads, hd)) == dev.get(eager[name], (n, heads, hd))).all()
    hip.graph_destroy(graph, ready)


def test_two_streams_at_once(hip, engine, dev):
    """The same call on two streams, each with a workspace of its own, many times: always the same bits."""
    rng = np.random.default_rng(13)
    heads, kv, hd, page, length = 8, 8, 32, 16, 4000
    width = length // page
    cache = P.CacheDesc(dtype=P.F16, n_kv_heads=kv, head_dim=hd, page_size=page, n_pages=width, n_seqs=1, table_pages=width)
    push = P.PagedAttnPush(cache=cache, n_heads=heads, left=-1, sinks=0, max_len=length, scale=0.2, q_seq_stride=heads * hd,
                           q_head_stride=hd, out_seq_stride=heads * hd, out_head_stride=hd)
    need = engine.paged_attn_workspace(push)
    k, v = (dev.put(normal(rng, (width, kv, page, hd), "fp16")) for _ in "kv")
    table, lens = dev.put(rng.permutation(width).astype(np.int32)), dev.put(np.array([length], np.int32))
    q = [dev.put(normal(rng, (1, heads, hd), "fp16")) for _ in range(2)]
    out = [[dev.put(np.zeros((heads, hd), np.uint16)) for _ in range(10)] for _ in range(2)]
    ws, streams = [dev.put(np.zeros(need // 2, np.uint16)) for _ in range(2)], [hip.stream() for _ in range(2)]
    hip.sync()
    for i in range(10):
        for j in range(2):
            engine.paged_attn(push, q[j], k, v, table, lens, out[j][i], ws[j], need, streams[j])
    hip.sync()
    for j in range(2):
        first = dev.get(out[j][0], (heads, hd))
        assert np.isfinite(values(first, "fp16")).all() and first.any()
        for o in out[j]:
            assert (dev.get(o, (heads, hd)) == first).all()


def test_refused_calls(hip, engine, dev):
    """Refusals that need a context; nothing runs."""
    import test_seq_rules as R
    a = dev.put(np.zeros(4096, np.uint16))

    def refused(call, *args):
        with pytest.raises(P.PrismError) as e:
            call(*args)
        assert e.value.code in (P.ERR_INVALID, P.ERR_UNSUPPORTED) and engine.error()

    refused(engine.rope, R.rope(), None, a, a)
    refused(engine.rope, R.rope(), a, None, a)
    refused(engine.rope, R.rope(), a + 2, a, a)
    refused(engine.rope, R.rope(in_token_stride=256), a, a, a)  # in place with unequal strides
    refused(engine.rope, R.rope(head_dim=12), a, a, a)
    refused(engine.cache_append, R.append(), a, a, a, a, None, a, a)
    refused(engine.cache_append, R.append(), a, a + 8, a, a, a, a, a)
    refused(engine.cache_append, R.append(n_new=-1), a, a, a, a, a, a, a)
    refused(engine.paged_attn, R.paged(), None, a, a, a, a, a, a, 1 << 20)
    refused(engine.paged_attn, R.paged(), a, a, None, a, a, a, a, 1 << 20)
    refused(engine.paged_attn, R.paged(), a, a, a, a, a, a + 4, a, 1 << 20)
    long = R.paged(cache=R.cache(n_seqs=1, table_pages=1000), max_len=16000)
    need = engine.paged_attn_workspace(long)
    assert need > 0
    refused(engine.paged_attn, long, a, a, a, a, a, a, a, need - 1)
    refused(engine.paged_attn, long, a, a, a, a, a, a, None, need)
    refused(engine.paged_attn, long, a, a, a, a, a, a, a + 4, need)
    refused(engine.seq_attn, R.seq(), a, None, a, a, a, a)
    refused(engine.seq_attn, R.seq(n_seqs=3), a, a, a, None, None, a)  # 10 rows are not 3 equal sequences
    refused(engine.seq_attn, R.seq(n_kv_heads=3), a, a, a, a, a, a)
    # more threads than a launch has
    refused(engine.cache_append, R.append(cache=R.cache(n_kv_heads=65536), n_new=2 ** 30), a, a, a, a, a, a, a)
    refused(engine.paged_attn, R.paged(cache=R.cache(n_seqs=2 ** 30), out_seq_stride=128), a, a, a, a, a, a, a, 0)
    refused(engine.seq_attn, R.seq(n_seqs=MAX), a, a, a, a, a, a)
    # calls without rows are fine, whatever the buffers are
    engine.rope(R.rope(n_tokens=0), None, None, None)
    engine.cache_append(R.append(n_new=0), *[None] * 7)
    engine.paged_attn(R.paged(cache=R.cache(n_seqs=0)), *[None] * 7, 0)
    engine.seq_attn(R.seq(n_q=0), *[None] * 6)
    engine.seq_attn(R.seq(n_seqs=0), *[None] * 6)


def test_no_keys_at_all(engine, dev):
    """Caches without pages and sequences without keys: zeros."""
    import test_seq_rules as R
    q = dev.put(np.ones(3 * 4 * 32, np.uint16))
    for c in (dict(n_pages=0), dict(table_pages=0)):
        out = dev.put(np.full(3 * 4 * 32, NAN["fp16"], np.uint16))
        push = R.paged(cache=R.cache(**c), max_len=0)
        need = engine.paged_attn_workspace(push)
        ws = dev.put(np.zeros(need // 2, np.uint16))
        engine.paged_attn(push, q, None, None, None, dev.put(np.full(3, 9, np.int32)), out, ws, need)
        assert not dev.get(out, 3 * 4 * 32).any()
    out = dev.put(np.full(10 * 4 * 64, NAN["bf16"], np.uint16))
    engine.seq_attn(R.seq(n_k=0), dev.put(np.ones(10 * 4 * 64, np.uint16)), None, None, None, None, out)
    assert not dev.get(out, 10 * 4 * 64).any()
