"""Paths of the sequence operators that the choice of kernels takes at sizes of their own, on the GPU: several tokens a
workgroup, waves that work alone, runs of heads per XCD, few queries behind many keys; and calls on other streams and from
other threads. Definitions and bounds as in test_gpu_sequence.py."""
import ctypes as C
import math
import threading

import numpy as np
import pytest

import prism_amd as P
from seqlib import NAN, TYPES, attention_row, normal, values, visible
from test_gpu_sequence import FILL, LENGTHS, check_paged, check_seq, dev, outside, rope_ref  # noqa: F401 (dev: fixture)
from test_seq_rules import rules  # noqa: F401 (fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,heads,hd,pairs,layout,ladder,inverse", [
    (2049, 3, 32, (4, 6, 6), P.ROPE_HALVES, 0, 0),    # whole chunks of 8 pairs
    (4099, 2, 64, (8, 8, 8), P.ROPE_HALVES, 1, 1),    # and channels that do not turn
    (20_001, 1, 24, (8,), P.ROPE_HALVES, 0, 0),       # rows of an odd number of chunks
    (2049, 5, 128, (24, 20, 11), P.ROPE_HALVES, 0, 0),  # pairs that do not fill chunks: rows through LDS
    (4099, 3, 72, (11, 0, 14), P.ROPE_HALVES, 1, 1),  # rows that do not fill the workgroup's threads
    (20_001, 1, 24, (3, 4, 2), P.ROPE_HALVES, 0, 0), (5001, 2, 8, (3,), P.ROPE_HALVES, 0, 0),
    (2049, 3, 32, (4, 6, 6), P.ROPE_ADJACENT, 0, 1), (4099, 3, 72, (11, 0, 14), P.ROPE_ADJACENT, 1, 0),
    (20_001, 1, 24, (3, 4, 2), P.ROPE_ADJACENT, 0, 0), (4099, 2, 128, (1, 1, 1, 1), P.ROPE_ADJACENT, 0, 0),
    (40_003, 2, 16, (2, 3, 3), P.ROPE_ADJACENT, 0, 0),
])
def test_rope_several_tokens_a_workgroup(engine, dev, rules, dtype, tokens, heads, hd, pairs, layout, ladder, inverse):  # noqa: F811
    tile = rules.tile(tokens, sum(pairs))
    assert tile > 1 and tokens % tile  # the last workgroup has fewer
    rng = np.random.default_rng(tokens + hd)
    rows = normal(rng, (tokens, heads + 1, hd), dtype)
    pos = rng.integers(-50, 5000, (len(pairs), tokens)).astype(np.int32)
    x, p, y = dev.put(rows), dev.put(pos), dev.put(np.full((tokens + 2, heads, hd), NAN[dtype], np.uint16))
    push = P.RopePush(dtype=TYPES[dtype], n_tokens=tokens, n_heads=heads, head_dim=hd, n_axes=len(pairs),
                      pairs=pairs + (0,) * (4 - len(pairs)), layout=layout, ladder=ladder, inverse=inverse, base=10000.0,
                      in_token_stride=(heads + 1) * hd, in_head_stride=hd, out_token_stride=heads * hd, out_head_stride=hd,
                      pos_stride=tokens)
    print(f"[rope] {dtype} layout {layout} {tokens} x {heads} x {hd}, {tile} tokens a workgroup", flush=True)
    engine.rope(push, x, p, y)
    got = dev.get(y, (tokens + 2, heads, hd))
    assert (got[tokens:] == NAN[dtype]).all()
    got = got[:tokens]
    want, bound = rope_ref(values(rows[:, :heads], dtype), pos, pairs, layout, ladder, inverse, 10000.0, dtype)
    assert not outside(values(got, dtype), want, bound)
    assert (got[..., 2 * sum(pairs):] == rows[:, :heads, 2 * sum(pairs):]).all()
    push.out_token_stride = push.in_token_stride
    engine.rope(push, x, p, x)  # in place: the same bits, the other heads untouched
    there = dev.get(x, rows.shape)
    assert (there[:, :heads] == got).all() and (there[:, heads:] == rows[:, heads:]).all()


def paged_waves(rules, n_seqs, kv, group, hd, max_len):  # noqa: F811
    out = (C.c_longlong * 6)()
    rules.paged(C.byref(P.PagedAttnPush(
        cache=P.CacheDesc(dtype=0, n_kv_heads=kv, head_dim=hd, page_size=16, n_pages=9, n_seqs=n_seqs, table_pages=99),
        n_heads=kv * group, left=-1, sinks=0, max_len=max_len, scale=1.0, q_seq_stride=kv * group * hd, q_head_stride=hd,
        out_seq_stride=kv * group * hd, out_head_stride=hd)), out)
    return out[2]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("kv,group", [(8, 1), (2, 2), (1, 3), (2, 4), (1, 17)])
def test_paged_a_wave_alone(engine, dev, rules, dtype, hd, kv, group):  # noqa: F811
    """Announced as short (and then longer, too): every kernel with a wave for each item."""
    assert paged_waves(rules, len(LENGTHS), kv, group, hd, 16) == 1
    check_paged(engine, dev, np.random.default_rng(hd + 7 * group), dtype, hd, kv, group, 16, LENGTHS, -1, 0, max_len=16)


@pytest.mark.parametrize("hd,kv,group,seqs", [(32, 3, 1, 1367), (16, 1, 3, 4097), (64, 3, 2, 1367)])
def test_paged_many_items(engine, dev, rules, hd, kv, group, seqs):  # noqa: F811
    """So many sequences that each has a wave, however long; the last workgroup is not full."""
    assert paged_waves(rules, seqs, kv, group, hd, 100) == 1 and seqs * kv >= 4096 and seqs * kv % 4
    rng = np.random.default_rng(hd)
    lengths = [int(x) for x in rng.integers(0, 9, seqs)]
    lengths[seqs // 2], lengths[-1] = 100, 77
    check_paged(engine, dev, rng, "fp16", hd, kv, group, 4, lengths, 40, 3, max_len=100)


@pytest.mark.parametrize("hd,kv,group", [(16, 16, 1), (32, 24, 2), (128, 16, 2), (64, 32, 1)])
@FILL
def test_seq_heads_of_an_xcd(engine, dev, hd, kv, group, fill):  # noqa: F811
    """16 groups of heads and more, a multiple of 8: each XCD takes several."""
    check_seq(engine, dev, np.random.default_rng(hd), "bf16", hd, kv, group, [(9, 20), (1, 1), (0, 3), (130, 131)], 25, 0, 2, fill=fill)


@pytest.mark.parametrize("dtype,hd,kv,group,lens,left,sinks", [
    ("fp16", 32, 2, 1, [(5, 30_000)], -1, 0), ("bf16", 128, 1, 4, [(17, 9001), (1, 20_001)], -1, 0),
    ("fp16", 64, 1, 8, [(3, 12_345), (0, 100), (33, 2049)], 7000, 100), ("bf16", 16, 1, 1, [(130, 5000)], -1, 0),
])
@FILL
def test_seq_few_queries_behind_many_keys(engine, dev, dtype, hd, kv, group, lens, left, sinks, fill):  # noqa: F811
    check_seq(engine, dev, np.random.default_rng(hd), dtype, hd, kv, group, lens, left, 0, sinks, fill=fill)


def test_calls_of_several_threads(hip, dev):  # noqa: F811
    """Four threads, each with a context, a stream and buffers of its own, call the operators at once: each gets its own
    results, and the refusals of one do not reach another's calls."""
    heads, kv, hd, n, calls = 4, 2, 64, 700, 20
    st = dict(q_token_stride=heads * hd, q_head_stride=hd, k_token_stride=kv * hd, k_head_stride=hd, v_token_stride=kv * hd,
              v_head_stride=hd, out_token_stride=heads * hd, out_head_stride=hd)
    push = P.SeqAttnPush(dtype=P.F16, n_seqs=1, n_q=n, n_k=n, n_heads=heads, n_kv_heads=kv, head_dim=hd, left=100, right=0, sinks=2,
                         scale=0.125, **st)
    wrong = P.SeqAttnPush(dtype=P.F16, n_seqs=1, n_q=n, n_k=n, n_heads=3, n_kv_heads=kv, head_dim=hd, left=100, right=0, sinks=2,
                          scale=0.125, **st)
    data, outs, streams, failed = [], [], [hip.stream() for _ in range(4)], []
    for t in range(4):
        rng = np.random.default_rng(t)
        data.append([normal(rng, (n, h, hd), "fp16") for h in (heads, kv, kv)])
        outs.append([dev.put(np.full((n, heads, hd), NAN["fp16"], np.uint16)) for _ in range(calls)])
    ptrs = [[dev.put(a) for a in d] for d in data]
    engines = [P.Engine(0) for _ in range(4)]
    hip.sync()

    def work(t):
        try:
            for i in range(calls):
                engines[t].seq_attn(push, *ptrs[t], None, None, outs[t][i], streams[t])
                if t == 0:
                    with pytest.raises(P.PrismError):
                        engines[t].seq_attn(wrong, *ptrs[t], None, None, outs[t][i], streams[t])
        except BaseException as e:  # a thread's own exceptions do not reach the test
            failed.append(e)

    threads = [threading.Thread(target=work, args=(t,)) for t in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    hip.sync()
    for e in engines:
        e.close()
    assert not failed
    for t in range(4):
        first = dev.get(outs[t][0], (n, heads, hd))
        for o in outs[t][1:]:
            assert (dev.get(o, first.shape) == first).all()
        q, k, v = (values(a, "fp16") for a in data[t])
        got = values(first, "fp16")
        for i in range(0, n, 37):
            for h in range(heads):
                want, bound = attention_row(q[i, h], k[:, h // 2], v[:, h // 2], visible(i, n, 100, 0, 2), 0.125, "fp16")
                assert not outside(got[i, h], want, bound), (t, i, h)


def test_two_graphs_that_share_a_workspace(hip, engine, dev):  # noqa: F811
    """Two captured calls of unlike splits with one workspace, replayed in turn on one stream: the eager calls' bits."""
    rng = np.random.default_rng(3)
    heads, kv, hd, page, n, width = 8, 2, 64, 16, 2, 250
    cache = P.CacheDesc(dtype=P.F16, n_kv_heads=kv, head_dim=hd, page_size=page, n_pages=n * width, n_seqs=n, table_pages=width)
    pushes = [P.PagedAttnPush(cache=cache, n_heads=heads, left=left, sinks=0, max_len=4000, scale=1 / math.sqrt(hd),
                              q_seq_stride=heads * hd, q_head_stride=hd, out_seq_stride=heads * hd, out_head_stride=hd)
              for left in (-1, 900)]
    needs = [engine.paged_attn_workspace(p) for p in pushes]
    assert min(needs) > 0 and needs[0] != needs[1]
    ws = dev.put(np.full(max(needs) // 2, NAN["fp16"], np.uint16))
    k, v = (dev.put(normal(rng, (n * width, kv, page, hd), "fp16")) for _ in "kv")
    table, lens = dev.put(rng.permutation(n * width).astype(np.int32)), dev.put(np.array([4000, 2711], np.int32))
    q = dev.put(np.zeros((n, heads, hd), np.uint16))
    out, eager = ([dev.put(np.zeros((n, heads, hd), np.uint16)) for _ in pushes] for _ in range(2))
    s, ready = hip.stream(), []
    hip.sync()
    for p, o, need in zip(pushes, out, needs):
        hip.begin_capture(s)
        engine.paged_attn(p, q, k, v, table, lens, o, ws, need, s)
        graph = hip.end_capture(s)
        ready.append((graph, hip.graph_instantiate(graph)))
    for _ in range(4):
        hip.upload(q, normal(rng, (n, heads, hd), "fp16"))
        for _, g in ready + ready:
            hip.graph_launch(g, s)
        hip.stream_sync(s)
        for p, o, need in zip(pushes, eager, needs):
            engine.paged_attn(p, q, k, v, table, lens, o, ws, need)
        for a, b in zip(out, eager):
            first = dev.get(a, (n, heads, hd))
            assert first.any() and (first == dev.get(b, (n, heads, hd))).all()
    for graph, g in ready:
        hip.graph_destroy(graph, g)
