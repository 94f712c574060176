"""The sequence operators' checks of arguments and index arithmetic, on the CPU (csrc/engine/seq_rules.h,
csrc/seq_index.h), and the C entries' refusals that need no device."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import prism_amd as P
from conftest import ROOT
from seqlib import visible

MAX = 2 ** 31 - 1


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("seq") / "seq_rules.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-shared", "-fPIC", "-I", os.path.join(ROOT, "include"),
                    os.path.join(ROOT, "tests", "seq_rules.cpp"), "-o", so], check=True, timeout=120)
    lib = C.CDLL(so)
    lib.rows.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_void_p]
    lib.tile.argtypes = [C.c_longlong, C.c_int]
    lib.seq_tiles.argtypes, lib.seq_tiles.restype = [C.c_longlong, C.c_longlong, C.c_int], C.c_longlong
    lib.grid_ok.argtypes = [C.c_longlong, C.c_int]
    return lib


def rope(**kw):
    d = dict(dtype=P.F16, n_tokens=5, n_heads=4, head_dim=32, n_axes=3, pairs=(4, 6, 6, 0), layout=0, ladder=0, inverse=0,
             base=10000.0, in_token_stride=128, in_head_stride=32, out_token_stride=128, out_head_stride=32, pos_stride=5)
    return P.RopePush(**{**d, **kw})


def cache(**kw):
    d = dict(dtype=P.F16, n_kv_heads=2, head_dim=32, page_size=16, n_pages=9, n_seqs=3, table_pages=4)
    return P.CacheDesc(**{**d, **kw})


def append(**kw):
    d = dict(cache=cache(), n_new=5, k_token_stride=64, k_head_stride=32, v_token_stride=64, v_head_stride=32)
    return P.AppendPush(**{**d, **kw})


def paged(**kw):
    d = dict(cache=cache(), n_heads=4, left=-1, sinks=0, max_len=64, scale=0.2, q_seq_stride=128, q_head_stride=32,
             out_seq_stride=128, out_head_stride=32)
    return P.PagedAttnPush(**{**d, **kw})


def seq(**kw):
    d = dict(dtype=P.BF16, n_seqs=2, n_q=10, n_k=20, n_heads=4, n_kv_heads=2, head_dim=64, left=-1, right=0, sinks=0,
             scale=0.2, q_token_stride=256, q_head_stride=64, k_token_stride=128, k_head_stride=64, v_token_stride=128,
             v_head_stride=64, out_token_stride=256, out_head_stride=64)
    return P.SeqAttnPush(**{**d, **kw})


nan, inf = float("nan"), float("inf")
STRIDES = [-8, 4, 2 ** 41]


@pytest.mark.parametrize("bad", [
    dict(dtype=2), dict(dtype=-1), dict(n_tokens=-1), dict(n_heads=0), dict(n_heads=65537), dict(head_dim=12),
    dict(head_dim=264), dict(head_dim=0), dict(n_axes=0), dict(n_axes=5), dict(pairs=(4, -1, 6, 0)), dict(pairs=(0, 0, 0, 9)),
    dict(pairs=(5, 6, 6, 0)), dict(pairs=(MAX, MAX, 6, 0)), dict(layout=2), dict(ladder=-1), dict(inverse=2), dict(base=0.0),
    dict(base=-3.0), dict(base=0.99), dict(base=nan), dict(base=inf), dict(pos_stride=-1), dict(out_token_stride=64),
    dict(out_head_stride=0), dict(out_head_stride=16), dict(out_token_stride=0),
] + [{f: s} for f in ("in_token_stride", "in_head_stride", "out_token_stride", "out_head_stride") for s in STRIDES])
def test_rope_refusals(rules, bad):
    assert rules.rope_check(C.byref(rope(**bad))) < 0


@pytest.mark.parametrize("good", [
    {}, dict(n_tokens=0), dict(head_dim=8, pairs=(1, 0, 2, 0)), dict(head_dim=256, out_head_stride=256, out_token_stride=1024),
    dict(in_head_stride=0), dict(in_token_stride=0), dict(out_head_stride=160, out_token_stride=32),  # heads outermost
    dict(n_axes=1, pairs=(16, 99, 0, 0)), dict(n_axes=4, pairs=(4, 4, 4, 4)), dict(base=1.0), dict(pos_stride=0),
])
def test_rope_accepts(rules, good):
    assert rules.rope_check(C.byref(rope(**good))) == 0


CACHES = [dict(dtype=3), dict(n_kv_heads=0), dict(head_dim=48), dict(head_dim=256), dict(page_size=0), dict(page_size=24),
          dict(page_size=8192), dict(page_size=-16), dict(n_pages=-1), dict(n_seqs=-1), dict(table_pages=-1),
          dict(table_pages=2 ** 18 + 1, page_size=4096)]


@pytest.mark.parametrize("bad", [dict(cache=cache(**c)) for c in CACHES] + [dict(n_new=-1)] +
                         [{f: s} for f in ("k_token_stride", "k_head_stride", "v_token_stride", "v_head_stride")
                          for s in STRIDES])
def test_append_refusals(rules, bad):
    assert rules.append_check(C.byref(append(**bad))) < 0
    assert rules.append_check(C.byref(append())) == 0


@pytest.mark.parametrize("bad", [dict(cache=cache(**c)) for c in CACHES] + [
    dict(n_heads=0), dict(n_heads=5), dict(n_heads=-2), dict(n_heads=65538), dict(sinks=-1), dict(max_len=-1), dict(scale=0.0),
    dict(scale=-1.0), dict(scale=nan), dict(scale=inf), dict(scale=3e38), dict(out_head_stride=16), dict(out_seq_stride=96),
] + [{f: s} for f in ("q_seq_stride", "q_head_stride", "out_seq_stride", "out_head_stride") for s in STRIDES])
def test_paged_refusals(rules, bad):
    assert rules.paged_check(C.byref(paged(**bad))) < 0
    assert P.lib().prism_paged_attn_workspace(C.byref(paged(**bad))) < 0
    assert rules.paged_check(C.byref(paged())) == 0


@pytest.mark.parametrize("bad", [
    dict(dtype=9), dict(n_seqs=-1), dict(n_q=-1), dict(n_k=-1), dict(n_heads=3), dict(n_kv_heads=0), dict(head_dim=40),
    dict(k_token_stride=2 ** 22 + 8), dict(v_token_stride=2 ** 22 + 8), dict(n_q=2 ** 30 + 1), dict(n_k=MAX), dict(sinks=-2),
    dict(scale=0.0), dict(scale=nan), dict(scale=3e38), dict(out_token_stride=192), dict(out_head_stride=32),
] + [{f: s} for f in ("q_token_stride", "k_head_stride", "v_token_stride", "out_token_stride") for s in STRIDES])
def test_seq_refusals(rules, bad):
    assert rules.seq_check(C.byref(seq(**bad))) < 0
    assert rules.seq_check(C.byref(seq())) == 0


def test_entries_without_a_context():
    lib = P.lib()
    assert lib.prism_rope(None, C.byref(rope()), None, None, None, None) == P.ERR_INVALID
    assert lib.prism_cache_append(None, C.byref(append()), *[None] * 8) == P.ERR_INVALID
    assert lib.prism_paged_attn(None, C.byref(paged()), *[None] * 7, 0, None) == P.ERR_INVALID
    assert lib.prism_seq_attn(None, C.byref(seq()), *[None] * 7) == P.ERR_INVALID
    assert lib.prism_paged_attn_workspace(None) == P.ERR_INVALID
    assert lib.prism_paged_attn_workspace(C.byref(paged())) >= 0


def test_keys_a_query_sees(rules):
    """Against the definition, for every small position, window and number of sinks."""
    out = (C.c_int32 * 3)()
    for n in (0, 1, 2, 5, 9):
        for p in range(-4, n + 3):
            for left in (-1, 0, 1, 3, 20):
                for right in (-1, 0, 2, 20):
                    for sinks in (0, 1, 4, 30):
                        rules.keys(p, n, left, right, sinks, out)
                        sink, lo, hi = out
                        assert 0 <= sink <= lo <= hi <= n
                        got = np.zeros(n, bool)
                        got[:sink] = True
                        got[lo:hi] = True
                        assert (got == visible(p, n, left, right, sinks)).all(), (n, p, left, right, sinks)


@pytest.mark.parametrize("p,n,left,right,sinks,want", [
    (MAX - 1, MAX, MAX, MAX, MAX, (0, 0, MAX)), (MAX - 1, MAX, 0, 0, MAX, (MAX - 1, MAX - 1, MAX)),
    (-MAX, 5, MAX, 0, 4, (0, 0, 0)), (-MAX, 5, MAX, MAX, 4, (0, 0, 1)),
])
def test_keys_at_the_ends_of_the_range(rules, p, n, left, right, sinks, want):
    out = (C.c_int32 * 3)()
    rules.keys(p, n, left, right, sinks, out)
    assert tuple(out) == want


@pytest.mark.parametrize("cu,n", [([0, 3, 3, 10], 10), ([0, 30, -5, 10], 10), ([-7, -7, MAX, 4], 10), ([9, 8, 7, 6], 10),
                                  ([0, 0, 0, 0], 0), ([2, 4, 6, 8], 10)])
def test_rows_stay_in_range(rules, cu, n):
    a = np.array(cu, np.int32)
    out = (C.c_int32 * 2)()
    for s in range(3):
        rules.rows(a.ctypes.data, s, 3, n, out)
        assert 0 <= out[0] <= out[1] <= n
        if 0 <= cu[s] <= cu[s + 1] <= n:
            assert (out[0], out[1]) == (cu[s], cu[s + 1])
    rules.rows(None, 2, 3, 12, out)
    assert tuple(out) == (8, 12)


def test_pages_out_of_the_pool(rules):
    assert [rules.page(e, 4) for e in (-2 ** 31, -1, 0, 3, 4, MAX)] == [0, 0, 1, 1, 0, 0]
    assert rules.page(0, 0) == 0


@pytest.mark.parametrize("kw", [{}, dict(n_axes=1, pairs=(16, 3, 3, 3)), dict(pairs=(0, 5, 0, 0)),
                                dict(n_axes=4, pairs=(1, 2, 3, 4))])
def test_pairs_of_an_axis(rules, kw):
    p = rope(**kw)
    end = (C.c_int32 * 4)()
    pairs = list(p.pairs)[:p.n_axes] + [0] * (4 - p.n_axes)
    assert rules.axes(C.byref(p), end) == sum(pairs) and list(end) == list(np.cumsum(pairs))


@pytest.mark.parametrize("tokens,pairs,tile", [(1, 1, 1), (2047, 8, 1), (2048, 8, 2), (10 ** 9, 8, 128), (10 ** 9, 128, 8),
                                               (10 ** 9, 48, 16), (10 ** 9, 9, 64), (130560, 16, 64)])
def test_tokens_of_a_workgroup(rules, tokens, pairs, tile):
    """The table of angles holds them, and the GPU is filled first."""
    assert rules.tile(tokens, pairs) == tile and tile * -(-pairs // 8) * 8 <= 1024


@pytest.mark.parametrize("kw,many,tiles,waves,splits", [
    (dict(n_heads=2), 0, 1, 4, 1), (dict(n_heads=4), 0, 1, 4, 1), (dict(n_heads=6), 1, 1, 4, 1),  # 1, 2, 3 heads a key head
    (dict(n_heads=34), 1, 2, 4, 1),                                                   # 17
    (dict(max_len=33), 0, 1, 4, 1), (dict(max_len=32), 0, 1, 1, 1),
    (dict(max_len=0), 0, 1, 4, 1), (dict(max_len=10 ** 6, left=30), 0, 1, 1, 1),      # the table's 64 | the window's 31 keys
    (dict(max_len=1023), 0, 1, 4, 1), (dict(max_len=1024), 0, 1, 4, 16),              # 32 channels: worth a second launch
    (dict(max_len=2000, left=800, sinks=9), 0, 1, 4, 1), (dict(max_len=16000), 0, 1, 4, 63), (dict(max_len=10 ** 6), 0, 1, 4, 64),
])
def test_paged_plan(rules, kw, many, tiles, waves, splits):
    out = (C.c_longlong * 6)()
    p = paged(out_seq_stride=2048, **kw)
    rules.paged(C.byref(p), out)
    assert list(out)[:4] == [many, tiles, waves, splits]
    items = 3 * 2 * tiles
    assert out[4] == (-(-items // 4) if waves == 1 else items * splits)
    assert out[5] == (0 if splits == 1 else 3 * p.n_heads * splits * 34 * 4) == P.lib().prism_paged_attn_workspace(C.byref(p))


@pytest.mark.parametrize("seqs,kv,max_len,waves,splits", [
    (24, 8, 20001, 4, 10), (1, 8, 131075, 4, 64), (8160, 8, 75, 1, 1), (128, 8, 128, 1, 1), (128, 8, 129, 4, 1), (127, 8, 128, 4, 1),
    (16, 8, 500, 4, 4), (16, 8, 16000, 4, 15), (200, 8, 100000, 4, 1),
])
def test_paged_plan_of_many(rules, seqs, kv, max_len, waves, splits):
    out = (C.c_longlong * 6)()
    rules.paged(C.byref(paged(cache=cache(n_seqs=seqs, n_kv_heads=kv, head_dim=128), n_heads=kv, max_len=max_len)), out)
    assert (out[2], out[3]) == (waves, splits)


@pytest.mark.parametrize("heads,kv,side", [(8, 8, 1), (32, 8, 4), (15, 5, 3), (32, 1, 32), (33, 1, 1), (4096, 1, 1)])
def test_seq_rows_of_a_workgroup(rules, heads, kv, side):
    assert rules.tile_heads(heads, kv) == side and heads % side == 0


def test_seq_tiles_suffice(rules):
    """A sequence's tiles start at floor(start / tile) + its number: enough for its rows before the next one's."""
    rng = np.random.default_rng(0)
    for tile in (4, 42, 128):
        cu = np.concatenate([[rng.integers(0, 300)], rng.integers(0, 400, 50)]).cumsum()
        first = cu[:-1] // tile + np.arange(50)
        need = -(-np.diff(cu) // tile)
        assert (first[:-1] + need[:-1] <= first[1:]).all()
        assert first[-1] + need[-1] <= rules.seq_tiles(int(cu[-1]), 50, tile)


FOUR, EIGHT, NARROW = 0, 1, 2


@pytest.mark.parametrize("kw,kind,side,tile,grid", [  # 2 groups of 2 heads, 64 queries a tile of 128 rows
    (dict(n_seqs=1, n_q=1, n_k=192), NARROW, 2, 32, 2), (dict(n_seqs=1, n_q=1, n_k=191), FOUR, 2, 64, 2),
    (dict(n_seqs=1, n_q=80 * 64, n_k=5120), NARROW, 2, 32, 322), (dict(n_seqs=1, n_q=81 * 64, n_k=5120), EIGHT, 2, 64, 164),  # 160 | 162
    (dict(n_seqs=1, n_q=128 * 64, n_k=384), EIGHT, 2, 64, 258), (dict(n_seqs=1, n_q=128 * 64, n_k=383), FOUR, 2, 64, 258),
    (dict(n_seqs=1, n_q=129 * 64, n_k=1289), FOUR, 2, 64, 260), (dict(n_seqs=1, n_q=129 * 64, n_k=1290), EIGHT, 2, 64, 260),
    (dict(n_seqs=1, n_q=129 * 64, n_k=8000, left=1200), FOUR, 2, 64, 260),
    (dict(n_seqs=1, n_q=384 * 64, n_k=24576), EIGHT, 2, 64, 770), (dict(n_seqs=1, n_q=385 * 64, n_k=24640), FOUR, 2, 64, 772),
    (dict(n_seqs=1, n_q=384 * 64, n_k=24576, head_dim=32), NARROW, 2, 32, 1538),
    (dict(n_seqs=1, n_q=1, n_k=512, head_dim=128, k_head_stride=128, out_head_stride=128, out_token_stride=512), EIGHT, 2, 64, 2),
    (dict(n_heads=32, n_kv_heads=1, n_k=400, out_token_stride=2048), NARROW, 32, 2, 7),
    (dict(n_heads=33, n_kv_heads=1, n_k=400, out_token_stride=4096), NARROW, 1, 64, 66), (dict(n_seqs=0, n_q=0, n_k=0), FOUR, 2, 64, 0),
])
def test_seq_plan(rules, kw, kind, side, tile, grid):
    out = (C.c_longlong * 4)()
    p = seq(**kw)
    assert rules.seq_check(C.byref(p)) == 0
    rules.seq(C.byref(p), out)
    assert list(out) == [kind, side, tile, grid]


def test_launches_fit_32_bits(rules):
    assert [rules.grid_ok(n, 256) for n in (1, 2 ** 24 - 1, 2 ** 24, 2 ** 40)] == [1, 1, 0, 0]
    assert [rules.grid_ok(n, 512) for n in (2 ** 23 - 1, 2 ** 23)] == [1, 0]
