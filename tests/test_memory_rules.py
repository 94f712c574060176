"""Checks of arguments of the 4-bit cache and of linear attention, on the CPU, the C entries' refusals that
need no device, and the tests' own definition of a 4-bit block against searched values."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import prism_amd as P
from conftest import ROOT
from memlib import MAGNITUDES, POWERS, dequantise, quantise

MAX = 2 ** 31 - 1
nan, inf = float("nan"), float("inf")
STRIDES = [-8, 4, 2 ** 41]


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("memory") / "memory_rules.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-shared", "-fPIC", "-I", os.path.join(ROOT, "include"),
                    os.path.join(ROOT, "tests", "memory_rules.cpp"), "-o", so], check=True, timeout=120)
    return C.CDLL(so)


def cache(**kw):
    d = dict(dtype=P.F16, n_kv_heads=2, head_dim=32, page_size=16, n_pages=9, n_seqs=3, table_pages=4)
    return P.CacheDesc(**{**d, **kw})


def rope_append(**kw):
    d = dict(cache=cache(), format=P.CACHE_4, n_new=5, n_heads=4, n_axes=3, pairs=(4, 6, 6, 0), layout=0, ladder=0,
             base=10000.0, q_token_stride=256, q_head_stride=32, k_token_stride=256, k_head_stride=32, v_token_stride=256,
             v_head_stride=32, out_token_stride=128, out_head_stride=32, pos_stride=5)
    return P.RopeAppendPush(**{**d, **kw})


def cache_read(**kw):
    d = dict(cache=cache(), format=P.CACHE_4, n_rows=5, k_token_stride=64, k_head_stride=32, v_token_stride=64,
             v_head_stride=32)
    return P.CacheReadPush(**{**d, **kw})


def linear(**kw):
    d = dict(dtype=P.BF16, n_seqs=5, n_tokens=5, n_heads=4, n_kv_heads=2, head_dim=64, n_states=6, scale=0.2,
             q_token_stride=256, q_head_stride=64, k_token_stride=128, k_head_stride=64, v_token_stride=128,
             v_head_stride=64, out_token_stride=256, out_head_stride=64)
    return P.LinearAttnPush(**{**d, **kw})


CACHES = [dict(dtype=3), dict(n_kv_heads=0), dict(head_dim=48), dict(head_dim=256), dict(head_dim=8), dict(page_size=0),
          dict(page_size=24), dict(page_size=8192), dict(n_pages=-1), dict(n_seqs=-1), dict(table_pages=-1),
          dict(table_pages=2 ** 18 + 1, page_size=4096)]


@pytest.mark.parametrize("bad", [dict(cache=cache(**c)) for c in CACHES] + [
    dict(format=2), dict(format=-1), dict(n_new=-1), dict(n_heads=-1), dict(n_heads=65537), dict(n_axes=-1), dict(n_axes=5),
    dict(pairs=(5, 6, 6, 0)), dict(pairs=(0, 0, 0, 4)), dict(pairs=(4, -1, 6, 0)), dict(pairs=(MAX, MAX, 6, 0)), dict(layout=2),
    dict(ladder=-1), dict(base=0.5), dict(base=nan), dict(base=inf), dict(pos_stride=-1), dict(out_token_stride=64),
    dict(out_head_stride=16), dict(n_new=2 ** 30, q_token_stride=2 ** 40),
] + [{f: s} for f in ("q_token_stride", "q_head_stride", "k_token_stride", "k_head_stride", "v_token_stride",
                      "v_head_stride", "out_token_stride", "out_head_stride") for s in STRIDES])
def test_rope_append_refusals(rules, bad):
    assert rules.rope_append_check(C.byref(rope_append(**bad))) < 0


@pytest.mark.parametrize("good", [
    {}, dict(n_new=0), dict(n_heads=0, q_token_stride=-1, out_token_stride=0), dict(n_axes=0, pairs=(-9, 0, 0, 0), base=nan),
    dict(format=P.CACHE_16), dict(n_axes=1, pairs=(16, 99, 0, 0)), dict(q_token_stride=0, k_head_stride=0),
])
def test_rope_append_accepts(rules, good):
    assert rules.rope_append_check(C.byref(rope_append(**good))) == 0


@pytest.mark.parametrize("bad", [dict(cache=cache(**c)) for c in CACHES] + [
    dict(format=2), dict(n_rows=-1), dict(k_token_stride=32), dict(v_token_stride=0), dict(k_head_stride=16),
] + [{f: s} for f in ("k_token_stride", "k_head_stride", "v_token_stride", "v_head_stride") for s in STRIDES])
def test_cache_read_refusals(rules, bad):
    assert rules.cache_read_check(C.byref(cache_read(**bad))) < 0
    assert rules.cache_read_check(C.byref(cache_read())) == 0


@pytest.mark.parametrize("bad", [
    dict(dtype=9), dict(n_seqs=-1), dict(n_tokens=-1), dict(n_states=-1), dict(n_heads=3), dict(n_kv_heads=0), dict(head_dim=40),
    dict(n_tokens=2 ** 30 + 1), dict(scale=nan), dict(scale=inf), dict(out_token_stride=192), dict(out_head_stride=32),
    dict(n_states=MAX, n_heads=65536, head_dim=128),
] + [{f: s} for f in ("q_token_stride", "q_head_stride", "k_head_stride", "v_token_stride", "out_token_stride")
     for s in STRIDES])
def test_linear_refusals(rules, bad):
    assert rules.linear_check(C.byref(linear(**bad))) < 0
    assert rules.linear_step_check(C.byref(linear(**bad))) < 0
    assert P.lib().prism_linear_attn_workspace(C.byref(linear(**bad))) < 0
    assert rules.linear_check(C.byref(linear(scale=-1.0, n_states=0))) == 0


def test_a_step_is_one_token_a_sequence(rules):
    assert rules.linear_step_check(C.byref(linear())) == 0
    assert rules.linear_check(C.byref(linear(n_tokens=10))) == 0
    assert rules.linear_step_check(C.byref(linear(n_tokens=10))) < 0


def test_entries_without_a_context():
    lib, pages = P.lib(), P.CachePages()
    assert lib.prism_rope_append(None, C.byref(rope_append()), *[None] * 8, C.byref(pages), None) == P.ERR_INVALID
    assert lib.prism_cache_read(None, C.byref(cache_read()), C.byref(pages), *[None] * 6) == P.ERR_INVALID
    assert lib.prism_paged_attn4(None, None, None, C.byref(pages), *[None] * 4, 0, None) == P.ERR_INVALID
    assert lib.prism_linear_attn(None, C.byref(linear()), *[None] * 10, 0, None) == P.ERR_INVALID
    assert lib.prism_linear_step(None, C.byref(linear()), *[None] * 9) == P.ERR_INVALID
    assert lib.prism_paged_attn4_workspace(None) == P.ERR_INVALID
    assert lib.prism_linear_attn_workspace(None) == P.ERR_INVALID
    assert lib.prism_linear_attn_workspace(C.byref(linear())) >= 0


def numbers(call, push, n):
    out = (C.c_int64 * n)()
    call(C.byref(push), out)
    return list(out)


@pytest.mark.parametrize("hd", [16, 32, 64, 128])
def test_tokens_that_are_turned_together(rules, hd):
    """Fit their tables in LDS, at any size, and are never none."""
    most = rules.append_tile_channels() // hd
    for n in (1, 255, 256, 8160, 10 ** 6, MAX):
        for heads in (1, 3, 24, 65536 + 2 * 65536):
            tile = rules.append_tile_of(C.c_int64(n), C.c_int64(heads), hd)
            assert 1 <= tile <= most and tile & (tile - 1) == 0


@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("kv,group", [(1, 1), (8, 1), (2, 3), (1, 65536), (8, 4)])
def test_splits_of_a_long_cache(rules, hd, kv, group):
    """All keys expected have a wave, whole tiles each; splits are what the joining launch has room for and an odd number."""
    for n in (1, 5, 64, 8160):
        for page, pages in ((1, 1), (16, 4), (16, 1000), (64, 3000), (4096, 2 ** 18)):
            for max_len, left, sinks in ((0, -1, 0), (300, -1, 0), (5000, 0, 0), (0, MAX, MAX), (0, 700, 5), (MAX, -1, 0)):
                p = P.PagedAttnPush(cache=cache(n_kv_heads=kv, head_dim=hd, page_size=page, n_pages=9, n_seqs=n, table_pages=pages),
                                    n_heads=kv * group, left=left, sinks=sinks, max_len=max_len, scale=1.0)
                many, tiles, waves, splits, grid, each, keys, space = numbers(rules.paged4_of, p, 8)
                assert tiles * 16 >= group and waves in (1, 4) and 1 <= splits <= 95 and splits % 2 == 1
                assert many or (group <= 2 and hd <= 32)
                assert each % 64 == 0 and each > 0 and (4 * splits * each >= keys or each == 2 ** 30)
                assert grid == (-(-n * kv * tiles // 4) if waves == 1 else n * kv * tiles * splits) and (waves == 4 or splits == 1)
                assert space == (0 if splits == 1 else n * kv * group * splits * (hd + 2) * 4)


@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("heads", [1, 5, 32])
def test_segments_of_long_sequences(rules, hd, heads):
    """Whole chunks, and a number for each of them whatever the lengths: sequence s has those from start / segment + s on."""
    rng = np.random.default_rng(hd)
    for n, tokens in ((1, 1), (1, 255), (1, 256), (1, 8160), (3, 1000), (9, 3), (64, 64000), (1, 2 ** 30), (511, 2 ** 20), (2, 0)):
        p = linear(n_seqs=n, n_tokens=tokens, n_heads=heads, n_kv_heads=heads, head_dim=hd)
        segment, split, segments, space = numbers(rules.linear_of, p, 4)
        assert space == (segments * heads * hd * hd * 4 if split else 0)
        if not split:
            assert segments == n and segment == MAX
            continue
        assert segment % 64 == 0 and segment > 0
        for _ in range(20):
            cuts = np.sort(rng.integers(0, tokens + 1, n + 1))
            first = cuts[:-1] // segment + np.arange(n)
            last = first + np.maximum(np.diff(cuts) - 1, 0) // segment
            assert last[-1] < segments and (last[:-1] < first[1:]).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_the_definition_of_a_block(dtype):
    """Against a search over all sixteen numbers; what fits comes back as it was."""
    rng = np.random.default_rng(1)
    low, high = POWERS[dtype]
    for e in (low, low + 1, -3, 0, 5, high):
        x = rng.standard_normal((7, 64)).astype(np.float32) * np.float32(2.0 ** e)
        codes, scales = quantise(x, dtype)
        back = dequantise(codes, scales)
        for row, b, s in zip(x, back, scales):
            for i in range(2):
                part, power = row[32 * i:32 * i + 32].astype(np.float64), 2.0 ** (float(s[i]) - 127)
                assert np.abs(part).max() <= 7 * power or s[i] == high + 127
                assert s[i] == low + 127 or np.abs(part).max() > 3.5 * power
                grid = np.concatenate((MAGNITUDES, -MAGNITUDES)) * power
                assert (np.abs(b[32 * i:32 * i + 32] - part) == np.abs(grid - part[:, None]).min(1)).all()
        again = quantise(back.astype(np.float32), dtype)
        assert (dequantise(*again) == back).all()
    borders = np.array([6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, -.25, -.75, -1.25, -1.75, -2.5, -3.5, -5, -0.0], np.float32)
    codes, scales = quantise(borders, dtype)
    assert (dequantise(codes, scales) == [6, 0, 1, 1, 2, 2, 4, 4, 0, -1, -1, -2, -2, -4, -4, 0]).all() and scales == 127
    assert codes[-1] >> 4 == 8  # a zero keeps its sign


@pytest.mark.parametrize("field", ["q_token_stride", "k_token_stride", "v_token_stride", "out_token_stride"])
def test_linear_token_strides(rules, field):
    """Rows of a chunk are addressed with 32 bits: 2^22 elements from one to the next, at most."""
    for call in (rules.linear_check, rules.linear_step_check):
        assert call(C.byref(linear(**{field: 2 ** 22}))) == 0
        assert call(C.byref(linear(**{field: 2 ** 22 + 8}))) == P.ERR_UNSUPPORTED
        for bad in STRIDES:
            assert call(C.byref(linear(**{field: bad}))) < 0
    assert P.lib().prism_linear_attn_workspace(C.byref(linear(**{field: 2 ** 22 + 8}))) == P.ERR_UNSUPPORTED


@pytest.mark.parametrize("hd,kv,group,lengths,max_len,splits", [(32, 2, 1, 2, 100, 1), (128, 1, 4, 2, 100, 1), (32, 1, 2, 2, 2000, 5),
                                                                (64, 1, 1, 2, 2000, 5), (128, 2, 4, 2, 2000, 5)])
def test_a_wave_of_a_cache_longer_than_expected(rules, hd, kv, group, lengths, max_len, splits):
    """The calls of test_paged4_longer_than_expected are of four waves, with these splits."""
    p = P.PagedAttnPush(cache=cache(n_kv_heads=kv, head_dim=hd, page_size=64, n_seqs=lengths, table_pages=97), n_heads=kv * group,
                        left=-1, max_len=max_len, scale=1.0)
    many, _, waves, got, _, each, _, _ = numbers(rules.paged4_of, p, 8)
    assert waves == 4 and got == splits and many == (group > 2 or hd > 32) and 4 * splits * each < 6000
