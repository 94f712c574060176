"""Offsets of the sequence operators fit 64 bits: sizes and strides whose product does not are refused (a UBSan build of
csrc/engine/seq_rules.h)."""
import ctypes as C

import pytest

import prism_amd as P
from test_seq_rules import MAX, append, cache, paged, rope, rules, seq  # noqa: F401 (rules: the built checks)

FAR = 2 ** 40


@pytest.mark.parametrize("bad", [
    dict(n_tokens=2 ** 24 + 1, out_token_stride=FAR), dict(n_tokens=MAX, out_token_stride=FAR), dict(n_tokens=MAX, in_token_stride=FAR),
    dict(n_tokens=2 ** 24 + 1, out_token_stride=FAR, out_head_stride=FAR), dict(n_axes=4, n_tokens=MAX, in_token_stride=2 ** 31),
])
def test_rope_offsets(rules, bad):  # noqa: F811
    assert rules.rope_check(C.byref(rope(**bad))) < 0


@pytest.mark.parametrize("bad", [
    dict(n_new=MAX, k_token_stride=FAR), dict(n_new=2 ** 24, v_token_stride=FAR),
    dict(cache=cache(n_pages=MAX, n_kv_heads=65536, page_size=4096, head_dim=128)),
    dict(cache=cache(n_seqs=MAX, table_pages=2 ** 30, page_size=1)),
])
def test_append_offsets(rules, bad):  # noqa: F811
    assert rules.append_check(C.byref(append(**bad))) < 0


@pytest.mark.parametrize("bad", [
    dict(cache=cache(n_seqs=MAX), q_seq_stride=FAR), dict(cache=cache(n_seqs=MAX), out_seq_stride=FAR),
    dict(cache=cache(n_pages=MAX, n_kv_heads=65536, page_size=4096, head_dim=128), n_heads=65536, out_seq_stride=2 ** 23,
         out_head_stride=128),
])
def test_paged_offsets(rules, bad):  # noqa: F811
    assert rules.paged_check(C.byref(paged(**bad))) < 0
    assert P.lib().prism_paged_attn_workspace(C.byref(paged(**bad))) < 0


@pytest.mark.parametrize("bad", [dict(n_q=2 ** 30, q_token_stride=FAR), dict(n_q=2 ** 30, out_token_stride=FAR),
                                 dict(n_q=2 ** 24 + 1, out_token_stride=FAR, out_head_stride=FAR)])
def test_seq_offsets(rules, bad):  # noqa: F811
    assert rules.seq_check(C.byref(seq(**bad))) < 0


def test_strides_of_rows_that_are_not_there(rules):  # noqa: F811
    """One row, one head or none: the stride is not used, whatever it is within 2^40."""
    assert rules.rope_check(C.byref(rope(n_tokens=1, in_token_stride=FAR, out_token_stride=FAR))) == 0
    assert rules.rope_check(C.byref(rope(n_tokens=MAX, n_heads=1, in_head_stride=FAR, out_head_stride=FAR))) == 0
    assert rules.append_check(C.byref(append(n_new=1, k_token_stride=FAR))) == 0
    assert rules.seq_check(C.byref(seq(n_q=0, q_token_stride=FAR, out_token_stride=FAR))) == 0
    assert rules.paged_check(C.byref(paged(cache=cache(n_seqs=1), q_seq_stride=FAR, out_seq_stride=FAR))) == 0


def test_outputs_that_overlap_or_do_not_at_large_strides(rules):  # noqa: F811
    """Rows within heads: the next head begins behind the last row, to the element."""
    rows, token = 2 ** 20 + 1, 2 ** 30
    end = (rows - 1) * token + 32  # past a head's last row
    for head, ok in ((end, False), (2 ** 40, False)):  # 2^50: strides end at 2^40
        assert (rules.rope_check(C.byref(rope(n_tokens=rows, out_token_stride=token, out_head_stride=head))) == 0) == ok
    rows, token = 2 ** 9 + 1, 2 ** 30
    end = (rows - 1) * token + 32
    for head, ok in ((end, True), (end - 8, False)):
        assert (rules.rope_check(C.byref(rope(n_tokens=rows, out_token_stride=token, out_head_stride=head))) == 0) == ok
