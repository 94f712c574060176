"""Linear attention where rows of one call differ much in size or are not finite, and calls that take rarer paths, against memlib.py's
definitions and bounds."""
import numpy as np
import pytest

from memlib import linear
from seqlib import NAN, TYPES, Device, normal, to_bits, values
from test_gpu_memory import check_linear, check_paged4, linear_push, outside, run_linear

pytestmark = pytest.mark.gpu
GUARD = 3


@pytest.fixture
def dev(hip, device_arena):
    return Device(hip, device_arena)


def check_rows(engine, dev, dtype, q, k, v, lens, rates, state_in=None):
    """q, k, v [tokens][heads][hd] in 64 bits, sequences one behind the other; every output and state within its bound."""
    tokens, heads, hd = q.shape
    rows = np.full((tokens + 2 * GUARD, 3 * heads, hd), NAN[dtype], np.uint16)
    rows[GUARD:-GUARD] = to_bits(np.concatenate((q, k, v), 1), dtype)
    x = values(rows[GUARD:-GUARD], dtype)
    assert np.isfinite(x).all()
    rates = np.array(rates, np.float32)
    print(f"[linear] {dtype} {heads} x {hd} lengths {lens}", flush=True)
    got, new = run_linear(engine, dev, dtype, rows, heads, heads, lens, rates, None, state_in, len(lens), None, GUARD)
    at = 0
    for s, n in enumerate(lens):
        for h in range(heads):
            first = np.zeros((hd, hd)) if state_in is None else state_in[s, h].astype(np.float64)
            part = x[at:at + n]
            o, b, S, B = linear(part[:, h], part[:, heads + h], part[:, 2 * heads + h], float(rates[h]), first, hd ** -0.5, dtype)
            assert not outside(values(got[GUARD + at:GUARD + at + n, h], dtype), o, b), (s, h)
            assert not outside(new[s, h].astype(np.float64), S, B), (s, h)
        at += n


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("usual,large", [(1.0, 8000.0), (1.0, 40000.0), (0.1, 65000.0)])
@pytest.mark.parametrize("lens,query,key", [
    ([64], 63, 63), ([40], 39, 39), ([104], 103, 103), ([90, 70], 60, 89),  # the chunk's last; a query of the chunk before a short one
    ([64], 0, 0), ([100], 70, 20)])
def test_linear_one_large_token(engine, dev, dtype, hd, usual, large, lens, query, key):
    """One channel of one query and another of one key are large: tokens that do not see it keep their bits, as do those whose
    weights are small beside it. Values are small, so that outputs stay in fp16's range (65,000 sqrt(64) 4 / 64)."""
    rng = np.random.default_rng(hd)
    tokens, heads = sum(lens), 4
    q, k, v = (rng.standard_normal((tokens, heads, hd)) * usual for _ in "qkv")
    q[query, :, 3] = large
    k[key, :, 7] = -large
    check_rows(engine, dev, dtype, q, k, v / 64, lens, [0.0, 0.003, 0.05, 0.7])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("lens", [[64], [50], [200], [1500, 777]])
def test_linear_keys_of_zero_after_others(engine, dev, dtype, hd, lens):
    """Every sequence's last 32 tokens have keys of zero (padding, gates that are closed), and every third channel has a key in
    one token of 29 alone: states and outputs are sums of values that decayed far below the newest one's."""
    rng = np.random.default_rng(hd)
    tokens, heads = sum(lens), 4
    q, k, v = (rng.standard_normal((tokens, heads, hd)) for _ in "qkv")
    k[np.arange(tokens) % 29 != 0, :, 0::3] = 0
    for end in np.cumsum(lens):
        k[end - 32:end] = 0
    check_rows(engine, dev, dtype, q, k, v, lens, [0.0, 0.3, 0.7, 1.4])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
def test_linear_values_of_unlike_sizes(engine, dev, dtype, hd):
    """Tokens' values from 2^-14 to 2^14 under keys that share no channel with the next token's: a state's rows are of any size
    beside each other, and queries look at some of them alone."""
    rng = np.random.default_rng(hd)
    n, heads = 150, 2
    q, k = (rng.standard_normal((n, heads, hd)) for _ in "qk")
    v = rng.standard_normal((n, heads, hd)) * 2.0 ** (14.0 - 28.0 * (np.arange(n) % 2))[:, None, None] / 4
    k[0::2, :, 0::2] = 0
    k[1::2, :, 1::2] = 0
    q[0::3, :, 1::2] = 0
    q[1::3, :, 0::2] /= 256
    q /= 16
    check_rows(engine, dev, dtype, q, k, v, [n], [0.0, 0.2])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
def test_linear_states_of_unlike_sizes(engine, dev, dtype, hd):
    """A row of the carried state is 2^30 and no query looks at its channel: the others' bits stay."""
    rng = np.random.default_rng(hd)
    lens, heads = [70, 5, 600], 2
    q, k, v = (rng.standard_normal((sum(lens), heads, hd)) for _ in "qkv")
    s0 = (rng.standard_normal((len(lens), heads, hd, hd))).astype(np.float32)
    s0[:, :, hd // 2] = 2.0 ** 30
    q[:, :, hd // 2] = 0
    check_rows(engine, dev, dtype, q, k / 64, v / 64, lens, [0.0, 0.01], s0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("which", "qkv")
@pytest.mark.parametrize("other", [1.0, 0.0])
def test_linear_step_values_that_are_not_finite(engine, dev, dtype, hd, what, which, other):
    """They reach their row and head, channel and column, or head and row of the state, also where all that they meet is zero."""
    rng, n, heads, s, h, c = np.random.default_rng(hd), 3, 2, 1, 1, hd - 3
    rows = normal(rng, (n, 3 * heads, hd), dtype)
    s0 = rng.standard_normal((n, heads, hd, hd)).astype(np.float32) * np.float32(other)
    rows[s, h::heads] = to_bits(values(rows[s, h::heads], dtype) * other, dtype)
    push = linear_push(dtype, n, n, heads, heads, hd, n, 0.2, 3 * heads * hd)

    def run():
        x, out, new = dev.put(rows), dev.put(np.full((n, heads, hd), NAN[dtype], np.uint16)), dev.put(np.full(s0.shape, np.nan, np.float32))
        engine.linear_step(push, x, x + 2 * heads * hd, x + 4 * heads * hd, dev.put(np.array([0.0, 0.1], np.float32)), None, dev.put(s0),
                           out, new)
        return dev.get(out, (n, heads, hd)), dev.get(new, s0.shape, np.float32)

    clean, cs = run()
    rows[s, {"q": 0, "k": heads, "v": 2 * heads}[which] + h, c] = to_bits(np.array(what), dtype)
    got, gs = run()
    bad, bad_state = np.zeros(got.shape, bool), np.zeros(gs.shape, bool)
    bad[s, h, c if which == "v" else slice(None)] = True
    if which != "q":
        bad_state[s, h][(slice(None), c) if which == "v" else c] = True
    assert (~np.isfinite(values(got, dtype)) == bad).all() and (got[~bad] == clean[~bad]).all()
    assert (~np.isfinite(gs) == bad_state).all() and (gs[~bad_state] == cs[~bad_state]).all()


# ------------------------------------------------------------- rarer paths

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,kv,group", [(32, 2, 1), (32, 1, 2), (64, 1, 1), (128, 1, 4), (128, 2, 4)])
@pytest.mark.parametrize("lengths,max_len", [([1500, 40], 100), ([6000, 900], 2000)])
def test_paged4_longer_than_expected(engine, dev, dtype, hd, kv, group, lengths, max_len):
    """Sequences past max_len, four waves of a workgroup alone or in splits: all keys are seen."""
    check_paged4(engine, dev, np.random.default_rng(hd), dtype, hd, kv, group, 64, lengths, -1, 0, max_len)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("start", ["all", "none"])
def test_linear_long_without_a_state(engine, dev, dtype, hd, start):
    """Long sequences in segments, two of which have numbers of states out of range (-1 and as many as there are)."""
    lens = [900, 1500, 777, 300]
    assert engine.linear_attn_workspace(linear_push(dtype, len(lens), sum(lens) + 2 * GUARD, 2, 2, hd, 6, 1.0, 6 * hd)) > 0
    check_linear(engine, dev, np.random.default_rng(hd), dtype, hd, 2, 1, lens, start)
