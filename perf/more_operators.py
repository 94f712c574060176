"""What the operators for a cheaper past are measured on: queries and keys turned on their way into a paged
cache of 16 or 4 bits and the cache read back, one new token against a cache of 4 bits, and linear attention
with a decay for each head, over whole sequences and a token at a time.

listed() and draw() name the cases, prepare() makes a case's inputs on the GPU, run() is one pass:
in plain torch operations, or (own) through the library's entry points. exact() is the definition
in 64 bits. The lengths of a case follow from the case, everything else from the seed.

A value of the 4-bit cache is a sign and one of MAGNITUDES, times a power of two that a block of 32 channels of a
head shares (of 16 where a head has 16): channel 2i is the low half of byte i, the power 2^e is the byte e + 127.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
POWERS = {"fp16": (-23, 13), "bf16": (-125, 125)}  # those whose values all fit the type
CHUNK = 64  # tokens of a step of the plain linear attention
_engine = None


def listed():
    return [
        # one stream gets a token: queries and keys turned, keys and values kept in 16 bits; latency counts
        {"name": "write16 1 stream 8x32", "kind": "write", "dtype": "fp16", "bits": 16, "seqs": 1, "min_new": 1,
         "max_new": 1, "heads": 8, "kv_heads": 8, "head_dim": 32, "page": 16, "min_len": 37, "max_len": 37,
         "pairs_t": 4, "pairs_h": 6, "pairs_w": 6, "layout": "halves", "ladder": "axis", "far": 100_000},
        # a new frame: every place of the 68x120 grid is a stream and gets one token, kept in 4 bits
        {"name": "write4 8160 streams 8x32", "kind": "write", "dtype": "fp16", "bits": 4, "seqs": 8160, "min_new": 1,
         "max_new": 1, "heads": 8, "kv_heads": 8, "head_dim": 32, "page": 16, "min_len": 0, "max_len": 7,
         "pairs_t": 4, "pairs_h": 6, "pairs_w": 6, "layout": "halves", "ladder": "axis", "far": 1_000_000},
        # prompts of a few streams, ragged, wide heads, a part of each turned
        {"name": "write4 prompts 32/8x128", "kind": "write", "dtype": "bf16", "bits": 4, "seqs": 24, "min_new": 1,
         "max_new": 2051, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "min_len": 0, "max_len": 0,
         "pairs_t": 12, "pairs_h": 18, "pairs_w": 18, "layout": "adjacent", "ladder": "one", "far": 10_000},
        # one stream with a short history: the smallest step, latency counts
        {"name": "paged4 1 stream 8x32", "kind": "paged", "dtype": "fp16", "seqs": 1, "heads": 8, "kv_heads": 8,
         "head_dim": 32, "page": 16, "min_len": 91, "max_len": 91, "left": -1, "sinks": 0},
        # attention along time at every place of the grid: the last 48 frames and the first 4
        {"name": "paged4 8160 streams 8x32", "kind": "paged", "dtype": "fp16", "seqs": 8160, "heads": 8, "kv_heads": 8,
         "head_dim": 32, "page": 16, "min_len": 40, "max_len": 75, "left": 47, "sinks": 4},
        # a server's batch of streams of unlike length, shared key heads
        {"name": "paged4 24 streams 32/8x128", "kind": "paged", "dtype": "bf16", "seqs": 24, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 64, "min_len": 1000, "max_len": 20_001, "left": -1, "sinks": 0},
        # one long stream alone: the work has to be split over its length
        {"name": "paged4 1 long stream 32/8x128", "kind": "paged", "dtype": "fp16", "seqs": 1, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 32, "min_len": 131_075, "max_len": 131_075, "left": -1, "sinks": 0},
        # a handful of short ragged sequences of the small model
        {"name": "linear 9 short 8x16", "kind": "linear", "dtype": "fp16", "seqs": 9, "heads": 8, "kv_heads": 8,
         "head_dim": 16, "min_q": 1, "max_q": 130, "carried": False},
        # the 8160 tokens of a frame in scan order, on top of the frame before
        {"name": "linear 8160 tokens 8x32", "kind": "linear", "dtype": "fp16", "seqs": 1, "heads": 8, "kv_heads": 8,
         "head_dim": 32, "min_q": 8160, "max_q": 8160, "carried": True},
        # long ragged sequences, wide heads
        {"name": "linear 5 long 32x128", "kind": "linear", "dtype": "bf16", "seqs": 5, "heads": 32, "kv_heads": 32,
         "head_dim": 128, "min_q": 1025, "max_q": 8101, "carried": True},
        # a new token of a few streams
        {"name": "step 3 streams 8x64", "kind": "step", "dtype": "bf16", "seqs": 3, "heads": 8, "kv_heads": 4,
         "head_dim": 64},
        # a new frame: every place of the grid has its states
        {"name": "step 8160 streams 8x32", "kind": "step", "dtype": "fp16", "seqs": 8160, "heads": 8, "kv_heads": 8,
         "head_dim": 32},
    ]


def draw(rng):
    def log_int(a, b):
        return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))

    kind = rng.choice(("write", "paged", "linear", "step"))
    kv = rng.randint(1, 8)
    heads = kv * rng.choice((1, 1, 2, 3, 4, 5, 8))
    hd = rng.choice((16, 32, 64, 128))
    case = {"kind": kind, "dtype": rng.choice(("fp16", "bf16")), "heads": heads, "kv_heads": kv, "head_dim": hd}
    if kind == "write":
        turned = rng.randint(max(3, hd // 4), hd // 2)
        t = rng.randint(1, turned - 2)
        y = rng.randint(1, turned - t - 1)
        seqs = log_int(1, 8160)
        new = log_int(1, max(1, min(4099, 80_000_000 // (seqs * (heads + 2 * kv) * hd))))
        low = rng.randint(1, new)
        old = rng.choice((0, log_int(1, 1 + min(100, 40_000_000 // (seqs * kv * hd)))))
        return {**case, "bits": rng.choice((16, 4, 4)), "seqs": seqs, "min_new": low, "max_new": new,
                "page": rng.choice((16, 32, 64, 128)), "min_len": 0, "max_len": old, "pairs_t": t, "pairs_h": y,
                "pairs_w": turned - t - y, "layout": rng.choice(("halves", "adjacent")),
                "ladder": rng.choice(("axis", "one")), "far": log_int(1, 1_000_000)}
    if kind == "paged":
        left, sinks = rng.choice(((-1, 0), (log_int(1, 4000), 0), (log_int(1, 4000), log_int(1, 130))))
        seqs = log_int(1, 8160)
        most = log_int(1, max(1, min(131_075, 200_000_000 // (seqs * kv * hd))))
        return {**case, "seqs": seqs, "page": rng.choice((16, 32, 64, 128)), "min_len": rng.randint(1, most),
                "max_len": most, "left": left, "sinks": sinks}
    if kind == "linear":
        seqs = log_int(1, 64)
        most = log_int(1, max(1, min(8160, 60_000_000 // (seqs * heads * hd))))
        return {**case, "seqs": seqs, "min_q": rng.randint(1, most), "max_q": most, "carried": rng.random() < 0.5}
    return {**case, "seqs": log_int(1, max(1, min(8160, 60_000_000 // (heads * hd * hd))))}


# ------------------------------------------------------------------ lengths

def spread(n, low, high):
    """n lengths from low to high in mixed order; the first is the longest."""
    if n == 1:
        return [high]
    return [high - (i * 7919 % n) * (high - low) // (n - 1) for i in range(n)]


def starts_of(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def seen_keys(length, left, sinks):
    """Keys that the last of `length` tokens sees."""
    low = 0 if left < 0 else max(0, length - 1 - left)
    return length - low + min(low, sinks)


def block_of(hd):
    return min(hd, 32)


def turned_of(case):
    return case["pairs_t"] + case["pairs_h"] + case["pairs_w"]


# --------------------------------------------------------------- four bits

def quantise(x, dtype):
    """fp32 [..., hd] -> (codes [..., hd / 2], powers [..., blocks]), both uint8."""
    b = x.unflatten(-1, (-1, block_of(x.shape[-1])))
    top = b.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)  # top = m 2^e, m from 1/2 on: m <= 7/8 means top <= 7 * 2^(e - 3)
    low, high = POWERS[dtype]
    e = torch.where(top == 0, low, torch.where(m <= 0.875, e - 3, e - 2)).clamp(low, high)
    a = torch.ldexp(b.abs(), -e)
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
            + torch.signbit(b).to(torch.uint8) * 8)
    fine = torch.isfinite(top)
    code = torch.where(fine, code, 0).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, torch.where(fine, e + 127, 255).to(torch.uint8).squeeze(-1)


def dequantise(codes, powers):
    """-> fp32 [..., hd]."""
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)
    v = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1).flatten(-2)
    scale = torch.ldexp(torch.ones((), device=codes.device), powers.int() - 127)
    scale = torch.where(powers == 255, math.nan, scale)
    return (v.unflatten(-1, (powers.shape[-1], -1)) * scale[..., None]).flatten(-2)


# ------------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1_000_003 + 29)
    dt = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    s = {"case": case}
    H, K, hd, n = case["heads"], case["kv_heads"], case["head_dim"], case["seqs"]
    if case["kind"] in ("linear", "step"):
        lengths = spread(n, case["min_q"], case["max_q"]) if case["kind"] == "linear" else [1] * n
        cu = starts_of(lengths)
        rows = normal(cu[-1], H + 2 * K, hd)  # the fused rows of a projection
        s["q"], s["k"], s["v"] = rows[:, :H], rows[:, H:H + K], rows[:, H + K:]
        s["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
        # from a memory of two tokens to one of hundreds, another ladder for each seed
        s["rates"] = 2.0 ** (-8.0 * (torch.arange(H, device="cuda") + torch.rand(1, generator=g, device="cuda")) / H)
        s["state"] = None
        if case["kind"] == "step" or case["carried"]:
            s["state"] = torch.randn(n, H, hd, hd, generator=g, device="cuda") * 3
        s["out"] = torch.empty(cu[-1], H, hd, device="cuda", dtype=dt)
        s["state_out"] = torch.empty(n, H, hd, hd, device="cuda")
        return s
    # a paged cache whose pages lie in any order, with stale values where nothing was written yet
    page, old = case["page"], spread(n, case["min_len"], case["max_len"])
    new = spread(n, case["min_new"], case["max_new"]) if case["kind"] == "write" else [0] * n
    live = [a + b for a, b in zip(old, new)]
    need = [-(-a // page) for a in live]
    width, total = max(max(need), 1), sum(need)
    pool = total + 1 + total // 16
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    used = torch.arange(width, device="cuda")[None, :] < torch.tensor(need, device="cuda")[:, None]
    table[used] = torch.randperm(pool, generator=g, device="cuda")[:total].to(torch.int32)
    s["table"] = table
    bits = case.get("bits", 4)
    for name in ("k", "v"):
        if bits == 16:
            s[name + "_pages"], s[name + "_scales"] = normal(pool, K, page, hd), None
            continue
        s[name + "_pages"] = torch.empty(pool, K, page, hd // 2, dtype=torch.uint8, device="cuda")
        s[name + "_scales"] = torch.empty(pool, K, page, hd // block_of(hd), dtype=torch.uint8, device="cuda")
        some = max(1, 2 ** 25 // (K * page * hd))
        for at in range(0, pool, some):
            part = slice(at, min(pool, at + some))
            s[name + "_pages"][part], s[name + "_scales"][part] = quantise(
                normal(part.stop - at, K, page, hd).float(), case["dtype"])
    if case["kind"] == "paged":
        s["lengths"] = torch.tensor(old, dtype=torch.int32, device="cuda")
        s["q"] = normal(n, H, hd)
        s["out"] = torch.empty(n, H, hd, device="cuda", dtype=dt)
        return s

    def numbered(counts, first):
        """(sequence, position) of counts[i] tokens of each sequence i, from position first[i] on."""
        c = torch.tensor(counts, device="cuda")
        seq = torch.repeat_interleave(torch.arange(n, device="cuda"), c)
        at = torch.arange(sum(counts), device="cuda") - (torch.cumsum(c, 0) - c)[seq]
        return seq.to(torch.int32), (at + torch.tensor(first, device="cuda")[seq]).to(torch.int32)

    s["seq"], s["at"] = numbered(new, old)
    s["live_seq"], s["live_at"] = numbered(live, [0] * n)
    t = sum(new)
    rows = normal(t, H + 2 * K, hd)
    s["q"], s["k"], s["v"] = rows[:, :H], rows[:, H:H + K], rows[:, H + K:]
    first = torch.randint(0, case["far"] + 1, (1,), generator=g, device="cuda")
    s["pos"] = torch.stack((first + s["at"], s["seq"] // 120 % 68, s["seq"] % 120)).to(torch.int32).contiguous()
    s["q_out"] = torch.empty(t, H, hd, device="cuda", dtype=dt)
    s["live_k"] = torch.empty(sum(live), K, hd, device="cuda", dtype=dt)
    s["live_v"] = torch.empty(sum(live), K, hd, device="cuda", dtype=dt)
    return s


# -------------------------------------------------------------- plain forms

def ladder(case, dev):
    """(axis, frequency in 64 bits) of every turned pair of channels."""
    pairs = torch.tensor([case["pairs_t"], case["pairs_h"], case["pairs_w"]], device=dev)
    axis = torch.repeat_interleave(torch.arange(3, device=dev), pairs, output_size=turned_of(case))
    i = torch.arange(turned_of(case), device=dev)
    first = torch.cumsum(pairs, 0) - pairs
    e = i.double() / turned_of(case) if case["ladder"] == "one" else (i - first[axis]).double() / pairs[axis].double()
    return axis, torch.pow(torch.tensor(10000.0, dtype=torch.float64, device=dev), -e)


def turn(x, pos, case):
    """In 64 bits: which of two 4-bit values a key goes to hangs on it. fp32 result."""
    n, x = turned_of(case), x.double()
    axis, f = ladder(case, x.device)
    angle = pos.double()[axis].t() * f
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    if case["layout"] == "halves":
        a, b = x[..., :n], x[..., n:2 * n]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * n:]), -1)
    else:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        y = torch.cat((torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2), x[..., 2 * n:]), -1)
    return y.float()


def plain_write(s, case):
    dt = TYPES[case["dtype"]]
    pos, size = s["at"].long(), case["page"]
    page = s["table"][s["seq"].long(), pos // size].long()
    live = s["live_at"].long()
    live_page = s["table"][s["live_seq"].long(), live // size].long()
    outs = [turn(s["q"], s["pos"], case).to(dt)]
    for name in ("k", "v"):
        x = turn(s["k"], s["pos"], case) if name == "k" else s["v"].float()
        pages, scales = s[name + "_pages"], s[name + "_scales"]
        if scales is None:
            pages[page, :, pos % size] = x.to(dt)
            outs.append(pages[live_page, :, live % size])
            continue
        pages[page, :, pos % size], scales[page, :, pos % size] = quantise(x, case["dtype"])
        outs.append(dequantise(pages[live_page, :, live % size], scales[live_page, :, live % size]).to(dt))
    return tuple(outs)


def plain_paged(s, case):
    """Gathers the positions that a stream's new token sees: its window, and the sinks before it."""
    left, most = case["left"], case["max_len"]
    left = most - 1 if left < 0 else min(left, most - 1)
    sinks = min(case["sinks"], most)
    last = s["lengths"].long()[:, None] - 1
    near = last - torch.arange(left + 1, device=last.device)
    first = torch.arange(sinks, device=last.device).expand(last.shape[0], -1)
    pos = torch.cat((near, first), 1)
    seen = torch.cat((near >= 0, (first < last - left) & (first <= last)), 1)
    pos = torch.where(seen, pos, 0)
    page, slot = torch.where(seen, torch.gather(s["table"].long(), 1, pos // case["page"]), 0), pos % case["page"]
    k = dequantise(s["k_pages"][page, :, slot], s["k_scales"][page, :, slot]).permute(0, 2, 3, 1)
    v = dequantise(s["v_pages"][page, :, slot], s["v_scales"][page, :, slot]).permute(0, 2, 1, 3)
    n, H, hd = s["q"].shape
    q = s["q"].float().view(n, case["kv_heads"], -1, hd)
    score = torch.matmul(q, k).mul_(1.0 / math.sqrt(hd))
    score = score.masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    return (torch.matmul(p, v) / p.sum(-1, keepdim=True)).view(n, H, hd).to(s["q"].dtype)


def plain_linear(s, case):
    """The sequences side by side, padded to the longest, CHUNK tokens at a time."""
    H, K, hd, n = case["heads"], case["kv_heads"], case["head_dim"], case["seqs"]
    cu = s["cu"].long()
    lens = cu[1:] - cu[:-1]
    most = -(-case["max_q"] // CHUNK) * CHUNK
    at = torch.arange(most, device=cu.device)
    real = at < lens[:, None]
    rows = torch.where(real, cu[:-1, None] + at, 0)

    def heads_first(x):
        x = torch.where(real[..., None, None], x[rows].float(), 0.0)
        return torch.repeat_interleave(x, H // x.shape[2], 2).permute(0, 2, 1, 3)

    q, k, v = heads_first(s["q"]), heads_first(s["k"]), heads_first(s["v"])
    state = torch.zeros(n, H, hd, hd, device=cu.device) if s["state"] is None else s["state"].clone()
    out = torch.empty(n, H, most, hd, device=cu.device)
    r, i = s["rates"][:, None, None], torch.arange(CHUNK, device=cu.device)
    gap = i[:, None] - i
    within = torch.where(gap >= 0, torch.exp(-r * gap.clamp(min=0)), 0.0)
    for c in range(0, most, CHUNK):
        qc, kc, vc = q[:, :, c:c + CHUNK], k[:, :, c:c + CHUNK], v[:, :, c:c + CHUNK]
        before = torch.matmul(qc, state) * torch.exp(-r * (i[:, None] + 1))
        out[:, :, c:c + CHUNK] = before + torch.matmul(torch.matmul(qc, kc.transpose(2, 3)) * within, vc)
        count = (lens - c).clamp(0, CHUNK)[:, None, None, None]  # of a sequence's tokens in this chunk
        fade = torch.exp(-r * (count - 1 - i[:, None]).clamp(min=0))
        state = state * torch.exp(-r * count) + torch.matmul(kc.transpose(2, 3), vc * fade)
    t = torch.arange(s["q"].shape[0], device=cu.device)
    of = torch.searchsorted(cu[1:], t, right=True)
    return (out.transpose(1, 2)[of, t - cu[of]] / math.sqrt(hd)).to(s["q"].dtype), state


def plain_step(s, case):
    H, hd = case["heads"], case["head_dim"]
    q = s["q"].float()
    k, v = (torch.repeat_interleave(s[x].float(), H // case["kv_heads"], 1) for x in ("k", "v"))
    state = s["state"] * torch.exp(-s["rates"])[:, None, None] + k[..., None] * v[..., None, :]
    o = torch.matmul(q[..., None, :], state).squeeze(-2) / math.sqrt(hd)
    return o.to(s["q"].dtype), state


def run(s):
    case = s["case"]
    if own:
        return library(s, case)
    plain = {"write": plain_write, "paged": plain_paged, "linear": plain_linear, "step": plain_step}
    return plain[case["kind"]](s, case)


# --------------------------------------------------------------- the library

def engine():
    """The program's context: one for all calls."""
    global _engine
    if _engine is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "prism-inference_amd"))
        import prism_amd

        _engine = (prism_amd, prism_amd.Engine(torch.cuda.current_device()))
    return _engine


def address(x):
    return None if x is None else x.data_ptr()


def calls(s, case, prism, eng):
    """The parameters of a case's calls, which a program fills in once."""
    dt = prism.BF16 if case["dtype"] == "bf16" else prism.F16
    H, K, hd, n = case["heads"], case["kv_heads"], case["head_dim"], case["seqs"]
    q, kind = s["q"], case["kind"]
    if kind in ("linear", "step"):
        push = prism.LinearAttnPush(
            dtype=dt, n_seqs=n, n_tokens=q.shape[0], n_heads=H, n_kv_heads=K, head_dim=hd, n_states=n,
            scale=1.0 / math.sqrt(hd), q_token_stride=q.stride(0), q_head_stride=q.stride(1),
            k_token_stride=s["k"].stride(0), k_head_stride=s["k"].stride(1), v_token_stride=s["v"].stride(0),
            v_head_stride=s["v"].stride(1), out_token_stride=s["out"].stride(0), out_head_stride=s["out"].stride(1))
        if kind == "linear":
            s["ws"] = torch.empty(max(1, eng.linear_attn_workspace(push)), dtype=torch.uint8, device="cuda")
        return push
    cache = prism.CacheDesc(dtype=dt, n_kv_heads=K, head_dim=hd, page_size=case["page"],
                            n_pages=s["k_pages"].shape[0], n_seqs=n, table_pages=s["table"].shape[1])
    pages = prism.CachePages(k=address(s["k_pages"]), v=address(s["v_pages"]), k_scales=address(s["k_scales"]),
                             v_scales=address(s["v_scales"]))
    if kind == "paged":
        push = prism.PagedAttnPush(
            cache=cache, n_heads=H, left=case["left"], sinks=case["sinks"], max_len=case["max_len"],
            scale=1.0 / math.sqrt(hd), q_seq_stride=q.stride(0), q_head_stride=q.stride(1),
            out_seq_stride=s["out"].stride(0), out_head_stride=s["out"].stride(1))
        s["ws"] = torch.empty(max(1, eng.paged_attn4_workspace(push)), dtype=torch.uint8, device="cuda")
        return push, pages
    bits = prism.CACHE_4 if case["bits"] == 4 else prism.CACHE_16
    write = prism.RopeAppendPush(
        cache=cache, format=bits, n_new=q.shape[0], n_heads=H, n_axes=3,
        pairs=(case["pairs_t"], case["pairs_h"], case["pairs_w"], 0),
        layout=prism.ROPE_HALVES if case["layout"] == "halves" else prism.ROPE_ADJACENT,
        ladder=prism.ROPE_ONE_LADDER if case["ladder"] == "one" else prism.ROPE_AXIS_LADDER, base=10000.0,
        q_token_stride=q.stride(0), q_head_stride=q.stride(1), k_token_stride=s["k"].stride(0),
        k_head_stride=s["k"].stride(1), v_token_stride=s["v"].stride(0), v_head_stride=s["v"].stride(1),
        out_token_stride=s["q_out"].stride(0), out_head_stride=s["q_out"].stride(1), pos_stride=s["pos"].stride(0))
    read = prism.CacheReadPush(
        cache=cache, format=bits, n_rows=s["live_k"].shape[0], k_token_stride=s["live_k"].stride(0),
        k_head_stride=s["live_k"].stride(1), v_token_stride=s["live_v"].stride(0), v_head_stride=s["live_v"].stride(1))
    return write, read, pages


def library(s, case):
    prism, eng = engine()
    stream = torch.cuda.current_stream().cuda_stream
    if "call" not in s:
        s["call"] = calls(s, case, prism, eng)
    call, kind = s["call"], case["kind"]
    if kind == "write":
        write, read, pages = call
        eng.rope_append(write, s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["pos"].data_ptr(),
                        s["q_out"].data_ptr(), s["seq"].data_ptr(), s["at"].data_ptr(), s["table"].data_ptr(), pages,
                        stream)
        eng.cache_read(read, pages, s["live_seq"].data_ptr(), s["live_at"].data_ptr(), s["table"].data_ptr(),
                       s["live_k"].data_ptr(), s["live_v"].data_ptr(), stream)
        return s["q_out"], s["live_k"], s["live_v"]
    if kind == "paged":
        push, pages = call
        eng.paged_attn4(push, s["q"].data_ptr(), pages, s["table"].data_ptr(), s["lengths"].data_ptr(),
                        s["out"].data_ptr(), s["ws"].data_ptr(), s["ws"].numel(), stream)
        return s["out"]
    if kind == "linear":
        eng.linear_attn(call, s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["rates"].data_ptr(),
                        s["cu"].data_ptr(), None, address(s["state"]), s["out"].data_ptr(), s["state_out"].data_ptr(),
                        s["ws"].data_ptr(), s["ws"].numel(), stream)
    else:
        eng.linear_step(call, s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["rates"].data_ptr(), None,
                        s["state"].data_ptr(), s["out"].data_ptr(), s["state_out"].data_ptr(), stream)
    return s["out"], s["state_out"]


# ---------------------------------------------------------------- work, exact

def work(case):
    H, K, hd, n = case["heads"], case["kv_heads"], case["head_dim"], case["seqs"]
    held = 4 * K * hd  # bytes of a token's keys and values
    if case.get("bits", 4) == 4:
        held = K * hd + 2 * K * hd // block_of(hd)
    if case["kind"] == "write":
        new = sum(spread(n, case["min_new"], case["max_new"]))
        live = new + sum(spread(n, case["min_len"], case["max_len"]))
        return {"bytes": new * (4 * H * hd + 4 * K * hd + held + 20) + live * (held + 4 * K * hd + 8),
                "flops": 6 * new * (H + K) * turned_of(case)}
    if case["kind"] == "paged":
        seen = sum(seen_keys(x, case["left"], case["sinks"]) for x in spread(n, case["min_len"], case["max_len"]))
        return {"bytes": seen * held + 4 * n * H * hd + 4 * seen // case["page"], "flops": 4 * seen * H * hd}
    tokens = sum(spread(n, case["min_q"], case["max_q"])) if case["kind"] == "linear" else n
    states = 2 if case["kind"] == "step" or case["carried"] else 1
    return {"bytes": 4 * tokens * (H + K) * hd + 4 * states * n * H * hd * hd, "flops": 4 * tokens * H * hd * hd}


def exact_values(codes, powers, hd):
    """Stored bytes [..., hd / 2] and [..., blocks] -> 64 bits, by the formula of a float with two exponent bits and one
    fraction bit."""
    c = torch.empty(*codes.shape[:-1], hd, dtype=torch.int64, device=codes.device)
    c[..., 0::2], c[..., 1::2] = codes.long() % 16, codes.long() // 16
    power, fraction = c % 8 // 2, c % 2
    size = torch.where(power == 0, fraction * 0.5, (1 + fraction * 0.5) * 2.0 ** (power - 1).double())
    b = powers.long().repeat_interleave(block_of(hd), -1)
    return torch.where(b == 255, math.nan, torch.where(c >= 8, -size, size) * 2.0 ** (b - 127).double())


def exact_rounded(x, dtype):
    """fp32 values as the 4-bit cache gives them back, in 64 bits: the nearest of the magnitudes by distance."""
    x = x.double().unflatten(-1, (-1, block_of(x.shape[-1])))
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / 7.0)).nan_to_num(neginf=-1000.0)
    e = torch.where(top > 7.0 * 2.0 ** e, e + 1, torch.where(top <= 7.0 * 2.0 ** (e - 1), e - 1, e))  # log2's rounding
    e = e.clamp(*POWERS[dtype])
    a, best = x.abs() / 2.0 ** e, torch.zeros_like(x)
    for i, m in enumerate(MAGNITUDES):
        nearer = (a - m).abs() < (a - best).abs()
        tie = ((a - m).abs() == (a - best).abs()) & (i % 2 == 0)
        best = torch.where(nearer | tie, m, best)
    return (torch.sign(x) * best * 2.0 ** e).flatten(-2)


def exact_turn(x, pos, case):
    y, x = x.double().clone(), x.double()
    n, i = turned_of(case), 0
    for axis, count in enumerate((case["pairs_t"], case["pairs_h"], case["pairs_w"])):
        for j in range(count):
            f = 10000.0 ** -(i / n if case["ladder"] == "one" else j / count)
            a, b = (i, i + n) if case["layout"] == "halves" else (2 * i, 2 * i + 1)
            phi = (pos[axis].double() * f)[:, None]
            y[..., a] = x[..., a] * torch.cos(phi) - x[..., b] * torch.sin(phi)
            y[..., b] = x[..., b] * torch.cos(phi) + x[..., a] * torch.sin(phi)
            i += 1
    return y


def exact_write(s, case):
    hd, size = case["head_dim"], case["page"]
    q, k = exact_turn(s["q"], s["pos"], case), exact_turn(s["k"], s["pos"], case)
    outs = [q]
    page = s["table"].long()[s["live_seq"].long(), s["live_at"].long() // size]
    slot = s["live_at"].long() % size
    # a stream's new tokens are its last, in the order of the rows
    new = torch.bincount(s["seq"].long(), minlength=case["seqs"])
    live = torch.bincount(s["live_seq"].long(), minlength=case["seqs"])
    fresh = s["live_at"].long() >= (live - new)[s["live_seq"].long()]
    for name, x in (("k", k), ("v", s["v"].double())):
        if case["bits"] == 16:
            y = s[name + "_pages"][page, :, slot].double()
            y[fresh] = x.to(TYPES[case["dtype"]]).double() if name == "v" else x
        else:
            y = exact_values(s[name + "_pages"][page, :, slot], s[name + "_scales"][page, :, slot], hd)
            y[fresh] = exact_rounded(x.float(), case["dtype"])
        outs.append(y)
    return tuple(outs)


def exact_paged(s, case):
    H, K, hd, size = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    out = torch.zeros(case["seqs"], H, hd, dtype=torch.float64, device="cuda")
    for i, length in enumerate(spread(case["seqs"], case["min_len"], case["max_len"])):
        low = 0 if case["left"] < 0 else max(0, length - 1 - case["left"])
        pos = torch.cat((torch.arange(min(low, case["sinks"]), device="cuda"), torch.arange(low, length, device="cuda")))
        page, slot = s["table"][i].long()[pos // size], pos % size
        k = exact_values(s["k_pages"][page, :, slot], s["k_scales"][page, :, slot], hd).permute(1, 2, 0).contiguous()
        v = exact_values(s["v_pages"][page, :, slot], s["v_scales"][page, :, slot], hd).permute(1, 0, 2).contiguous()
        z = torch.matmul(s["q"][i].double().view(K, H // K, hd), k) / math.sqrt(hd)
        out[i] = torch.matmul(torch.softmax(z, -1), v).view(H, hd)
    return out


def exact_linear(s, case):
    """Every token against every one before it, no state in between."""
    H, K, hd = case["heads"], case["kv_heads"], case["head_dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    state = torch.zeros(case["seqs"], H, hd, hd, dtype=torch.float64, device="cuda")
    at = 0
    for i, n in enumerate(spread(case["seqs"], case["min_q"], case["max_q"]) if case["kind"] == "linear"
                          else [1] * case["seqs"]):
        t = torch.arange(n, device="cuda", dtype=torch.float64)
        for h in range(H):
            r = s["rates"][h].double()
            q, k, v = s["q"][at:at + n, h].double(), *(s[x][at:at + n, h * K // H].double() for x in ("k", "v"))
            start = state[i, h] if s["state"] is None else s["state"][i, h].double()
            for b in range(0, n, 2048):
                e = min(n, b + 2048)
                gap = t[b:e, None] - t[:e]
                w = torch.where(gap >= 0, torch.exp(-r * gap), 0.0) * (q[b:e] @ k[:e].T)
                out[at + b:at + e, h] = w @ v[:e] + torch.exp(-r * (t[b:e, None] + 1)) * (q[b:e] @ start)
            state[i, h] = torch.exp(-r * n) * start + (k * torch.exp(-r * (n - 1 - t))[:, None]).T @ v
        at += n
    return out / math.sqrt(hd), state


def exact_step(s, case):
    group, hd = case["heads"] // case["kv_heads"], case["head_dim"]
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    state = torch.empty(s["state"].shape, dtype=torch.float64, device=q.device)
    for h in range(case["heads"]):
        keep = torch.exp(-s["rates"][h].double())
        state[:, h] = s["state"][:, h].double() * keep + k[:, h // group, :, None] * v[:, h // group, None, :]
        out[:, h] = (q[:, h, :, None] * state[:, h]).sum(1) / math.sqrt(hd)
    return out, state


def exact(case, seed):
    s = prepare(case, seed)
    return {"write": exact_write, "paged": exact_paged, "linear": exact_linear, "step": exact_step}[case["kind"]](s, case)
