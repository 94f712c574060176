"""What the sequence operators are measured on: rotary positions with several axes, writing to the
paged cache, one new token against it, and attention over whole sequences with a window and sinks.

listed() and draw() name the cases, prepare() makes a case's inputs on the GPU, run() is one pass:
in plain torch operations, or (own) through the library's entry points. exact() is the definition
in 64 bits. The lengths of a case follow from the case, everything else from the seed.
"""
import math
import os
import sys

import torch

own = False

MAX_SCORES = 2_400_000_000  # query x key pairs of the plain form, all heads and padded sequences
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_engine = None


def listed():
    return [
        # one frame of the small model between its QKV product and attention: queries and keys turned,
        # read out of the fused rows; latency counts
        {"name": "rope frame 68x120 8x16", "kind": "rope", "dtype": "fp16", "tokens": 8160, "heads": 16, "extra": 8,
         "head_dim": 16, "pairs_t": 2, "pairs_h": 3, "pairs_w": 3, "h": 68, "w": 120, "layout": "halves",
         "ladder": "axis", "inverse": False, "far": 100_000},
        # a clip of 16 frames of the wide models
        {"name": "rope 16 frames 8x32", "kind": "rope", "dtype": "fp16", "tokens": 130_560, "heads": 16, "extra": 8,
         "head_dim": 32, "pairs_t": 4, "pairs_h": 6, "pairs_w": 6, "h": 68, "w": 120, "layout": "adjacent",
         "ladder": "axis", "inverse": False, "far": 1_000_000},
        # the gradient's way back (the inverse turn) at native 1080p, wide heads, part of each head unturned
        {"name": "rope inverse 135x240 40x128", "kind": "rope", "dtype": "bf16", "tokens": 32_401, "heads": 40,
         "extra": 0, "head_dim": 128, "pairs_t": 12, "pairs_h": 18, "pairs_w": 18, "h": 135, "w": 240,
         "layout": "halves", "ladder": "one", "inverse": True, "far": 10_000},
        # a new frame: every place of the 68x120 grid is a stream of its own and gets one token
        {"name": "append 8160 streams 8x32", "kind": "append", "dtype": "fp16", "seqs": 8160, "min_new": 1,
         "max_new": 1, "kv_heads": 8, "head_dim": 32, "page": 16, "min_len": 0, "max_len": 63},
        # prompts of a few streams, ragged, written in one call
        {"name": "append prompts 8x128", "kind": "append", "dtype": "bf16", "seqs": 24, "min_new": 1,
         "max_new": 4099, "kv_heads": 8, "head_dim": 128, "page": 64, "min_len": 0, "max_len": 1500},
        # one stream with a short history: the smallest step, latency counts
        {"name": "paged 1 stream 8x32", "kind": "paged", "dtype": "fp16", "seqs": 1, "heads": 8, "kv_heads": 8,
         "head_dim": 32, "page": 16, "min_len": 91, "max_len": 91, "left": -1, "sinks": 0},
        # attention along time at every place of the grid: the last 48 frames and the first 4
        {"name": "paged 8160 streams 8x32", "kind": "paged", "dtype": "fp16", "seqs": 8160, "heads": 8, "kv_heads": 8,
         "head_dim": 32, "page": 16, "min_len": 40, "max_len": 75, "left": 47, "sinks": 4},
        # a server's batch of streams of unlike length, shared key heads
        {"name": "paged 24 streams 32/8x128", "kind": "paged", "dtype": "bf16", "seqs": 24, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 64, "min_len": 1000, "max_len": 20_001, "left": -1, "sinks": 0},
        # one long stream alone: the work has to be split over its length
        {"name": "paged 1 long stream 32/8x128", "kind": "paged", "dtype": "fp16", "seqs": 1, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 32, "min_len": 131_075, "max_len": 131_075, "left": -1, "sinks": 0},
        # a handful of short ragged sequences of the small model
        {"name": "seq 9 short 8x16", "kind": "seq", "dtype": "fp16", "seqs": 9, "heads": 8, "kv_heads": 8,
         "head_dim": 16, "min_q": 1, "max_q": 130, "past": 0, "left": 63, "right": 0, "sinks": 4, "fused": True},
        # the 8160 tokens of a frame in scan order: the 1024 before each, and the first row of the frame
        {"name": "seq 8160 tokens 8x32", "kind": "seq", "dtype": "fp16", "seqs": 1, "heads": 8, "kv_heads": 8,
         "head_dim": 32, "min_q": 8160, "max_q": 8160, "past": 0, "left": 1023, "right": 0, "sinks": 120,
         "fused": True},
        # long ragged sequences with shared key heads, some keys from before
        {"name": "seq 2 long 32/8x128", "kind": "seq", "dtype": "bf16", "seqs": 2, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "min_q": 4501, "max_q": 5800, "past": 123, "left": 2047, "right": 0, "sinks": 4,
         "fused": False},
    ]


def draw(rng):
    def log_int(a, b):
        return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))

    kind = rng.choice(("rope", "append", "paged", "seq"))
    case = {"kind": kind, "dtype": rng.choice(("fp16", "bf16"))}
    if kind == "rope":
        hd = rng.choice((16, 32, 64, 128))
        turned = rng.randint(max(3, hd // 4), hd // 2)
        t = rng.randint(1, turned - 2)
        y = rng.randint(1, turned - t - 1)
        heads = rng.randint(1, 48)
        return {**case, "tokens": log_int(1, max(2, 160_000_000 // (heads * hd))), "heads": heads,
                "extra": rng.choice((0, heads)), "head_dim": hd, "pairs_t": t, "pairs_h": y,
                "pairs_w": turned - t - y, "h": rng.randint(1, 135), "w": rng.randint(1, 240),
                "layout": rng.choice(("halves", "adjacent")), "ladder": rng.choice(("axis", "one")),
                "inverse": rng.random() < 0.5, "far": log_int(1, 1_000_000)}
    if kind == "append":
        hd, kv = rng.choice((16, 32, 64, 128)), rng.randint(1, 12)
        seqs = log_int(1, 8160)
        new = log_int(1, max(1, min(4099, 40_000_000 // (seqs * kv * hd))))
        return {**case, "seqs": seqs, "min_new": rng.randint(1, new), "max_new": new, "kv_heads": kv, "head_dim": hd,
                "page": rng.choice((16, 32, 64, 128)), "min_len": 0, "max_len": log_int(1, 200)}
    kv = rng.randint(1, 8)
    heads = kv * rng.choice((1, 1, 2, 3, 4, 5, 8))
    hd = rng.choice((16, 32, 64, 128))
    left, sinks = rng.choice(((-1, 0), (log_int(1, 4000), 0), (log_int(1, 4000), log_int(1, 130))))
    if kind == "paged":
        seqs = log_int(1, 8160)
        most = log_int(1, max(1, min(131_075, 240_000_000 // (seqs * kv * hd))))
        return {**case, "seqs": seqs, "heads": heads, "kv_heads": kv, "head_dim": hd,
                "page": rng.choice((16, 32, 64, 128)), "min_len": rng.randint(1, most), "max_len": most, "left": left,
                "sinks": sinks}
    seqs = log_int(1, 64)
    past = rng.choice((0, 0, log_int(1, 1000)))
    side = int(math.sqrt(MAX_SCORES / (seqs * heads))) - past
    most = log_int(1, max(1, min(8160, side)))
    return {**case, "seqs": seqs, "heads": heads, "kv_heads": kv, "head_dim": hd, "min_q": rng.randint(1, most),
            "max_q": most, "past": past, "left": left, "right": rng.choice((0, 0, 0, rng.randint(1, 300))),
            "sinks": sinks, "fused": rng.random() < 0.5 and not past}


# ------------------------------------------------------------------ lengths

def spread(n, low, high):
    """n lengths from low to high in mixed order; the first is the longest."""
    if n == 1:
        return [high]
    return [high - (i * 7919 % n) * (high - low) // (n - 1) for i in range(n)]


def lengths_of(case):
    return spread(case["seqs"], case["min_len"], case["max_len"])


def starts_of(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def visible_pairs(q, past, left, right, sinks):
    """Visible (query, key) pairs of a sequence of q queries behind `past` keys."""
    k, n = q + past, 0
    for p in range(past, k):
        top = min(k, p + right + 1)
        low = 0 if left < 0 else max(0, p - left)
        n += top - low + min(low, sinks)
    return n


# ------------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1_000_003 + 17)
    dt = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    s = {"case": case}
    hd = case["head_dim"]
    if case["kind"] == "rope":
        t, heads, row = case["tokens"], case["heads"], case["heads"] + case["extra"]
        s["x"] = normal(t, row, hd)[:, :heads]  # the queries and keys of fused rows
        s["out"] = torch.empty(t, heads, hd, device="cuda", dtype=dt)
        i = torch.arange(t, device="cuda")
        first = torch.randint(0, case["far"] + 1, (1,), generator=g, device="cuda")
        w, h = case["w"], case["h"]
        s["pos"] = torch.stack((first + i // (h * w), i // w % h, i % w)).to(torch.int32).contiguous()
        return s
    if case["kind"] == "seq":
        ql = spread(case["seqs"], case["min_q"], case["max_q"])
        cq, ck = starts_of(ql), starts_of([n + case["past"] for n in ql])
        H, K = case["heads"], case["kv_heads"]
        if case["fused"]:
            rows = normal(cq[-1], H + 2 * K, hd)
            s["q"], s["k"], s["v"] = rows[:, :H], rows[:, H:H + K], rows[:, H + K:]
        else:
            s["q"], s["k"], s["v"] = normal(cq[-1], H, hd), normal(ck[-1], K, hd), normal(ck[-1], K, hd)
        s["cu_q"] = torch.tensor(cq, dtype=torch.int32, device="cuda")
        s["cu_k"] = torch.tensor(ck, dtype=torch.int32, device="cuda")
        s["out"] = torch.empty(cq[-1], H, hd, device="cuda", dtype=dt)
        return s
    # a paged cache whose pages lie in any order, with stale values where nothing was written yet
    page, n, K = case["page"], case["seqs"], case["kv_heads"]
    old = lengths_of(case)
    new = spread(n, case["min_new"], case["max_new"]) if case["kind"] == "append" else [0] * n
    need = [-(-(a + b) // page) for a, b in zip(old, new)]
    width, total = max(max(need), 1), sum(need)
    pool = total + 1 + total // 16
    order = torch.randperm(pool, generator=g, device="cuda")[:total].to(torch.int32)
    count = torch.tensor(need, device="cuda")
    live = torch.arange(width, device="cuda")[None, :] < count[:, None]
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    table[live] = order
    s["table"] = table
    s["k_pages"], s["v_pages"] = normal(pool, K, page, hd), normal(pool, K, page, hd)
    if case["kind"] == "append":
        grown = torch.tensor(new, device="cuda")
        s["seq"] = torch.repeat_interleave(torch.arange(n, device="cuda"), grown).to(torch.int32)
        at = torch.arange(sum(new), device="cuda") - torch.repeat_interleave(torch.cumsum(grown, 0) - grown, grown)
        s["pos"] = (at + torch.tensor(old, device="cuda")[s["seq"].long()]).to(torch.int32)
        rows = normal(sum(new), 2 * K, hd)
        s["k"], s["v"] = rows[:, :K], rows[:, K:]
        return s
    s["lengths"] = torch.tensor(old, dtype=torch.int32, device="cuda")
    s["q"] = normal(n, case["heads"], hd)
    s["out"] = torch.empty(n, case["heads"], hd, device="cuda", dtype=dt)
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


def turned_of(case):
    return case["pairs_t"] + case["pairs_h"] + case["pairs_w"]


def plain_rope(s, case):
    n, x = turned_of(case), s["x"].float()
    axis, f = ladder(case, x.device)
    angle = s["pos"].double()[axis].t() * f
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    sin = -sin if case["inverse"] else sin
    if case["layout"] == "halves":
        a, b = x[..., :n], x[..., n:2 * n]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * n:]), -1)
    else:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        y = torch.cat((torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2), x[..., 2 * n:]), -1)
    return y.to(s["x"].dtype)


def plain_append(s, case):
    pos = s["pos"].long()
    page = s["table"][s["seq"].long(), pos // case["page"]].long()
    s["k_pages"][page, :, pos % case["page"]] = s["k"]
    s["v_pages"][page, :, pos % case["page"]] = s["v"]
    return s["k_pages"], s["v_pages"]


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
    page = torch.where(seen, torch.gather(s["table"].long(), 1, pos // case["page"]), 0)
    k = s["k_pages"][page, :, pos % case["page"]].float().permute(0, 2, 3, 1)  # [stream][head][channel][key]
    v = s["v_pages"][page, :, pos % case["page"]].float().permute(0, 2, 1, 3)
    n, H, hd = s["q"].shape
    q = s["q"].float().view(n, case["kv_heads"], -1, hd)
    score = torch.matmul(q, k).mul_(1.0 / math.sqrt(hd))
    score = score.masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    return (torch.matmul(p, v) / p.sum(-1, keepdim=True)).view(n, H, hd).to(s["q"].dtype)


def plain_seq(s, case):
    """The sequences side by side, padded to the longest."""
    H, K, hd = case["heads"], case["kv_heads"], case["head_dim"]
    mq, mk = case["max_q"], case["max_q"] + case["past"]
    cq, ck = s["cu_q"].long(), s["cu_k"].long()
    ql, kl = (cq[1:] - cq[:-1])[:, None], (ck[1:] - ck[:-1])[:, None]
    i, j = torch.arange(mq, device=cq.device), torch.arange(mk, device=cq.device)
    qi = torch.where(i < ql, cq[:-1, None] + i, 0)
    kj = torch.where(j < kl, ck[:-1, None] + j, 0)
    q = s["q"][qi].float().unflatten(2, (K, -1)).permute(0, 2, 3, 1, 4).reshape(len(qi), K, -1, hd)
    k, v = s["k"][kj].float().permute(0, 2, 3, 1), s["v"][kj].float().permute(0, 2, 1, 3)
    p, at = (kl - ql + i)[:, :, None], j[None, None]
    near = at >= p - case["left"] if case["left"] >= 0 else at >= 0
    seen = (at <= p + case["right"]) & (near | (at < case["sinks"])) & (j < kl)[:, None]
    score = torch.matmul(q, k).mul_(1.0 / math.sqrt(hd)).view(len(qi), K, -1, mq, mk)
    score.masked_fill_(~seen[:, None, None], -math.inf)
    score.sub_(score.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = score.sum(-1, keepdim=True).clamp_(min=1e-30)
    o = torch.matmul(score.view(len(qi), K, -1, mk), v).view(len(qi), K, -1, mq, hd) / total
    rows = torch.arange(s["q"].shape[0], device=cq.device)
    of = torch.searchsorted(cq[1:], rows, right=True)
    return o.flatten(1, 2).transpose(1, 2)[of, rows - cq[of]].to(s["q"].dtype)


def run(s):
    case = s["case"]
    if own:
        return library(s, case)
    plain = {"rope": plain_rope, "append": plain_append, "paged": plain_paged, "seq": plain_seq}
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


def library(s, case):
    prism, eng = engine()
    stream = torch.cuda.current_stream().cuda_stream
    call = s.get("call")  # the parameters of the call, which a program fills in once
    dt = prism.BF16 if case["dtype"] == "bf16" else prism.F16
    hd, kind = case["head_dim"], case["kind"]
    if kind == "rope":
        if call is None:
            call = s["call"] = prism.RopePush(
                dtype=dt, n_tokens=case["tokens"], n_heads=case["heads"], head_dim=hd, n_axes=3,
                pairs=(case["pairs_t"], case["pairs_h"], case["pairs_w"], 0),
                layout=prism.ROPE_HALVES if case["layout"] == "halves" else prism.ROPE_ADJACENT,
                ladder=prism.ROPE_ONE_LADDER if case["ladder"] == "one" else prism.ROPE_AXIS_LADDER,
                inverse=int(case["inverse"]), base=10000.0, in_token_stride=s["x"].stride(0),
                in_head_stride=s["x"].stride(1), out_token_stride=s["out"].stride(0),
                out_head_stride=s["out"].stride(1), pos_stride=s["pos"].stride(0))
        eng.rope(call, s["x"].data_ptr(), s["pos"].data_ptr(), s["out"].data_ptr(), stream)
        return s["out"]
    if kind == "seq":
        q, k, v, o = s["q"], s["k"], s["v"], s["out"]
        if call is None:
            call = s["call"] = prism.SeqAttnPush(
                dtype=dt, n_seqs=case["seqs"], n_q=q.shape[0], n_k=k.shape[0], n_heads=case["heads"],
                n_kv_heads=case["kv_heads"], head_dim=hd, left=case["left"], right=case["right"],
                sinks=case["sinks"], scale=1.0 / math.sqrt(hd), q_token_stride=q.stride(0), q_head_stride=q.stride(1),
                k_token_stride=k.stride(0), k_head_stride=k.stride(1), v_token_stride=v.stride(0),
                v_head_stride=v.stride(1), out_token_stride=o.stride(0), out_head_stride=o.stride(1))
        eng.seq_attn(call, q.data_ptr(), k.data_ptr(), v.data_ptr(), s["cu_q"].data_ptr(), s["cu_k"].data_ptr(),
                     o.data_ptr(), stream)
        return o
    if call is None:
        cache = prism.CacheDesc(dtype=dt, n_kv_heads=case["kv_heads"], head_dim=hd, page_size=case["page"],
                                n_pages=s["k_pages"].shape[0], n_seqs=case["seqs"], table_pages=s["table"].shape[1])
        if kind == "append":
            call = prism.AppendPush(cache=cache, n_new=s["k"].shape[0], k_token_stride=s["k"].stride(0),
                                    k_head_stride=s["k"].stride(1), v_token_stride=s["v"].stride(0),
                                    v_head_stride=s["v"].stride(1))
        else:
            call = prism.PagedAttnPush(cache=cache, n_heads=case["heads"], left=case["left"], sinks=case["sinks"],
                                       max_len=case["max_len"], scale=1.0 / math.sqrt(hd), q_seq_stride=s["q"].stride(0),
                                       q_head_stride=s["q"].stride(1), out_seq_stride=s["out"].stride(0),
                                       out_head_stride=s["out"].stride(1))
            s["ws"] = torch.empty(max(1, eng.paged_attn_workspace(call)), dtype=torch.uint8, device="cuda")
        s["call"] = call
    if kind == "append":
        eng.cache_append(call, s["k"].data_ptr(), s["v"].data_ptr(), s["seq"].data_ptr(), s["pos"].data_ptr(),
                         s["table"].data_ptr(), s["k_pages"].data_ptr(), s["v_pages"].data_ptr(), stream)
        return s["k_pages"], s["v_pages"]
    eng.paged_attn(call, s["q"].data_ptr(), s["k_pages"].data_ptr(), s["v_pages"].data_ptr(), s["table"].data_ptr(),
                   s["lengths"].data_ptr(), s["out"].data_ptr(), s["ws"].data_ptr(), s["ws"].numel(), stream)
    return s["out"]


# ---------------------------------------------------------------- work, exact

def work(case):
    hd = case["head_dim"]
    if case["kind"] == "rope":
        n = case["tokens"] * case["heads"]
        return {"bytes": 4 * n * hd + 12 * case["tokens"], "flops": 6 * n * turned_of(case)}
    if case["kind"] == "append":
        n = sum(spread(case["seqs"], case["min_new"], case["max_new"]))
        return {"bytes": 8 * n * case["kv_heads"] * hd + 12 * n, "flops": 0}
    H, K = case["heads"], case["kv_heads"]
    if case["kind"] == "paged":
        seen = sum(visible_pairs(1, n - 1, case["left"], 0, case["sinks"]) for n in lengths_of(case))
        return {"bytes": 4 * seen * K * hd + 4 * case["seqs"] * H * hd + 4 * seen // case["page"],
                "flops": 4 * seen * H * hd}
    ql = spread(case["seqs"], case["min_q"], case["max_q"])
    seen = sum(visible_pairs(n, case["past"], case["left"], case["right"], case["sinks"]) for n in ql)
    return {"bytes": 4 * sum(ql) * H * hd + 4 * sum(n + case["past"] for n in ql) * K * hd,
            "flops": 4 * seen * H * hd}


def exact_attention(q, k, v, first, left, right, sinks):
    """Softmax attention in 64 bits: q [heads][queries][channels] at positions from `first` on, k and v
    [heads][keys][channels]; query rows a few at a time, each over the keys from its window's start and the sinks."""
    H, n, hd = q.shape
    out = torch.zeros(H, n, hd, dtype=torch.float64, device=q.device)
    keys = torch.arange(k.shape[1], device=q.device)
    for r in range(0, n, 1024):
        p = first + torch.arange(r, min(n, r + 1024), device=q.device)
        hidden = keys[None] > p[:, None] + right
        if left >= 0:
            hidden |= (keys[None] < p[:, None] - left) & (keys[None] >= sinks)
        for h in range(H):
            z = (q[h, r:r + 1024].double() @ k[h * k.shape[0] // H].double().T) / math.sqrt(hd)
            z[hidden] = -math.inf
            out[h, r:r + 1024] = torch.nan_to_num(torch.softmax(z, -1)) @ v[h * v.shape[0] // H].double()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    hd = case["head_dim"]
    if case["kind"] == "rope":
        n, x = turned_of(case), s["x"].double()
        y, i = x.clone(), 0
        for axis, pairs in enumerate((case["pairs_t"], case["pairs_h"], case["pairs_w"])):
            for j in range(pairs):
                f = 10000.0 ** -(i / n if case["ladder"] == "one" else j / pairs)
                phi = s["pos"][axis].double()[:, None] * (-f if case["inverse"] else f)
                a, b = (i, i + n) if case["layout"] == "halves" else (2 * i, 2 * i + 1)
                z = torch.polar(torch.ones_like(phi), phi) * torch.complex(x[..., a], x[..., b])
                y[..., a], y[..., b] = z.real, z.imag
                i += 1
        return y
    if case["kind"] == "append":
        got = []
        for new, pages in (("k", "k_pages"), ("v", "v_pages")):
            pool, page = s[pages].double(), case["page"]
            flat = pool.transpose(1, 2).reshape(-1, case["kv_heads"], hd)  # by slot
            pos, seq = s["pos"].long(), s["seq"].long()
            slot = s["table"].long().reshape(-1)[seq * s["table"].shape[1] + pos // page] * page + pos % page
            flat.index_copy_(0, slot, s[new].double())
            got.append(flat.view(pool.shape[0], page, -1, hd).transpose(1, 2))
        return tuple(got)
    if case["kind"] == "seq":
        cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
        out = []
        for b in range(case["seqs"]):
            q, k, v = s["q"][cq[b]:cq[b + 1]], s["k"][ck[b]:ck[b + 1]], s["v"][ck[b]:ck[b + 1]]
            out.append(exact_attention(q.transpose(0, 1), k.transpose(0, 1), v.transpose(0, 1), len(k) - len(q),
                                       case["left"], case["right"], case["sinks"]).transpose(0, 1))
        return torch.cat(out)
    lengths, page, K = lengths_of(case), case["page"], case["kv_heads"]
    out = torch.empty(case["seqs"], case["heads"], hd, dtype=torch.float64, device="cuda")
    n, width = case["seqs"], max(lengths)
    step = max(1, 16_000_000 // (width * K * hd))  # streams at a time
    at = torch.arange(width, device="cuda")
    for b in range(0, n, step):
        last = s["lengths"][b:b + step].long()[:, None] - 1
        hidden = at > last
        if case["left"] >= 0:
            hidden = hidden | ((at < last - case["left"]) & (at >= case["sinks"]))
        rows = s["table"][b:b + step].long().clamp(min=0)
        k, v = (s[x][rows].transpose(2, 3).flatten(1, 2)[:, :width].double() for x in ("k_pages", "v_pages"))
        q = s["q"][b:b + step].double().unflatten(1, (K, -1))
        z = torch.stack([(q[:, h] @ k[:, :, h].transpose(1, 2).contiguous()) for h in range(K)], 1) / math.sqrt(hd)
        z = torch.softmax(z.masked_fill(hidden[:, None, None], -math.inf), -1)
        o = torch.stack([z[:, h] @ v[:, :, h].contiguous() for h in range(K)], 1)
        out[b:b + step] = o.flatten(1, 2)
    return out
