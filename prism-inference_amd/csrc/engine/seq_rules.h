/* seq_rules.h - which calls of the sequence operators are refused, and how their
 * work is split, as functions of the parameters alone (no HIP). Host plain
 * C++. Every check_* returns PRISM_OK or the error code, and why in a text. */
#ifndef PRISM_SEQ_RULES_H
#define PRISM_SEQ_RULES_H

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "../kernel_args.h"
#include "prism.h"

namespace prism {

/* Strides are held to 2^40 elements, and the offset of a buffer's last row to 2^60, so that none passes 64 bits in bytes. */
constexpr int64_t SEQ_MAX_STRIDE = int64_t(1) << 40;
constexpr int64_t SEQ_MAX_OFFSET = int64_t(1) << 60;
/* Rows of a sequence attention and tokens of a table's row: key numbers a tile past the
 * end stay in 32 bits. */
constexpr int64_t SEQ_MAX_ROWS = int64_t(1) << 30;
/* Key rows of a tile, and a linear attention's rows of a chunk, are addressed with 32 bits. */
constexpr int64_t SEQ_MAX_KEY_STRIDE = int64_t(1) << 22;

inline int seq_bad(const char** why, int code, const char* text) {
    if (why) *why = text;
    return code;
}

inline int check_dtype(int32_t dtype, const char** why) {
    return dtype == PRISM_F16 || dtype == PRISM_BF16 ? PRISM_OK
                                                     : seq_bad(why, PRISM_ERR_INVALID, "dtype is neither PRISM_F16 nor PRISM_BF16");
}

inline int check_strides(int64_t rows, int64_t heads, int64_t token, int64_t head, const char** why) {
    if (token < 0 || head < 0 || token % 8 || head % 8 || token > SEQ_MAX_STRIDE || head > SEQ_MAX_STRIDE)
        return seq_bad(why, PRISM_ERR_INVALID, "strides are multiples of 8 from 0 to 2^40");
    /* heads are 2^16 at most */
    if (token > 0 && rows - 1 > (SEQ_MAX_OFFSET - (heads - 1) * head) / token)
        return seq_bad(why, PRISM_ERR_UNSUPPORTED, "rows reach past 2^60 elements");
    return PRISM_OK;
}

/* An output's rows must not overlap: either all heads of a row lie before the
 * next row's, or all rows of a head before the next head's. */
inline int check_out(int64_t rows, int64_t heads, int64_t head_dim, int64_t token, int64_t head, const char** why) {
    if (int rc = check_strides(rows, heads, token, head, why)) return rc;
    const bool rows_apart = (heads == 1 || head >= head_dim) && (rows <= 1 || token >= (heads - 1) * head + head_dim);
    const bool heads_apart = (rows <= 1 || token >= head_dim) && (heads == 1 || head >= (rows - 1) * token + head_dim);
    if (!rows_apart && !heads_apart) return seq_bad(why, PRISM_ERR_INVALID, "output rows overlap");
    return PRISM_OK;
}

inline bool seq_head_dim(int32_t hd) { return hd == 16 || hd == 32 || hd == 64 || hd == 128; }

inline int check_heads(int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, const char** why) {
    if (n_kv_heads < 1 || n_heads < 1 || n_heads > 65536 || n_heads % n_kv_heads)
        return seq_bad(why, PRISM_ERR_INVALID, "n_heads is a multiple of n_kv_heads, from 1 to 65536");
    if (!seq_head_dim(head_dim))
        return seq_bad(why, PRISM_ERR_UNSUPPORTED, "head_dim is 16, 32, 64 or 128");
    return PRISM_OK;
}

/* the kernels work with powers of two */
inline float seq_scale_log2(float scale) { return scale * 1.4426950408889634f; }

inline int check_scale(float scale, const char** why) {
    return scale > 0.f && std::isfinite(seq_scale_log2(scale))
               ? PRISM_OK
               : seq_bad(why, PRISM_ERR_INVALID, "scale is not positive, or too large");
}

inline int check_rope(const prism_rope_push& p, const char** why) {
    if (int rc = check_dtype(p.dtype, why)) return rc;
    if (p.n_tokens < 0 || p.n_heads < 1 || p.n_heads > 65536)
        return seq_bad(why, PRISM_ERR_INVALID, "n_tokens or n_heads out of range");
    if (p.head_dim < 8 || p.head_dim > 256 || p.head_dim % 8)
        return seq_bad(why, PRISM_ERR_UNSUPPORTED, "head_dim is a multiple of 8 up to 256");
    if (p.n_axes < 1 || p.n_axes > 4) return seq_bad(why, PRISM_ERR_INVALID, "n_axes 1 to 4");
    int64_t n = 0;
    for (int a = 0; a < p.n_axes; ++a) {
        if (p.pairs[a] < 0) return seq_bad(why, PRISM_ERR_INVALID, "negative pairs");
        n += p.pairs[a];
    }
    if (n < 1 || 2 * n > p.head_dim) return seq_bad(why, PRISM_ERR_INVALID, "turned pairs do not fit the head");
    if ((p.layout != PRISM_ROPE_HALVES && p.layout != PRISM_ROPE_ADJACENT) ||
        (p.ladder != PRISM_ROPE_AXIS_LADDER && p.ladder != PRISM_ROPE_ONE_LADDER) || (p.inverse != 0 && p.inverse != 1))
        return seq_bad(why, PRISM_ERR_INVALID, "layout, ladder or inverse");
    if (!(p.base >= 1) || !std::isfinite(p.base)) return seq_bad(why, PRISM_ERR_INVALID, "base is less than 1");
    if (p.pos_stride < 0 || p.pos_stride > SEQ_MAX_STRIDE) return seq_bad(why, PRISM_ERR_INVALID, "pos_stride");
    if (int rc = check_strides(p.n_tokens, p.n_heads, p.in_token_stride, p.in_head_stride, why)) return rc;
    return check_out(p.n_tokens, p.n_heads, p.head_dim, p.out_token_stride, p.out_head_stride, why);
}

inline int check_cache(const prism_cache_desc& d, const char** why) {
    if (int rc = check_dtype(d.dtype, why)) return rc;
    if (!seq_head_dim(d.head_dim))
        return seq_bad(why, PRISM_ERR_UNSUPPORTED, "head_dim is 16, 32, 64 or 128");
    if (d.page_size < 1 || d.page_size > 4096 || (d.page_size & (d.page_size - 1)))
        return seq_bad(why, PRISM_ERR_INVALID, "page_size: a power of two up to 4096");
    if (d.n_kv_heads < 1 || d.n_kv_heads > 65536 || d.n_pages < 0 || d.n_seqs < 0 || d.table_pages < 0)
        return seq_bad(why, PRISM_ERR_INVALID, "cache sizes out of range");
    if ((int64_t)d.table_pages * d.page_size > SEQ_MAX_ROWS)
        return seq_bad(why, PRISM_ERR_UNSUPPORTED, "a table row of more than 2^30 tokens");
    if ((int64_t)d.n_pages * d.n_kv_heads * d.page_size > SEQ_MAX_OFFSET / d.head_dim ||
        (int64_t)d.n_seqs * d.table_pages > SEQ_MAX_OFFSET)
        return seq_bad(why, PRISM_ERR_UNSUPPORTED, "a pool or table of more than 2^60 elements");
    return PRISM_OK;
}

inline int check_append(const prism_append_push& p, const char** why) {
    if (int rc = check_cache(p.cache, why)) return rc;
    if (p.n_new < 0) return seq_bad(why, PRISM_ERR_INVALID, "n_new < 0");
    const int64_t heads = p.cache.n_kv_heads;
    if (int rc = check_strides(p.n_new, heads, p.k_token_stride, p.k_head_stride, why)) return rc;
    return check_strides(p.n_new, heads, p.v_token_stride, p.v_head_stride, why);
}

inline int check_paged(const prism_paged_attn_push& p, const char** why) {
    if (int rc = check_cache(p.cache, why)) return rc;
    if (int rc = check_heads(p.n_heads, p.cache.n_kv_heads, p.cache.head_dim, why)) return rc;
    if (p.sinks < 0 || p.max_len < 0) return seq_bad(why, PRISM_ERR_INVALID, "sinks or max_len < 0");
    if (int rc = check_scale(p.scale, why)) return rc;
    if (int rc = check_strides(p.cache.n_seqs, p.n_heads, p.q_seq_stride, p.q_head_stride, why)) return rc;
    return check_out(p.cache.n_seqs, p.n_heads, p.cache.head_dim, p.out_seq_stride, p.out_head_stride, why);
}

inline int check_seq(const prism_seq_attn_push& p, const char** why) {
    if (int rc = check_dtype(p.dtype, why)) return rc;
    if (int rc = check_heads(p.n_heads, p.n_kv_heads, p.head_dim, why)) return rc;
    if (p.n_seqs < 0 || p.n_q < 0 || p.n_k < 0) return seq_bad(why, PRISM_ERR_INVALID, "n_seqs, n_q or n_k < 0");
    if (p.n_q > SEQ_MAX_ROWS || p.n_k > SEQ_MAX_ROWS) return seq_bad(why, PRISM_ERR_UNSUPPORTED, "more than 2^30 rows");
    if (p.sinks < 0) return seq_bad(why, PRISM_ERR_INVALID, "sinks < 0");
    if (int rc = check_scale(p.scale, why)) return rc;
    if (int rc = check_strides(p.n_q, p.n_heads, p.q_token_stride, p.q_head_stride, why)) return rc;
    if (int rc = check_strides(p.n_k, p.n_kv_heads, p.k_token_stride, p.k_head_stride, why)) return rc;
    if (int rc = check_strides(p.n_k, p.n_kv_heads, p.v_token_stride, p.v_head_stride, why)) return rc;
    if (p.k_token_stride > SEQ_MAX_KEY_STRIDE || p.v_token_stride > SEQ_MAX_KEY_STRIDE)
        return seq_bad(why, PRISM_ERR_UNSUPPORTED, "k and v token strides are at most 2^22");
    return check_out(p.n_q, p.n_heads, p.head_dim, p.out_token_stride, p.out_head_stride, why);
}

inline int check_format(int32_t format, const char** why) {
    return format == PRISM_CACHE_16 || format == PRISM_CACHE_4
               ? PRISM_OK
               : seq_bad(why, PRISM_ERR_INVALID, "format is neither PRISM_CACHE_16 nor PRISM_CACHE_4");
}

/* the turn of a rope_append push, as a rope push of `heads` heads */
inline prism_rope_push turn_of(const prism_rope_append_push& p, int32_t heads, int64_t in_token, int64_t in_head) {
    prism_rope_push r = {p.cache.dtype, p.n_new, heads, p.cache.head_dim, p.n_axes, {}, p.layout, p.ladder, 0, p.base,
                         in_token, in_head, p.out_token_stride, p.out_head_stride, p.pos_stride};
    for (int a = 0; a < 4; ++a) r.pairs[a] = p.pairs[a];
    return r;
}

inline int check_rope_append(const prism_rope_append_push& p, const char** why) {
    if (int rc = check_cache(p.cache, why)) return rc;
    if (int rc = check_format(p.format, why)) return rc;
    if (p.n_new < 0 || p.n_heads < 0 || p.n_heads > 65536)
        return seq_bad(why, PRISM_ERR_INVALID, "n_new or n_heads out of range");
    prism_rope_push turn = turn_of(p, 1, 0, 0);
    turn.out_token_stride = turn.head_dim;
    turn.out_head_stride = turn.head_dim;
    turn.n_tokens = 0;
    if (p.n_axes != 0)
        if (int rc = check_rope(turn, why)) return rc;
    const int64_t heads = p.cache.n_kv_heads;
    if (int rc = check_strides(p.n_new, heads, p.k_token_stride, p.k_head_stride, why)) return rc;
    if (int rc = check_strides(p.n_new, heads, p.v_token_stride, p.v_head_stride, why)) return rc;
    if (p.n_heads == 0) return PRISM_OK;
    if (int rc = check_strides(p.n_new, p.n_heads, p.q_token_stride, p.q_head_stride, why)) return rc;
    return check_out(p.n_new, p.n_heads, p.cache.head_dim, p.out_token_stride, p.out_head_stride, why);
}

inline int check_cache_read(const prism_cache_read_push& p, const char** why) {
    if (int rc = check_cache(p.cache, why)) return rc;
    if (int rc = check_format(p.format, why)) return rc;
    if (p.n_rows < 0) return seq_bad(why, PRISM_ERR_INVALID, "n_rows < 0");
    const int64_t heads = p.cache.n_kv_heads;
    if (int rc = check_out(p.n_rows, heads, p.cache.head_dim, p.k_token_stride, p.k_head_stride, why)) return rc;
    return check_out(p.n_rows, heads, p.cache.head_dim, p.v_token_stride, p.v_head_stride, why);
}

inline int check_linear(const prism_linear_attn_push& p, const char** why) {
    if (int rc = check_dtype(p.dtype, why)) return rc;
    if (int rc = check_heads(p.n_heads, p.n_kv_heads, p.head_dim, why)) return rc;
    if (p.n_seqs < 0 || p.n_tokens < 0 || p.n_states < 0)
        return seq_bad(why, PRISM_ERR_INVALID, "n_seqs, n_tokens or n_states < 0");
    if (p.n_tokens > SEQ_MAX_ROWS) return seq_bad(why, PRISM_ERR_UNSUPPORTED, "more than 2^30 rows");
    if (!std::isfinite(p.scale)) return seq_bad(why, PRISM_ERR_INVALID, "scale is not finite");
    if ((int64_t)std::max(p.n_states, p.n_seqs) * p.n_heads > SEQ_MAX_OFFSET / (p.head_dim * p.head_dim))
        return seq_bad(why, PRISM_ERR_UNSUPPORTED, "states of more than 2^60 elements");
    if (int rc = check_strides(p.n_tokens, p.n_heads, p.q_token_stride, p.q_head_stride, why)) return rc;
    if (int rc = check_strides(p.n_tokens, p.n_kv_heads, p.k_token_stride, p.k_head_stride, why)) return rc;
    if (int rc = check_strides(p.n_tokens, p.n_kv_heads, p.v_token_stride, p.v_head_stride, why)) return rc;
    if (p.q_token_stride > SEQ_MAX_KEY_STRIDE || p.k_token_stride > SEQ_MAX_KEY_STRIDE || p.v_token_stride > SEQ_MAX_KEY_STRIDE ||
        p.out_token_stride > SEQ_MAX_KEY_STRIDE)
        return seq_bad(why, PRISM_ERR_UNSUPPORTED, "token strides are at most 2^22");
    return check_out(p.n_tokens, p.n_heads, p.head_dim, p.out_token_stride, p.out_head_stride, why);
}
inline int check_linear_step(const prism_linear_attn_push& p, const char** why) {
    if (int rc = check_linear(p, why)) return rc;
    return p.n_tokens == p.n_seqs ? PRISM_OK : seq_bad(why, PRISM_ERR_INVALID, "a step has one token a sequence");
}

/* How a linear attention is launched: tokens of a segment, and segments (some of them empty). Sequences of one segment each need no
 * first launch and no workspace.
 *
 * A workgroup's chunks follow each other, so few sequences are split; each segment but the first then starts from the sum of those
 * before it, which a launch of its own made: its keys and values are read twice. us without, and in segments of 64, 128, 256, 512,
 * 1024, 1536 (heads x channels), bf16:
 *   1 x 8,160, 8 x 32    206 | 37 22 19 26 43 59        5 x 4,500, 32 x 32   119 | 201 121 95 88 92 92
 *   1 x 8,160, 8 x 128   569 | 220 81 58 70 114 157     5 x 4,500, 32 x 128  352 | 2,385 632 378 318 325 280
 *   2 x 1,000, 8 x 32    29 | 10 12 16 24               64 x 1,000, 8 x 32   40 | 102 77 66 64
 *   3 x 500, 4 x 64      23 | 12 14 19                  64 x 1,000, 8 x 128  160 | 485 312 251 226
 *   1 x 32,000, 4 x 128  2,195 | - - 148 100 125 167    16 x 500, 8 x 128    45 | 58 44 53
 * fp16, whose products are more, takes 1.1 to 1.6 times as long and is best at the same lengths (5 x 4,500, 32 x 128: 547 | 2,413 716 494 444
 * 463 421; 1 x 8,160, 8 x 32: 284 | 39 25 24 33 57 81). Lengths are on the device, so the rule knows their mean alone: 8,160 tokens beside 31 or 63
 * sequences of one token, 8 x 32, are not split and take 206 us (fp16 285), by themselves 20 (24). */
struct LinearPlan {
    int32_t segment;
    bool split;
    int64_t segments;
};
inline LinearPlan linear_plan(const prism_linear_attn_push& p) {
    LinearPlan r = {INT32_MAX, false, std::max(p.n_seqs, 1)};
    const int64_t n_seqs = std::max(p.n_seqs, 1), each = p.n_tokens / n_seqs;
    const bool wide = p.head_dim >= 128; /* two workgroups fill a CU, and states are as large as chunks */
    if (n_seqs * p.n_heads >= (wide ? 256 : 512) || each < 4 * LINEAR_CHUNK) return r;
    /* as many workgroups as the GPU has room for, and segments as long as their number is costly */
    int64_t s = std::max((int64_t)p.n_tokens * p.n_heads / (wide ? 480 : 768), (int64_t)std::sqrt(8.0 * (double)each));
    s = (s + LINEAR_CHUNK - 1) / LINEAR_CHUNK * LINEAR_CHUNK;
    r.segment = (int32_t)s;
    r.split = true;
    r.segments = p.n_tokens / s + n_seqs;
    return r;
}
inline int64_t linear_workspace(const prism_linear_attn_push& p, const LinearPlan& r) {
    return r.split ? r.segments * p.n_heads * p.head_dim * p.head_dim * 4 : 0;
}

/* A launch's threads are counted in 32 bits. */
inline bool seq_grid_ok(int64_t grid, unsigned threads) { return grid <= (int64_t)(UINT32_MAX / threads); }

/* Where each axis' pairs end; returns the number of pairs. */
inline int rope_axes(const prism_rope_push& p, int32_t axis_end[4]) {
    int n = 0;
    for (int a = 0; a < 4; ++a) axis_end[a] = n += a < p.n_axes ? p.pairs[a] : 0;
    return n;
}

/* Tokens per workgroup of a rope launch: as many as the table of angles holds, but
 * not so many that the launch has fewer than 4 workgroups per CU. */
inline int rope_tile(int64_t n_tokens, int n_pairs) {
    const int most = ROPE_TILE_PAIRS / ((n_pairs + 7) & ~7);
    int tile = 1;
    while (2 * tile <= most && n_tokens >= (int64_t)2 * tile * 4 * 256) tile *= 2;
    return tile;
}

/* Tokens per workgroup of a launch that appends, as its tables allow: 12 wave's steps of 64 chunks at least where workgroups stay as many as
 * CUs, and up to 48 where they are many. us at 1, 2, 4, 8, 16, 32 tokens: 24,600 tokens, 48 heads x 128: 150, 126, 123, 132; 8,160,
 * 24 x 32: 23, 14, 12, 11, 12, 16; 50,000: 121, 66, 46, 37, 35, 38; 4,000, 24 x 64: 12, 9, 8, 9, 11; 40,000, 48 x 16: 94, 52, 36, 29, 26, 25. */
inline int append_tile(int64_t n_new, int64_t heads, int head_dim) {
    const int most = APPEND_TILE_CHANNELS / head_dim;
    const auto chunks = [&](int tile) { return tile * heads * (head_dim / 8); };
    int tile = 1;
    while (2 * tile <= most && chunks(tile) < 12 * 64 && n_new / (2 * tile) >= 256) tile *= 2;
    while (2 * tile <= most && chunks(2 * tile) <= 48 * 64 && n_new / (2 * tile) >= 2500) tile *= 2;
    return tile;
}

/* How a paged attention is launched. */
struct PagedPlan {
    bool many;      /* the MFMA kernel */
    int head_tiles; /* per key head */
    int waves;      /* per item: 1 or 4 */
    int splits;     /* workgroups per item */
    int64_t grid;
};
inline PagedPlan paged_plan(const prism_paged_attn_push& p) {
    PagedPlan r;
    const int group = p.n_heads / p.cache.n_kv_heads;
    r.many = group > 2;
    r.head_tiles = (group + PAGED_TILE_HEADS - 1) / PAGED_TILE_HEADS;
    const int64_t items = (int64_t)p.cache.n_seqs * p.cache.n_kv_heads * r.head_tiles;
    /* keys of the longest sequence expected */
    int64_t keys = p.max_len > 0 ? p.max_len : (int64_t)p.cache.table_pages * p.cache.page_size;
    if (p.left >= 0 && keys > (int64_t)p.left + 1 + p.sinks) keys = (int64_t)p.left + 1 + p.sinks;
    /* (Figures with one 16-bit number a weight; with two, 3 heads and more take up to 10 % longer.)
     * A wave alone where the waves are many and short: 64 keys, 1,600 items of 4 heads x 32 and x 128 5.6 and 12.3 us, four
     * waves an item 8.1 and 20.1; 512 items x 128 7.2 (1 head) and 7.5 (4), and 5.1 and 8.2; 200 keys, 512 items x 128 23.5 and
     * 13.2; 4,800 items of 64 to 1,000 keys 8.7 to 115 and 16.2 to 113. */
    r.waves = keys <= 32 || items >= 4096 || (items >= 1024 && keys <= 128) ? 1 : 4;
    /* Splits until the launch has about two workgroups per CU, more of them where a sequence is long (which is where
     * lengths differ); the join costs by the splits, so their number grows with the root of the length; and the
     * second launch has to pay. 1 head x 128 and 4 x 128, us at 1, 4, 16 and 64 splits: 8 items of 1,000 keys 19.2, 9.9, 6.9
     * and 20.2, 11.3, 9.0; of 16,000 372, 98, 30, 18 and 271, 76, 26, 19; 128 items of 1,000 keys 29, 17, 17 and 23, 19,
     * 26; of 16,000 541, 211, 192, 197 and 351, 197, 191, 208; 4 x 32, 8 items of 500 keys 7.4, 7.0. */
    r.splits = 1;
    if (r.waves == 4 && keys >= 384 && keys * p.cache.head_dim >= 32 * 1024) {
        int64_t most = 512 / std::max<int64_t>(items, 1);
        most = std::max(most, std::min(2048 / std::max<int64_t>(items, 1), keys / 1024));
        most = std::min(most, std::min((int64_t)(std::sqrt((double)keys) / 2), keys / 64));
        r.splits = (int)std::max<int64_t>(1, std::min<int64_t>(most, PAGED_MAX_SPLITS));
    }
    r.grid = r.waves == 1 ? (items + 3) / 4 : items * r.splits;
    return r;
}
/* keys that the longest sequence expected sees */
inline int64_t paged_keys(const prism_paged_attn_push& p) {
    const int64_t keys = p.max_len > 0 ? p.max_len : (int64_t)p.cache.table_pages * p.cache.page_size;
    return p.left >= 0 ? std::min(keys, (int64_t)p.left + 1 + p.sinks) : keys;
}
/* The same over a cache of 4 bits. The products' kernel is for more heads, and for all from 64 channels on: a lane's own channels are
 * many there. Splits are as long as those of the longest sequence expected (paged_attn4.hpp), so that of unlike lengths about half
 * have keys: 1,800 workgroups then are as many as the GPU holds at once, and one round of them is fastest. An odd number, so that
 * those that many sequences lack do not fall on the same XCD. us at 1, 5, 8, 9, 15, 16, 25, 63, 95, 191 splits: 24 sequences of 1,000 to
 * 20,001, 32/8 x 128: 218, 98, 98, 70, 77, 98, 77, 107, 127, 202; one of 131,075: 1,215, 255, 165, 147, 95, 89, 62, 43, 42, 46; one of
 * 16,000, 8/1 x 128: 134, 36, 26, 23, 19, 16, 15, 12, 13, 15; 64 of 500 to 4,000, 8 x 128: 55, 49, 60, 52, 62, 70, 75 and more. They go by
 * what is expected, not by the lengths: 24 streams of 4,096 take 36, 38, 75, 183 us where 4,096, 8,192, 32,768, 131,072 are. */
inline PagedPlan paged4_plan(const prism_paged_attn_push& p) {
    PagedPlan r = paged_plan(p);
    r.many = p.n_heads / p.cache.n_kv_heads > 2 || p.cache.head_dim > 32;
    const int64_t items = std::max<int64_t>((int64_t)p.cache.n_seqs * p.cache.n_kv_heads * r.head_tiles, 1), keys = paged_keys(p);
    /* us of waves by themselves, and of four a workgroup: 1,600 items of 300 keys x 64 14.7, 17.8; 520 of 1,000 x 128 43, 26; of 1,000 to 4,000 152, 52 */
    r.waves = keys <= 64 || items >= 4096 || (items >= 1024 && keys <= 400) ? 1 : 4;
    r.splits = 1;
    if (r.waves == 4 && keys >= 384 && keys * p.cache.head_dim >= 32 * 1024) {
        const int64_t most = std::min<int64_t>(std::min(1800 / items, keys / 320), PAGED4_MAX_SPLITS);
        r.splits = (int)std::max<int64_t>(1, (most - 1) | 1);
    }
    r.grid = r.waves == 1 ? (items + 3) / 4 : items * r.splits;
    return r;
}
/* Keys of a wave, of four in each split, so that they do for the longest sequence expected. */
inline int32_t paged4_each(const prism_paged_attn_push& p, const PagedPlan& r) {
    const int64_t each = (paged_keys(p) - 1) / (4 * r.splits) + 64;
    return (int32_t)std::min<int64_t>(each & ~int64_t(63), int64_t(1) << 30);
}
inline int64_t paged_workspace(const prism_paged_attn_push& p, const PagedPlan& r) {
    return r.splits == 1 ? 0 : (int64_t)p.cache.n_seqs * p.n_heads * r.splits * (p.cache.head_dim + 2) * 4;
}

/* Heads that a workgroup of a sequence attention takes side by side: those that share
 * a key head, unless they alone would fill it. */
inline int seq_tile_heads(int n_heads, int n_kv_heads) {
    const int group = n_heads / n_kv_heads;
    return group <= SEQ_ROWS / 4 ? group : 1;
}

/* Tiles of tile_q queries: enough for any lengths (seq_attn.hpp's seq_of_tile). */
inline int64_t seq_tiles(int64_t n_q, int64_t n_seqs, int tile_q) { return n_q / tile_q + n_seqs; }

/* How a sequence attention is launched. The workgroup: 128 rows by 4 waves (four); by 8, of which two share each 32
 * rows' keys (eight); or 64 rows by 8, of which four do (narrow; 128 channels have no LDS for it).
 *
 * More waves to a row shorten a workgroup; four's have the least LDS and registers, so the most of them run at once.
 * By the number of workgroups of 128 rows (those with rows, about) and the keys a query can see. us of four, eight and
 * narrow at 16 | 64 | 128 channels (32 go as 16 do), sequences that see all keys unless a window is named:
 *   workgroups, keys
 *   64, 130       8.2 7.8 7.9      | 8.2 8.8 8.8    | 9.5 10.7
 *   64, 500       10.2 9.5 8.2     | 13.0 11.7 10.5 | 16.4 15.5
 *   160, 2,500    31.5 25.9 17.3   | 41.7 31.7 22.3 | 52.8 41.6
 *   240, 250      9.3 10.9 10.7    | 11.8 11.9 17.6 | 15.9 16.2
 *   256, 1,000    16.7 15.0 15.2   | 21.3 17.7 23.4 | 28.4 24.0
 *   240, window 1,000  18.6 16.1 17.7 | 24.4 20.3 28.3 | 30.3 26.7
 *   320, 500      12.1 12.9 14.9   | 15.9 17.9 25.6 | 21.6 26.2
 *   320, 2,500    32.3 28.2 24.3   | 42.4 32.4 39.7 | 57.1 44.3
 *   320, window 1,000  21.3 21.7 22.8 | 27.1 33.8 39.0 | 36.8 49.2
 *   504, 8,000    89.0 75.1 65.4   | 124 99 116     | 178 147
 *   512, 1,000    19.7 19.0 24.4   | 25.9 31.4 41.2 | 34.9 44.4
 *   756, 8,000    140 131 109      | 185 183 197    | 297 264
 *   1,000, 8,000  110 108 122      | 166 191 232    | 279 288
 *   1,024, 1,000  29.4 34.9 42.6   | 42.8 52.9 79.2 | 62.3 75.3 */
enum { SEQ_FOUR = 0, SEQ_EIGHT = 1, SEQ_NARROW = 2 };
struct SeqPlan {
    int kind;
    int tile_heads, tile_q; /* of a workgroup */
    int64_t grid;
};
inline SeqPlan seq_plan(const prism_seq_attn_push& p) {
    SeqPlan r;
    r.tile_heads = seq_tile_heads(p.n_heads, p.n_kv_heads);
    r.tile_q = SEQ_ROWS / r.tile_heads;
    const int64_t groups = p.n_heads / r.tile_heads, n_seqs = std::max(p.n_seqs, 1);
    const int64_t work = std::max(n_seqs, p.n_q / r.tile_q + n_seqs / 2) * groups;
    int64_t keys = p.n_k / n_seqs;
    if (p.left >= 0 && p.right >= 0) keys = std::min(keys, (int64_t)p.left + p.right + 1 + p.sinks);
    const bool long_keys = work <= 768 && keys >= std::max<int64_t>(384, 5 * work);
    r.kind = SEQ_FOUR;
    if (long_keys || (work <= 256 && keys >= 384)) r.kind = SEQ_EIGHT;
    if ((long_keys && p.head_dim <= 32) || (work <= 160 && keys >= 192 && p.head_dim <= 64)) r.kind = SEQ_NARROW;
    if (r.kind == SEQ_NARROW) r.tile_q = SEQ_NARROW_ROWS / r.tile_heads;
    r.grid = seq_tiles(p.n_q, p.n_seqs, r.tile_q) * groups;
    return r;
}

}  // namespace prism

#endif
