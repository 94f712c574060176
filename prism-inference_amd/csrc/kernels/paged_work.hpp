/*
 * paged_work.hpp - what the kernels of paged attention share (paged_attn.hpp, paged_attn4.hpp):
 * which keys a wave has, sums over lanes, weights as two 16-bit numbers, the join of a workgroup's waves.
 */
#pragma once
#include "seq_types.hpp"

__device__ __forceinline__ float dot8(h8 a, h8 b, float c) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) c = __builtin_amdgcn_fdot2(h2{a[i], a[i + 1]}, h2{b[i], b[i + 1]}, c, false);
    return c;
}
__device__ __forceinline__ float dot8(b8 a, b8 b, float c) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) c = __builtin_amdgcn_fdot2_f32_bf16(b2{a[i], a[i + 1]}, b2{b[i], b[i + 1]}, c, false);
    return c;
}
/* Sum over groups of W consecutive lanes (2, 4, 8 or 16). */
template <int W>
__device__ __forceinline__ float lanes_sum(float v) {
    if constexpr (W == 2) return v + dpp<0xB1>(v);
    else return group_sum<W>(v);
}
/* The lanes of equal lane % W over the wave, combined by op (row_ror within 16 lanes, then rows). */
template <int W, class F>
__device__ __forceinline__ float across(float v, F op) {
    if constexpr (W <= 8) v = op(v, dpp<0x128>(v));
    if constexpr (W <= 4) v = op(v, dpp<0x124>(v));
    if constexpr (W <= 2) v = op(v, dpp<0x122>(v));
    float a, b;
    lanes_x16(v, a, b);
    lanes_x32(op(a, b), a, b);
    return op(a, b);
}

/* Two weights, each as the sum of two 16-bit numbers: hi has the bits cut off that the type does not hold, lo is what
 * they are, at least `least` where hi is not zero (r < hi then; a median of three is one instruction). */
__device__ __forceinline__ void two_numbers(float z0, float z1, float least, h2& hi, h2& lo) {
    hi = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(z0, z1));
    const float c0 = (float)hi[0], c1 = (float)hi[1];
    lo = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(__builtin_amdgcn_fmed3f(z0 - c0, least, c0),
                                                           __builtin_amdgcn_fmed3f(z1 - c1, least, c1)));
}
__device__ __forceinline__ void two_numbers(float z0, float z1, float least, b2& hi, b2& lo) {
    const unsigned u0 = __builtin_bit_cast(unsigned, z0), u1 = __builtin_bit_cast(unsigned, z1);
    hi = __builtin_bit_cast(b2, __builtin_amdgcn_perm(u1, u0, 0x07060302));
    const float c0 = __builtin_bit_cast(float, u0 & 0xFFFF0000u), c1 = __builtin_bit_cast(float, u1 & 0xFFFF0000u);
    lo = b2{(__bf16)opaque(__builtin_amdgcn_fmed3f(z0 - c0, least, c0)), (__bf16)opaque(__builtin_amdgcn_fmed3f(z1 - c1, least, c1))};
}

/* What a wave has to do: which sequence and heads, and which of the keys seen
 * (in the order: sinks, window). */
struct PagedWork {
    int seq, hk, head, heads; /* first head and number of heads            */
    int split;
    KeyRange kr;
    int i0, i1;
    __device__ __forceinline__ int key(int i) const { return i < kr.sink ? i : kr.lo + i - kr.sink; }
};
__device__ __forceinline__ bool paged_work(const PagedAttnArgs& a, int wave, PagedWork& w) {
    const int group = a.n_heads / a.n_kv_heads;
    /* a launch has fewer than 2^24 workgroups of 256, so items fit 32 bits */
    const unsigned items = (unsigned)a.n_seqs * a.n_kv_heads * a.head_tiles;
    unsigned item;
    int part;
    if (a.waves == 1) {
        item = blockIdx.x * 4 + wave;
        w.split = part = 0;
    } else {
        item = blockIdx.x / (unsigned)a.splits;
        w.split = blockIdx.x - item * a.splits;
        part = w.split * 4 + wave;
    }
    if (item >= items) return false;
    const unsigned tiles = a.head_tiles, kv = a.n_kv_heads, both = item / tiles;
    const int ht = (int)(item - both * tiles);
    w.seq = (int)(both / kv);
    w.hk = (int)(both - w.seq * kv);
    w.head = w.hk * group + ht * PAGED_TILE_HEADS;
    w.heads = min(group - ht * PAGED_TILE_HEADS, PAGED_TILE_HEADS);
    const int n = seq_clamp(a.lengths[w.seq], 0, a.table_pages << a.page_log2);
    w.kr = key_range(n - 1, n, a.left, 0, a.sinks);
    const int seen = w.kr.sink + w.kr.hi - w.kr.lo, parts = a.waves * a.splits;
    const int each = ((seen - 1) / parts + 16) & ~15; /* 16 keys at least; seen = 0: none */
    const int64_t at = (int64_t)part * each;
    w.i0 = at < seen ? (int)at : seen;
    w.i1 = seq_min(seen - w.i0, each) + w.i0;
    return true;
}
/* page of key j, -1 if the table names none of the pool */
__device__ __forceinline__ int paged_page(const PagedAttnArgs& a, const PagedWork& w, int j) {
    const int p = a.table[(int64_t)w.seq * a.table_pages + (j >> a.page_log2)];
    return page_ok(p, a.n_pages) ? p : -1;
}
template <int HD>
__device__ __forceinline__ int64_t paged_at(const PagedAttnArgs& a, const PagedWork& w, int page, int j) {
    return ((((int64_t)page * a.n_kv_heads + w.hk) << a.page_log2) + (j & ((1 << a.page_log2) - 1))) * HD;
}

/* The waves' results of `rows` heads (acc [wave][row][HD], m and l [wave][row] in LDS) into the output or, for
 * splits, the workspace: [seq][head][split] of HD + 2 floats (output, maximum, sum). */
template <class T, int HD>
__device__ __forceinline__ void paged_join_waves(const PagedAttnArgs& a, const PagedWork& w, int rows, const float* acc,
                                                 const float* m, const float* l, int row_stride) {
    for (int e = threadIdx.x; e < rows * HD; e += 256) {
        const int r = e / HD, c = e % HD;
        float top = -INFINITY, sum = 0.f, o = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) top = fmaxf(top, m[k * row_stride + r]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float mk = m[k * row_stride + r];
            const float f = mk == -INFINITY ? 0.f : fast_exp2(mk - top);
            sum = __builtin_fmaf(l[k * row_stride + r], f, sum);
            o = __builtin_fmaf(acc[(k * row_stride + r) * HD + c], f, o);
        }
        if (a.splits == 1) {
            st1<T>(a.out + w.seq * a.out_seq_stride + (w.head + r) * a.out_head_stride + c, sum == 0.f ? 0.f : o / sum);
        } else {
            float* ws = a.ws + (((int64_t)w.seq * a.n_heads + w.head + r) * a.splits + w.split) * (HD + 2);
            ws[c] = o;
            if (c == 0) {
                ws[HD] = top;
                ws[HD + 1] = sum;
            }
        }
    }
}
