/*
 * paged_attn.hpp - attention of one new token per sequence over its paged cache.
 *
 * The token is the last of its sequence (position L - 1, L = lengths[s]); it
 * sees the `left` keys before it, itself and the first `sinks` ones:
 *   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c (q.k_j) - m),  c = scale log2 e
 * with a running maximum m, so the keys are read once. Keys of a page that the
 * table does not name properly are not seen. No key: the row is zeros.
 */
#pragma once
#include "seq_types.hpp"

/* one wave a (sequence, head), a key per lane: the simple form */
template <class T, int HD>
__device__ __forceinline__ void paged_attn_body(const PagedAttnArgs& a) {
    const int h = blockIdx.x % a.n_heads, s = blockIdx.x / a.n_heads, lane = lane_id();
    const int hk = h / (a.n_heads / a.n_kv_heads);
    const int64_t cap64 = (int64_t)a.table_pages << a.page_log2;
    const int n = seq_clamp(a.lengths[s], 0, (int)(cap64 > INT32_MAX ? INT32_MAX : cap64));
    const KeyRange kr = key_range(n - 1, n, a.left, 0, a.sinks);
    const uint16_t* q = a.q + s * a.q_seq_stride + h * a.q_head_stride;
    float acc[HD] = {}, m = -INFINITY, l = 0.f;
    const int seen = kr.sink + kr.hi - kr.lo;
    for (int i = lane; i < seen; i += 64) {
        const int j = i < kr.sink ? i : kr.lo + i - kr.sink;
        const int page = a.table[(int64_t)s * a.table_pages + (j >> a.page_log2)];
        if (!page_ok(page, a.n_pages)) continue;
        const int64_t at = ((((int64_t)page * a.n_kv_heads + hk) << a.page_log2) + (j & ((1 << a.page_log2) - 1))) * HD;
        float d = 0.f;
        for (int c = 0; c < HD; ++c) d = __builtin_fmaf(ld1<T>(q + c), ld1<T>(a.k_pages + at + c), d);
        d *= a.scale_log2;
        const float mn = fmaxf(m, d), mu = mn == -INFINITY ? 0.f : mn;
        const float f = exp2f(m - mu), p = exp2f(d - mu);
        l = l * f + p;
#pragma unroll
        for (int c = 0; c < HD; ++c) acc[c] = __builtin_fmaf(p, ld1<T>(a.v_pages + at + c), acc[c] * f);
        m = mn;
    }
    float top = m;
    for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
    const float f = top == -INFINITY ? 0.f : exp2f(m - top);
    l = wave_sum(l * f);
    uint16_t* out = a.out + s * a.out_seq_stride + h * a.out_head_stride;
#pragma unroll
    for (int c = 0; c < HD; ++c) {
        const float o = wave_sum(acc[c] * f);
        if (lane == (c & 63)) st1<T>(out + c, l == 0.f ? 0.f : o / l);
    }
}

#define PAGED_ATTN(NAME, T, HD) \
    extern "C" __global__ void __launch_bounds__(64) prism_paged_attn_##NAME##_h##HD(PagedAttnArgs a) { paged_attn_body<T, HD>(a); }
PAGED_ATTN(f16, F16, 16) PAGED_ATTN(f16, F16, 32) PAGED_ATTN(f16, F16, 64) PAGED_ATTN(f16, F16, 128)
PAGED_ATTN(bf16, BF16, 16) PAGED_ATTN(bf16, BF16, 32) PAGED_ATTN(bf16, BF16, 64) PAGED_ATTN(bf16, BF16, 128)
#undef PAGED_ATTN
