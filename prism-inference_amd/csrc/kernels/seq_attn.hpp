/*
 * seq_attn.hpp - attention along (ragged) sequences with a sliding window and
 * sinks: query i of a sequence of nq queries and nk keys stands at position
 * p = nk - nq + i and sees keys j <= p + right with j >= p - left or j < sinks.
 */
#pragma once
#include "seq_types.hpp"

/* one wave a (query, head), a key per lane: the simple form */
template <class T, int HD>
__device__ __forceinline__ void seq_attn_body(const SeqAttnArgs& a) {
    const int h = blockIdx.x % a.n_heads, row = blockIdx.x / a.n_heads, lane = lane_id();
    const int hk = h / (a.n_heads / a.n_kv_heads);
    RowRange rq{0, 0};
    int s = 0;
    for (; s < a.n_seqs; ++s) {
        rq = row_range(a.cu_q, s, a.n_seqs, a.n_q);
        if (row >= rq.start && row < rq.end) break;
    }
    if (s == a.n_seqs) return;
    const RowRange rk = row_range(a.cu_k, s, a.n_seqs, a.n_k);
    const int nk = rk.end - rk.start, p0 = nk - (rq.end - rq.start) + (row - rq.start);
    const KeyRange kr = key_range(p0, nk, a.left, a.right, a.sinks);
    const uint16_t* q = a.q + row * a.q_token_stride + h * a.q_head_stride;
    float acc[HD] = {}, m = -INFINITY, l = 0.f;
    const int seen = kr.sink + kr.hi - kr.lo;
    for (int i = lane; i < seen; i += 64) {
        const int j = rk.start + (i < kr.sink ? i : kr.lo + i - kr.sink);
        const uint16_t* k = a.k + j * a.k_token_stride + hk * a.k_head_stride;
        const uint16_t* v = a.v + j * a.v_token_stride + hk * a.v_head_stride;
        float d = 0.f;
        for (int c = 0; c < HD; ++c) d = __builtin_fmaf(ld1<T>(q + c), ld1<T>(k + c), d);
        d *= a.scale_log2;
        const float mn = fmaxf(m, d), mu = mn == -INFINITY ? 0.f : mn;
        const float f = exp2f(m - mu), p = exp2f(d - mu);
        l = l * f + p;
#pragma unroll
        for (int c = 0; c < HD; ++c) acc[c] = __builtin_fmaf(p, ld1<T>(v + c), acc[c] * f);
        m = mn;
    }
    float top = m;
    for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
    const float f = top == -INFINITY ? 0.f : exp2f(m - top);
    l = wave_sum(l * f);
    uint16_t* out = a.out + row * a.out_token_stride + h * a.out_head_stride;
#pragma unroll
    for (int c = 0; c < HD; ++c) {
        const float o = wave_sum(acc[c] * f);
        if (lane == (c & 63)) st1<T>(out + c, l == 0.f ? 0.f : o / l);
    }
}

#define SEQ_ATTN(NAME, T, HD) \
    extern "C" __global__ void __launch_bounds__(64) prism_seq_attn_##NAME##_h##HD(SeqAttnArgs a) { seq_attn_body<T, HD>(a); }
SEQ_ATTN(f16, F16, 16) SEQ_ATTN(f16, F16, 32) SEQ_ATTN(f16, F16, 64) SEQ_ATTN(f16, F16, 128)
SEQ_ATTN(bf16, BF16, 16) SEQ_ATTN(bf16, BF16, 32) SEQ_ATTN(bf16, BF16, 64) SEQ_ATTN(bf16, BF16, 128)
#undef SEQ_ATTN
