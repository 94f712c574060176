/*
 * linear_attn.hpp - linear attention with a decay for each head:
 *   S_t = e^-r S_(t-1) + k_t^T v_t,  o_t = scale q_t S_t
 */
#pragma once
#include "seq_types.hpp"

/* number of the state of sequence s, -1 for none */
__device__ __forceinline__ int linear_state(const LinearAttnArgs& a, int s) {
    const int n = a.state_of ? a.state_of[s] : s;
    return (uint32_t)n < (uint32_t)a.n_states ? n : -1;
}
/* decays are e^-rate: rates below 0 and NaN count as 0 */
__device__ __forceinline__ float linear_rate(const LinearAttnArgs& a, int h) { return fmaxf(a.rates[h], 0.f) * 1.4426950408889634f; }

/* A head of a sequence by a workgroup, token by token: thread (p, c) has rows p, p + P, .. of column c. */
template <class T, int HD>
__device__ __forceinline__ void linear_tokens(const LinearAttnArgs& a) {
    constexpr int P = 256 / HD, R = HD / P;
    __shared__ float part[256];
    const int s = blockIdx.x / a.n_heads, h = blockIdx.x % a.n_heads, hk = h / (a.n_heads / a.n_kv_heads);
    const int c = threadIdx.x % HD, p = threadIdx.x / HD;
    const RowRange rows = row_range(a.cu, s, a.n_seqs, a.n_tokens);
    const int number = linear_state(a, s);
    const int64_t base = ((int64_t)max(number, 0) * a.n_heads + h) * HD * HD;
    const float keep = fast_exp2(-linear_rate(a, h));
    float S[R];
#pragma unroll
    for (int i = 0; i < R; ++i) S[i] = number >= 0 && a.state_in ? a.state_in[base + (p + P * i) * HD + c] : 0.f;
    for (int t = rows.start; t < rows.end; ++t) {
        const uint16_t* q = a.q + t * a.q_token_stride + h * a.q_head_stride;
        const uint16_t* k = a.k + t * a.k_token_stride + hk * a.k_head_stride;
        const float v = ld1<T>(a.v + t * a.v_token_stride + hk * a.v_head_stride + c);
        float o = 0.f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            S[i] = __builtin_fmaf(ld1<T>(k + p + P * i), v, S[i] * keep);
            o = __builtin_fmaf(ld1<T>(q + p + P * i), S[i], o);
        }
        part[threadIdx.x] = o;
        __syncthreads();
        if (p == 0) {
            for (int i = 1; i < P; ++i) o += part[i * HD + c];
            st1<T>(a.out + t * a.out_token_stride + h * a.out_head_stride + c, o * a.scale);
        }
        __syncthreads();
    }
    if (number >= 0 && a.state_out)
#pragma unroll
        for (int i = 0; i < R; ++i) a.state_out[base + (p + P * i) * HD + c] = S[i];
}

/* One token of a sequence and head by a workgroup. */
template <class T, int HD>
__device__ __forceinline__ void linear_step(const LinearAttnArgs& a) {
    constexpr int P = 256 / HD, R = HD / P;
    __shared__ float part[256];
    const int s = blockIdx.x / a.n_heads, h = blockIdx.x % a.n_heads, hk = h / (a.n_heads / a.n_kv_heads);
    const int c = threadIdx.x % HD, p = threadIdx.x / HD;
    const int number = linear_state(a, s);
    uint16_t* out = a.out + s * a.out_token_stride + h * a.out_head_stride + c;
    if (number < 0) {
        if (p == 0) st1<T>(out, 0.f);
        return;
    }
    const int64_t base = ((int64_t)number * a.n_heads + h) * HD * HD;
    const float keep = fast_exp2(-linear_rate(a, h));
    const uint16_t* q = a.q + s * a.q_token_stride + h * a.q_head_stride;
    const uint16_t* k = a.k + s * a.k_token_stride + hk * a.k_head_stride;
    const float v = ld1<T>(a.v + s * a.v_token_stride + hk * a.v_head_stride + c);
    float o = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int64_t at = base + (p + P * i) * HD + c;
        const float S = __builtin_fmaf(ld1<T>(k + p + P * i), v, a.state_in[at] * keep);
        a.state_out[at] = S;
        o = __builtin_fmaf(ld1<T>(q + p + P * i), S, o);
    }
    part[threadIdx.x] = o;
    __syncthreads();
    if (p == 0) {
        for (int i = 1; i < P; ++i) o += part[i * HD + c];
        st1<T>(out, o * a.scale);
    }
}

#define LINEAR(NAME, T, HD)                                                                                                   \
    extern "C" __global__ void __launch_bounds__(256) prism_linear_attn_##NAME##_h##HD(LinearAttnArgs a) { linear_tokens<T, HD>(a); } \
    extern "C" __global__ void __launch_bounds__(256) prism_linear_step_##NAME##_h##HD(LinearAttnArgs a) { linear_step<T, HD>(a); }
LINEAR(f16, F16, 16) LINEAR(f16, F16, 32) LINEAR(f16, F16, 64) LINEAR(f16, F16, 128)
LINEAR(bf16, BF16, 16) LINEAR(bf16, BF16, 32) LINEAR(bf16, BF16, 64) LINEAR(bf16, BF16, 128)
#undef LINEAR
