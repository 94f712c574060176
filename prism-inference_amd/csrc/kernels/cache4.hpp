/*
 * cache4.hpp - new tokens into a paged cache of 16 or 4 bits, keys and queries
 * turned on the way, and rows of such a cache back.
 *
 * A 4-bit block: 32 channels of a head (16 of 16) share the power 2^e, the smallest with
 * max |x| <= 7 * 2^e (7 rounds to 6, as anything does up to half a step past 6); a
 * value is the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 to |x| 2^-e, ties to even,
 * which is what the conversion instruction does.
 */
#pragma once
#include "seq_types.hpp"

template <class T>
struct Fp4;
template <>
struct Fp4<F16> {
    static constexpr int low = FP4_LOW_F16, high = FP4_HIGH_F16;
    template <int BYTE>
    static __device__ __forceinline__ h2 two(uint32_t w, float scale) {
        return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, BYTE);
    }
};
template <>
struct Fp4<BF16> {
    static constexpr int low = FP4_LOW_BF16, high = FP4_HIGH_BF16;
    template <int BYTE>
    static __device__ __forceinline__ b2 two(uint32_t w, float scale) {
        return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, BYTE);
    }
};
/* A block's byte as the scale that the conversions take: 2^(b - 127), NaN for 255. */
__device__ __forceinline__ float fp4_scale(uint32_t b) { return __builtin_bit_cast(float, b << 23); }
/* 8 channels (4 bytes of codes) as 16-bit values: exact. */
template <class T>
__device__ __forceinline__ typename T::v8 fp4_values(uint32_t w, float scale) {
    typename T::v2 r[4] = {Fp4<T>::template two<0>(w, scale), Fp4<T>::template two<1>(w, scale),
                           Fp4<T>::template two<2>(w, scale), Fp4<T>::template two<3>(w, scale)};
    typename T::v8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = r[i / 2][i % 2];
    return v;
}

/* Where token pos of sequence s lies: its slot's number in [page][head][slot] for head 0, -1 for none. */
template <class Args>
__device__ __forceinline__ int64_t cache_slot(const Args& a, int s, int pos) {
    if ((uint32_t)s >= (uint32_t)a.n_seqs || pos < 0) return -1;
    const int slot_page = pos >> a.page_log2;
    if (slot_page >= a.table_pages) return -1;
    const int page = a.table[(int64_t)s * a.table_pages + slot_page];
    if (!page_ok(page, a.n_pages)) return -1;
    return (((int64_t)page * a.n_kv_heads) << a.page_log2) + (pos & ((1 << a.page_log2) - 1));
}

/* 8 channels of a row that turns, from channel c on: x as it is kept, y in fp32. cs: cos and sin of the token's pairs. */
template <class T>
__device__ __forceinline__ void turned8(const RopeAppendArgs& a, const uint16_t* row, int c, const double2* cs,
                                        typename T::v8& x, float (&y)[8]) {
    const int n = a.n_pairs;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int at = c + e;
        if (at < 2 * n) {
            const bool second = a.adjacent ? at & 1 : at >= n;
            const int pair = a.adjacent ? at >> 1 : second ? at - n : at;
            const double other = ld1<T>(row + (a.adjacent ? at ^ 1 : second ? at - n : at + n));
            const double2 k = cs[pair];
            y[e] = (float)__builtin_fma((double)y[e], k.x, second ? other * k.y : -(other * k.y));
            x[e] = (typename T::el)opaque(y[e]);
        }
    }
}

template <class T, bool FOUR>
__device__ __forceinline__ void rope_append_body(const RopeAppendArgs& a) {
    __shared__ __attribute__((aligned(16))) double2 cs[ROPE_TILE_PAIRS]; /* [token][np] cos, sin */
    __shared__ double turns[64];
    const int n = a.n_pairs, np = (n + 7) & ~7;
    const int t0 = blockIdx.x * a.tile, tokens = min(a.tile, a.n_new - t0);
    const auto axis_of = [&](int j) { return (j >= a.axis_end[0]) + (j >= a.axis_end[1]) + (j >= a.axis_end[2]); };
    if (threadIdx.x < n) {
        const int j = threadIdx.x, axis = axis_of(j), first = axis ? a.axis_end[axis - 1] : 0;
        const double e = a.one_ladder ? (double)j / n : (double)(j - first) / (a.axis_end[axis] - first);
        turns[j] = a.turn * exp2(-e * a.log2_base);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < tokens * np; i += 256) {
        const int t = i / np, j = i - t * np;
        if (j < n) {
            const double rev = (double)a.pos[axis_of(j) * a.pos_stride + t0 + t] * turns[j];
            double s, c;
            sincospi(2.0 * (rev - rint(rev)), &s, &c);
            cs[i] = double2{c, s};
        }
    }
    __syncthreads();
    const int chunks = a.head_dim / 8, H = a.n_heads, K = a.n_kv_heads;
    const int per_token = (H + 2 * K) * chunks, units = tokens * per_token;
    const int block = FOUR ? min(chunks, 4) : 1; /* chunks of a 4-bit block */
    for (int u = threadIdx.x; u < units; u += 256) { /* a block's lanes are together: chunks is a power of two */
        const int t = u / per_token, r = u - t * per_token, row = r / chunks, c = r % chunks * 8;
        const int64_t tok = t0 + t;
        const bool query = row < H, value = row >= H + K;
        const int h = query ? row : value ? row - H - K : row - H;
        const uint16_t* x = query   ? a.q + tok * a.q_token_stride + h * a.q_head_stride
                            : value ? a.v + tok * a.v_token_stride + h * a.v_head_stride
                                    : a.k + tok * a.k_token_stride + h * a.k_head_stride;
        typename T::v8 o = ld8<T>(x + c);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = (float)o[e];
        if (!value) turned8<T>(a, x, c, cs + t * np, o, y);
        /* in place, a row's lanes, which are in one wave, have all read before one writes */
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (query) st8<T>(a.q_out + tok * a.out_token_stride + h * a.out_head_stride + c, o);
        float top = 0.f;
        bool fine = true;
        if constexpr (FOUR) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                top = fmaxf(top, fabsf(y[e]));
                fine = fine && fabsf(y[e]) < INFINITY;
            }
            top = fine ? top : INFINITY;
            for (int w = 1; w < block; w *= 2) top = fmaxf(top, __shfl_xor(top, w));
        }
        const int64_t slot = query ? -1 : cache_slot(a, a.seq_of[tok], a.pos_of[tok]);
        if (slot < 0) continue;
        const int64_t at = slot + ((int64_t)h << a.page_log2);
        if constexpr (!FOUR) {
            st8<T>(reinterpret_cast<uint16_t*>(value ? a.v_pages : a.k_pages) + at * a.head_dim + c, o);
        } else {
            const uint32_t bits = __builtin_bit_cast(uint32_t, top);
            /* 1.75 * 2^k = 7 * 2^(k-2) */
            int e = (int)(bits >> 23) - 129 + ((bits & 0x7FFFFFu) > 0x600000u);
            e = seq_clamp(e, Fp4<T>::low, Fp4<T>::high);
            uint32_t w = 0;
            if (top < INFINITY) {
                const float s = fp4_scale(e + 127);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[0], y[1], s, 0);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], s, 1);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[4], y[5], s, 2);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[6], y[7], s, 3);
            }
            *reinterpret_cast<uint32_t*>((value ? a.v_pages : a.k_pages) + at * (a.head_dim / 2) + c / 2) = w;
            if (c / 8 % block == 0)
                (value ? a.v_scales : a.k_scales)[at * (chunks / block) + c / 8 / block] = top < INFINITY ? (uint8_t)(e + 127) : 255;
        }
    }
}

template <class T, bool FOUR>
__device__ __forceinline__ void cache_read_body(const CacheReadArgs& a) {
    const int chunks = a.head_dim / 8, block = min(chunks, 4);
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t per_token = (int64_t)a.n_kv_heads * chunks;
    if (id >= a.n_rows * per_token) return;
    const int64_t t = id / per_token;
    const int r = (int)(id - t * per_token), h = r / chunks, c = r % chunks;
    const int64_t slot = a.n_seqs > 0 ? cache_slot(a, a.seq_of[t], a.pos_of[t]) : -1; /* no sequences: no arrays either */
    typename T::v8 k{}, v{};
    if (slot >= 0) {
        const int64_t at = slot + ((int64_t)h << a.page_log2), i = at * chunks + c;
        if constexpr (FOUR) {
            const int64_t j = at * (chunks / block) + c / block;
            k = fp4_values<T>(reinterpret_cast<const uint32_t*>(a.k_pages)[i], fp4_scale(a.k_scales[j]));
            v = fp4_values<T>(reinterpret_cast<const uint32_t*>(a.v_pages)[i], fp4_scale(a.v_scales[j]));
        } else {
            k = ld8<T>(reinterpret_cast<const uint16_t*>(a.k_pages) + i * 8);
            v = ld8<T>(reinterpret_cast<const uint16_t*>(a.v_pages) + i * 8);
        }
    }
    st8<T>(a.k + t * a.k_token_stride + h * a.k_head_stride + 8 * c, k);
    st8<T>(a.v + t * a.v_token_stride + h * a.v_head_stride + 8 * c, v);
}

#define CACHE4(NAME, T)                                                                                                      \
    extern "C" __global__ void __launch_bounds__(256) prism_rope_append_##NAME(RopeAppendArgs a) { rope_append_body<T, false>(a); } \
    extern "C" __global__ void __launch_bounds__(256) prism_rope_append4_##NAME(RopeAppendArgs a) { rope_append_body<T, true>(a); } \
    extern "C" __global__ void __launch_bounds__(256) prism_cache_read4_##NAME(CacheReadArgs a) { cache_read_body<T, true>(a); }
CACHE4(f16, F16) CACHE4(bf16, BF16)
#undef CACHE4
extern "C" __global__ void __launch_bounds__(256) prism_cache_read(CacheReadArgs a) { cache_read_body<F16, false>(a); }
