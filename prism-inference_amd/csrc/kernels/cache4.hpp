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

/* 8 values from anywhere in a row. */
template <class T>
__device__ __forceinline__ typename T::v8 ld8_any(const uint16_t* p) {
    typename T::v8 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}
/* v moved up by s elements (1 to 7), the lowest undefined */
template <class V>
__device__ __forceinline__ V shift_up(V v, int s) {
    union {
        V v;
        uint64_t w[2];
    } x{v}, y;
    const int bits = 16 * (s & 3);
    y.w[0] = x.w[0] << bits;
    y.w[1] = s >= 4 ? x.w[0] << bits : x.w[1] << bits | (bits ? x.w[0] >> (64 - bits) : 0);
    return y.v;
}

/* A chunk of 8 channels from c on of a row: itself, and the channels that its own turn with. */
template <class T>
struct Turned8 {
    typename T::v8 x, other;
};
template <class T>
__device__ __forceinline__ Turned8<T> turn_load(const RopeAppendArgs& a, const uint16_t* row, int c, bool turns) {
    Turned8<T> r;
    r.x = ld8<T>(row + c);
    r.other = r.x;
    const int n = a.n_pairs;
    if (!a.adjacent && turns && c < 2 * n) {
        /* All 8 of the first half: n channels on (16 more fit the row: n is at most head_dim / 2). The second: n back. The
           chunk with the border inside has both, of which the second half's would begin before the row. */
        r.other = ld8_any<T>(row + (c < n ? c + n : c - n));
        if (c < n && c + 8 > n) {
            const typename T::v8 back = shift_up(ld8<T>(row), n & 7);
#pragma unroll
            for (int e = 0; e < 8; ++e) r.other[e] = e >= (n & 7) ? back[e] : r.other[e];
        }
    }
    return r;
}

/* Tokens by a workgroup as in rope.hpp; the table holds for each channel what it is times and what its partner is times
 * (cos, and sin with its sign), as [token][channel % 8][channel / 8], so that lanes with chunks side by side read
 * side by side. A 4-bit key is turned in 64 bits, from a table of its own. */
template <class T, bool FOUR>
__device__ __forceinline__ void rope_append_body(const RopeAppendArgs& a) {
    typedef typename T::v8 v8;
    typedef typename T::el el;
    constexpr int U = 2;
    __shared__ __attribute__((aligned(16))) float2 cs[APPEND_TILE_CHANNELS];
    __shared__ __attribute__((aligned(16))) double2 cs64[FOUR ? APPEND_TILE_CHANNELS : 1];
    __shared__ double turns[64];
    __shared__ int64_t slots[APPEND_TILE_CHANNELS / 16];
    const int n = a.n_pairs, hd = a.head_dim, chunks = hd / 8, lc = __builtin_ctz(chunks);
    const int t0 = blockIdx.x * a.tile, tokens = min(a.tile, a.n_new - t0);
    const auto axis_of = [&](int j) { return (j >= a.axis_end[0]) + (j >= a.axis_end[1]) + (j >= a.axis_end[2]); };
    if (threadIdx.x < n) {
        const int j = threadIdx.x, axis = axis_of(j), first = axis ? a.axis_end[axis - 1] : 0;
        const double e = a.one_ladder ? (double)j / n : (double)(j - first) / (a.axis_end[axis] - first);
        turns[j] = a.turn * exp2(-e * a.log2_base);
    }
    if (a.n_kv_heads > 0 && threadIdx.x < tokens)
        slots[threadIdx.x] = cache_slot(a, a.seq_of[t0 + threadIdx.x], a.pos_of[t0 + threadIdx.x]);
    __syncthreads();
    for (int i = threadIdx.x; i < tokens * n; i += 256) {
        const int t = i / n, j = i - t * n;
        const double rev = (double)a.pos[axis_of(j) * a.pos_stride + t0 + t] * turns[j];
        double s, c;
        sincospi(2.0 * (rev - rint(rev)), &s, &c);
        const int c1 = a.adjacent ? 2 * j : j, c2 = a.adjacent ? c1 + 1 : j + n;
        const int i1 = t * hd + c1 % 8 * chunks + c1 / 8, i2 = t * hd + c2 % 8 * chunks + c2 / 8;
        cs[i1] = float2{(float)c, -(float)s};
        cs[i2] = float2{(float)c, (float)s};
        if constexpr (FOUR) {
            cs64[i1] = double2{c, -s};
            cs64[i2] = double2{c, s};
        }
    }
    __syncthreads();
    const int H = a.n_heads, K = a.n_kv_heads;
    const int per_token = (H + 2 * K) << lc;
    const int block = FOUR ? min(chunks, 4) : 1; /* chunks of a 4-bit block: lanes side by side, chunks is a power of two */
    const int dt = 256 / per_token, dr = 256 % per_token;
    int t = threadIdx.x / per_token, r = threadIdx.x % per_token;
    while (t < tokens) {
        Turned8<T> v[U];
        int tt[U], row[U], c[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            tt[u] = t < tokens ? t : -1;
            row[u] = r >> lc;
            c[u] = (r & (chunks - 1)) * 8;
            const int64_t tok = t0 + min(t, tokens - 1); /* past the end: read, not written */
            const uint16_t* x = row[u] < H     ? a.q + tok * a.q_token_stride + row[u] * a.q_head_stride
                                : row[u] < H + K ? a.k + tok * a.k_token_stride + (row[u] - H) * a.k_head_stride
                                               : a.v + tok * a.v_token_stride + (row[u] - H - K) * a.v_head_stride;
            v[u] = turn_load<T>(a, x, c[u], row[u] < H + K);
            t += dt;
            r += dr;
            if (r >= per_token) {
                r -= per_token;
                ++t;
            }
        }
        /* in place, a row's lanes, which are in one wave, have all read before one writes */
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (tt[u] < 0) continue;
            const bool query = row[u] < H, value = row[u] >= H + K;
            const int h = query ? row[u] : value ? row[u] - H - K : row[u] - H;
            v8 o = v[u].x;
            if (a.adjacent) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[u].other[e] = v[u].x[e ^ 1];
            }
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = (float)o[e];
            if (!value) {
                const int at = tt[u] * hd + c[u] / 8;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (c[u] + e >= 2 * n) break;
                    const float other = (float)v[u].other[e];
                    if (!FOUR || query) {
                        const float2 k = cs[at + e * chunks];
                        y[e] = __builtin_fmaf(y[e], k.x, other * k.y);
                    } else {
                        const double2 k = cs64[at + e * chunks];
                        y[e] = (float)__builtin_fma((double)y[e], k.x, (double)other * k.y);
                    }
                    o[e] = (el)opaque(y[e]);
                }
            }
            if (query) {
                st8<T>(a.q_out + (t0 + tt[u]) * a.out_token_stride + h * a.out_head_stride + c[u], o);
                continue;
            }
            const int64_t slot = slots[tt[u]];
            const int64_t at = slot + ((int64_t)h << a.page_log2);
            if constexpr (!FOUR) {
                if (slot >= 0) st8<T>(reinterpret_cast<uint16_t*>(value ? a.v_pages : a.k_pages) + at * hd + c[u], o);
            } else {
                float top = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) top = vmax(top, __builtin_fabsf(y[e])); /* NaN stays */
                top = vmax(top, dpp<0xB1>(top));
                if (block == 4) top = vmax(top, dpp<0x4E>(top));
                if (slot < 0) continue;
                const uint32_t bits = __builtin_bit_cast(uint32_t, top);
                /* 1.75 * 2^k = 7 * 2^(k-2) */
                int e = (int)(bits >> 23) - 129 + ((bits & 0x7FFFFFu) > 0x600000u);
                e = seq_clamp(e, Fp4<T>::low, Fp4<T>::high);
                const bool fine = top < INFINITY;
                uint32_t w = 0;
                const float s = fp4_scale(e + 127);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[0], y[1], s, 0);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], s, 1);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[4], y[5], s, 2);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[6], y[7], s, 3);
                *reinterpret_cast<uint32_t*>((value ? a.v_pages : a.k_pages) + at * (hd / 2) + c[u] / 2) = fine ? w : 0;
                if ((c[u] / 8 & (block - 1)) == 0)
                    (value ? a.v_scales : a.k_scales)[at * (chunks / block) + c[u] / 8 / block] = fine ? (uint8_t)(e + 127) : 255;
            }
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
