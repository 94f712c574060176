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

/* x / d by inverse = floor(2^32 / d) (2^32 - 1 for 1), which gives one less at times */
__device__ __forceinline__ uint32_t divide(uint32_t x, uint32_t d, uint32_t inverse) {
    const uint32_t q = __umulhi(x, inverse);
    return x - q * d >= d ? q + 1 : q;
}

/*
 * A workgroup takes a few tokens, as in rope.hpp. Its table holds for each channel what the channel is times and what its partner
 * is times (cos, and sin with its sign), as [token][channel % 8][channel / 8], so that lanes with chunks of 8 side by side read
 * side by side; a 4-bit key is turned in 64 bits, from a table of its own. Waves then take 64 chunks of queries, of keys or of values
 * at a time, two of these in flight: what a wave does is the same for all its lanes, and a lane's channels are always the same.
 * The partners of a chunk come as 8 values from anywhere in the row (a load that need not be aligned).
 *
 * Bound by HBM: 24,600 tokens of 32/8 heads x 128, 4 bits, 538 MB, 126 us (a copy of as much: 105); the vector units are 41 % busy.
 * The first rows are asked for before the angles are taken: 133 and 129.5 us, at 16 bits 141 and 127.
 */
template <class T, int HD, bool FOUR>
__device__ __forceinline__ void rope_append_body(const RopeAppendArgs& a) {
    typedef typename T::v8 v8;
    constexpr int U = 2, CH = HD / 8, TILE = APPEND_TILE_CHANNELS / HD;
    constexpr int BLOCK = CH < 4 ? CH : 4; /* chunks of a 4-bit block, lanes side by side */
    __shared__ __attribute__((aligned(16))) float2 cs[TILE * HD];
    __shared__ __attribute__((aligned(16))) double2 cs64[FOUR ? TILE * HD : 1];
    __shared__ double turns[64];
    __shared__ int64_t slots[TILE];
    const int n = a.n_pairs, lane = lane_id();
    const int64_t t0 = (int64_t)blockIdx.x * a.tile;
    const int tokens = min(a.tile, (int)(a.n_new - t0));
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int H = a.n_heads, K = a.n_kv_heads;
    const int nq = (tokens * H * CH + 63) / 64, nk = (tokens * K * CH + 63) / 64;
    const int k = lane % CH, c = 8 * k; /* the lane's chunk and channels */
    const int turned = max(min(2 * n - c, 8), 0); /* of them, the first */
    /* Partners, other than in the chunk itself: all of the first half n channels on, of the second n back. The chunk with the
       border inside has both, of which the second half's would begin before the row. */
    const bool far = !a.adjacent && turned > 0, border = far && c < n && c + 8 > n;
    const int partner = far ? (c < n ? c + n : c - n) : c; /* at most HD - 8: n is at most HD / 2, and c + 8 - n < 8 here */

    struct Unit {
        int kind, t, h; /* 0 queries, 1 keys, 2 values; -1: none */
        v8 x, other;
    };
    const auto load = [&](int w) {
        Unit u;
        u.kind = w < nq ? 0 : w < nq + nk ? 1 : w < nq + 2 * nk ? 2 : -1;
        if (u.kind < 0) return u;
        const uint32_t heads = u.kind == 0 ? H : K, inverse = u.kind == 0 ? a.by_heads : a.by_kv;
        const uint32_t rows = tokens * heads, row = (w - (u.kind == 0 ? 0 : u.kind == 1 ? nq : nq + nk)) * (64 / CH) + lane / CH;
        const uint32_t in = min(row, rows - 1);
        u.t = divide(in, heads, inverse);
        u.h = in - u.t * heads;
        const uint16_t* m = u.kind == 0 ? a.q : u.kind == 1 ? a.k : a.v;
        const int64_t ts = u.kind == 0 ? a.q_token_stride : u.kind == 1 ? a.k_token_stride : a.v_token_stride;
        const int64_t hs = u.kind == 0 ? a.q_head_stride : u.kind == 1 ? a.k_head_stride : a.v_head_stride;
        const uint16_t* x = m + t0 * ts + ((uint32_t)u.t * ts + (uint32_t)u.h * hs);
        u.x = ld8<T>(x + c);
        if (u.kind < 2 && !a.adjacent) {
            u.other = ld8_any<T>(x + partner);
            if (border) {
                const v8 back = shift_up(ld8<T>(x), n & 7);
#pragma unroll
                for (int e = 0; e < 8; ++e) u.other[e] = e >= (n & 7) ? back[e] : u.other[e];
            }
        }
        if (row >= rows) u.t = -1; /* past the end: read, not written */
        return u;
    };
    /* The first rows are asked for before the angles. In place, a row's lanes, which are in one wave, have all read before
       one writes. */
    Unit u[U];
#pragma unroll
    for (int i = 0; i < U; ++i) u[i] = load(wave + 4 * i);
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
        const int i1 = t * HD + c1 % 8 * CH + c1 / 8, i2 = t * HD + c2 % 8 * CH + c2 / 8;
        cs[i1] = float2{(float)c, -(float)s};
        cs[i2] = float2{(float)c, (float)s};
        if constexpr (FOUR) {
            cs64[i1] = double2{c, -s};
            cs64[i2] = double2{c, s};
        }
    }
    __syncthreads();

    const auto keep = [&](const Unit& u, const float (&y)[8], v8 o) { /* into the cache; a block's lanes are all here */
        uint8_t* pages = u.kind == 1 ? a.k_pages : a.v_pages;
        const int64_t slot = slots[max(u.t, 0)], at = slot + ((int64_t)u.h << a.page_log2);
        const bool on = u.t >= 0 && slot >= 0;
        if constexpr (!FOUR) {
            if (on) st8<T>(reinterpret_cast<uint16_t*>(pages) + at * HD + c, o);
        } else {
            float top = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) top = vmax(top, __builtin_fabsf(y[e])); /* NaN stays */
            top = vmax(top, dpp<0xB1>(top));
            if constexpr (BLOCK == 4) top = vmax(top, dpp<0x4E>(top));
            if (!on) return;
            const uint32_t bits = __builtin_bit_cast(uint32_t, top);
            /* 1.75 * 2^k = 7 * 2^(k-2) */
            int e = (int)(bits >> 23) - 129 + ((bits & 0x7FFFFFu) > 0x600000u);
            e = seq_clamp(e, Fp4<T>::low, Fp4<T>::high);
            const bool fine = top < INFINITY;
            const float s = fp4_scale(e + 127);
            uint32_t w = 0;
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[0], y[1], s, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], s, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[4], y[5], s, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[6], y[7], s, 3);
            *reinterpret_cast<uint32_t*>(pages + at * (HD / 2) + c / 2) = fine ? w : 0;
            if (k % BLOCK == 0) (u.kind == 1 ? a.k_scales : a.v_scales)[at * (CH / BLOCK) + k / BLOCK] = fine ? (uint8_t)(e + 127) : 255;
        }
    };
    const bool none = turned == 0, some = !none && turned < 8;
    const auto work = [&](const Unit& u) {
        if (u.kind < 0) return;
        float y[8], z[8], p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = (float)u.x[e];
        if (u.kind == 2) {
            keep(u, y, u.x);
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = a.adjacent ? y[e ^ 1] : (float)u.other[e];
        const int at = max(u.t, 0) * HD + k;
        if (!FOUR || u.kind == 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float2 f = cs[at + e * CH];
                z[e] = __builtin_fmaf(y[e], f.x, p[e] * f.y);
            }
            u4 w, x = __builtin_bit_cast(u4, u.x);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{opaque(z[2 * e]), opaque(z[2 * e + 1])}), typename T::v2));
            v8 o = __builtin_bit_cast(v8, none ? x : w); /* what does not turn keeps its bits, those of a NaN too */
            if (some)
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = e < turned ? o[e] : u.x[e];
            if (u.kind == 1) keep(u, y, o);
            else if (u.t >= 0)
                st8<T>(a.q_out + t0 * a.out_token_stride + ((uint32_t)u.t * a.out_token_stride + (uint32_t)u.h * a.out_head_stride) + c, o);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const double2 f = cs64[at + e * CH];
                z[e] = (float)__builtin_fma((double)y[e], f.x, (double)p[e] * f.y);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = none || (some && e >= turned) ? y[e] : z[e];
            keep(u, y, u.x);
        }
    };
    for (int w = wave; w < nq + 2 * nk;) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < U; ++i) work(u[i]);
        w += 4 * U;
#pragma unroll
        for (int i = 0; i < U; ++i) u[i] = load(w + 4 * i);
    }
}

template <class T, int HD, bool FOUR>
__device__ __forceinline__ void cache_read_body(const CacheReadArgs& a) {
    constexpr int CH = HD / 8, BLOCK = CH < 4 ? CH : 4;
    const uint32_t id = blockIdx.x * 256 + threadIdx.x, row = id / CH; /* 32 bits: a launch has fewer than 2^32 threads */
    const int c = id % CH;
    const int64_t t = divide(row, a.n_kv_heads, a.by_kv);
    const int h = (int)(row - (uint32_t)t * a.n_kv_heads);
    if (t >= a.n_rows) return;
    const int64_t slot = a.n_seqs > 0 ? cache_slot(a, a.seq_of[t], a.pos_of[t]) : -1; /* no sequences: no arrays either */
    typename T::v8 k{}, v{};
    if (slot >= 0) {
        const int64_t at = slot + ((int64_t)h << a.page_log2), i = at * CH + c;
        if constexpr (FOUR) {
            const int64_t j = at * (CH / BLOCK) + c / BLOCK;
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

#define CACHE4(NAME, T, HD)                                                                                                        \
    extern "C" __global__ void __launch_bounds__(256) prism_rope_append_##NAME##_h##HD(RopeAppendArgs a) { rope_append_body<T, HD, false>(a); } \
    extern "C" __global__ void __launch_bounds__(256) prism_rope_append4_##NAME##_h##HD(RopeAppendArgs a) { rope_append_body<T, HD, true>(a); } \
    extern "C" __global__ void __launch_bounds__(256) prism_cache_read4_##NAME##_h##HD(CacheReadArgs a) { cache_read_body<T, HD, true>(a); }
CACHE4(f16, F16, 16) CACHE4(f16, F16, 32) CACHE4(f16, F16, 64) CACHE4(f16, F16, 128)
CACHE4(bf16, BF16, 16) CACHE4(bf16, BF16, 32) CACHE4(bf16, BF16, 64) CACHE4(bf16, BF16, 128)
#undef CACHE4
#define CACHE16(HD) \
    extern "C" __global__ void __launch_bounds__(256) prism_cache_read_h##HD(CacheReadArgs a) { cache_read_body<F16, HD, false>(a); }
CACHE16(16) CACHE16(32) CACHE16(64) CACHE16(128)
#undef CACHE16
