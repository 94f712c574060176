/*
 * rope.hpp - rotary positions with several axes.
 *
 * Pair i of a head's channels (a, b) turns by phi = pos[axis(i)] * f_i:
 *   a' = a cos phi - b sin phi,  b' = b cos phi + a sin phi
 * with f_i = base^-e_i in turns (64 bits, negated for the inverse). phi is
 * reduced to [-1/2, 1/2] turns in 64 bits, so a position of millions keeps its
 * angle, and sin / cos are taken in fp32.
 *
 * All heads of a token turn by the same angles, and an angle (64-bit product,
 * reduction, sincos: ~80 instructions) costs far more than a turn, so a
 * workgroup takes a few tokens, puts their angles' cos and sin into LDS, and
 * then streams the tokens' rows. A unit is 8 pairs of one head: two chunks of 16
 * bytes (HALVES: channels i.. and i + n.., ADJACENT: 16 channels in a row; two
 * chunks of channels that do not turn), two units a thread in flight. HALVES
 * with n not a multiple of 8, whose second operands lie on no 16-byte boundary,
 * takes them from LDS, a chunk of 8 channels at a time. Bound by HBM traffic: x
 * read and written once.
 */
#pragma once
#include "seq_types.hpp"

/* (u, w) turned by (cos, sin) cs */
template <class T>
__device__ __forceinline__ void rope_turn(typename T::el& u, typename T::el& w, float2 cs) {
    const float a = (float)u, b = (float)w;
    u = (typename T::el)opaque(__builtin_fmaf(a, cs.x, -(b * cs.y)));
    w = (typename T::el)opaque(__builtin_fmaf(b, cs.x, a * cs.y));
}

/* Units of two aligned chunks: HALVES with n % 8 == 0, ADJACENT. */
template <class T, bool ADJACENT>
__device__ __forceinline__ void rope_units(const RopeArgs& a, const float2* cs, int np, int t0, int tokens) {
    typedef typename T::v8 v8;
    typedef typename T::el el;
    constexpr int U = 2;
    const int n = a.n_pairs, chunks = a.head_dim / 8;
    const int turned = ADJACENT ? (2 * n + 15) / 16 : n / 8;
    const int rest = chunks - 2 * turned; /* chunks behind them, of an odd number the last alone; -1: the last unit's own */
    const int per_head = turned + (a.copy && rest > 0 ? (rest + 1) / 2 : 0);
    const int per_token = per_head * a.n_heads, units = tokens * per_token;
    for (int u0 = threadIdx.x; u0 < units; u0 += 256 * U) {
        v8 p[U], q[U];
        uint16_t* y[U];
        int c1[U], c2[U], pair[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = min(u0 + 256 * i, units - 1); /* past the end: the last one, read and not written */
            const int t = u / per_token, r = u - t * per_token, h = r / per_head, k = r - h * per_head;
            const bool turn = k < turned;
            c1[i] = ADJACENT || !turn ? 2 * k : k;
            if (!ADJACENT && !turn) c1[i] = 2 * turned + 2 * (k - turned);
            c2[i] = min(ADJACENT || !turn ? c1[i] + 1 : k + turned, chunks - 1);
            pair[i] = turn ? t * np + 8 * k : -1;
            const uint16_t* x = a.in + (t0 + t) * a.in_token_stride + h * a.in_head_stride;
            y[i] = a.out + (t0 + t) * a.out_token_stride + h * a.out_head_stride;
            p[i] = ld8<T>(x + 8 * c1[i]);
            q[i] = ld8<T>(x + 8 * c2[i]);
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (u0 + 256 * i >= units) break;
            if (pair[i] >= 0) {
                const int left = n - 8 * (ADJACENT ? c1[i] / 2 : c1[i]); /* pairs that turn: 8, or ADJACENT's last ones */
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (ADJACENT && e >= left) break;
                    v8& vb = ADJACENT && e < 4 ? p[i] : q[i];
                    v8& va = ADJACENT ? vb : p[i];
                    const int ia = ADJACENT ? 2 * e % 8 : e, ib = ADJACENT ? ia + 1 : e;
                    el b = va[ia], d = vb[ib];
                    rope_turn<T>(b, d, cs[pair[i] + e]);
                    va[ia] = b;
                    vb[ib] = d;
                }
            }
            if (ADJACENT && !a.copy && 16 * (c1[i] / 2) + 16 > 2 * n) { /* in place: what does not turn is not written */
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (8 * c1[i] + e < 2 * n) reinterpret_cast<el*>(y[i])[8 * c1[i] + e] = e < 8 ? p[i][e] : q[i][e - 8];
            } else {
                st8<T>(y[i] + 8 * c1[i], p[i]);
                if (c2[i] != c1[i]) st8<T>(y[i] + 8 * c2[i], q[i]);
            }
        }
    }
}

/* HALVES with n % 8 != 0: rows (a token's heads) through LDS, whose second operands may lie anywhere. A thread
 * has up to two chunks of 8 channels, the next rows' on their way meanwhile. */
template <class T>
__device__ __forceinline__ void rope_loose_units(const RopeArgs& a, const float2* cs, int np, int t0, int tokens) {
    typedef typename T::v8 v8;
    typedef typename T::el el;
    constexpr int U = 2;
    __shared__ __attribute__((aligned(16))) uint16_t lrow[256 * U * 8];
    const int n = a.n_pairs, chunks = a.head_dim / 8, per = 256 * U / chunks; /* rows at a time */
    const int rows = tokens * a.n_heads;
    v8 v[U];
    const auto load = [&](int r0) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int id = threadIdx.x + 256 * i, r = min(r0 + id / chunks, rows - 1); /* past the end: the last row again */
            const int t = r / a.n_heads, h = r - t * a.n_heads;
            v[i] = ld8<T>(a.in + (t0 + t) * a.in_token_stride + h * a.in_head_stride + id % chunks * 8);
        }
    };
    load(0);
    for (int r0 = 0; r0 < rows; r0 += per) {
#pragma unroll
        for (int i = 0; i < U; ++i) st8<T>(lrow + 8 * (threadIdx.x + 256 * i), v[i]);
        __syncthreads(); /* the rows are in: in place, nothing is written before they are read */
        v8 x[U];
#pragma unroll
        for (int i = 0; i < U; ++i) x[i] = v[i];
        if (r0 + per < rows) load(r0 + per);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int id = threadIdx.x + 256 * i, lr = id / chunks, r = r0 + lr, c = id % chunks * 8;
            if (lr >= per || r >= rows || (c >= 2 * n && !a.copy)) continue;
            const int t = r / a.n_heads, h = r - t * a.n_heads;
            const el* row = reinterpret_cast<const el*>(lrow) + lr * a.head_dim;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int at = c + e;
                if (at >= 2 * n) break;
                const bool second = at >= n;
                const float2 k = cs[t * np + (second ? at - n : at)];
                const float own = (float)x[i][e], other = (float)row[second ? at - n : at + n] * (second ? k.y : -k.y);
                x[i][e] = (el)opaque(__builtin_fmaf(own, k.x, other));
            }
            st8<T>(a.out + (t0 + t) * a.out_token_stride + h * a.out_head_stride + c, x[i]);
        }
        __syncthreads(); /* everyone has read the rows */
    }
}

template <class T, bool LOOSE>
__device__ __forceinline__ void rope_body(const RopeArgs& a) {
    __shared__ __attribute__((aligned(16))) float2 cs[ROPE_TILE_PAIRS]; /* [token][np] cos, sin */
    __shared__ double turns[ROPE_MAX_PAIRS];
    const int n = a.n_pairs, np = (n + 7) & ~7;
    const int t0 = blockIdx.x * a.tile, tokens = min(a.tile, a.n_tokens - t0);
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
            float s, c;
            sincospif(2.0f * (float)(rev - rint(rev)), &s, &c);
            cs[i] = float2{c, s};
        }
    }
    __syncthreads();
    if constexpr (LOOSE) rope_loose_units<T>(a, cs, np, t0, tokens);
    else if (a.adjacent) rope_units<T, true>(a, cs, np, t0, tokens);
    else rope_units<T, false>(a, cs, np, t0, tokens);
}

extern "C" __global__ void __launch_bounds__(256) prism_rope_f16(RopeArgs a) { rope_body<F16, false>(a); }
extern "C" __global__ void __launch_bounds__(256) prism_rope_bf16(RopeArgs a) { rope_body<BF16, false>(a); }
extern "C" __global__ void __launch_bounds__(256) prism_rope_f16_loose(RopeArgs a) { rope_body<F16, true>(a); }
extern "C" __global__ void __launch_bounds__(256) prism_rope_bf16_loose(RopeArgs a) { rope_body<BF16, true>(a); }
