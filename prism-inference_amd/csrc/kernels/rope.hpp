/*
 * rope.hpp - rotary positions with several axes.
 *
 * Pair i of a head's channels (a, b) turns by phi = pos[axis(i)] * f_i:
 *   a' = a cos phi - b sin phi,  b' = b cos phi + a sin phi
 * The frequencies come from the host in turns (f_i / 2 pi, 64 bits; negated for
 * the inverse). phi is reduced to [-1/2, 1/2] turns in 64 bits, so a position
 * of millions keeps its angle, and sin / cos are taken in fp32.
 *
 * All heads of a token turn by the same angles, and an angle (64-bit product,
 * reduction, sincos: ~80 instructions) costs far more than a turn, so a
 * workgroup takes a few tokens, puts their angles' cos and sin into LDS, and
 * then streams the tokens' rows: a unit is 8 pairs of one head, 16 bytes per
 * operand. Where n is not a multiple of 8 the second operand of a HALVES unit
 * is a 16-byte access on a 2-byte boundary (global memory takes any), and
 * the last unit goes element by element. Bound by HBM traffic: x read and
 * written once.
 */
#pragma once
#include "seq_types.hpp"

/* 16 bytes on any 2-byte boundary */
template <class T>
struct Loose8 {
    typename T::v8 v;
} __attribute__((packed, aligned(2)));

/* (u, w) turned by (cos, sin) cs */
template <class T>
__device__ __forceinline__ void rope_turn(typename T::el& u, typename T::el& w, float2 cs) {
    const float a = (float)u, b = (float)w;
    u = (typename T::el)opaque(__builtin_fmaf(a, cs.x, -(b * cs.y)));
    w = (typename T::el)opaque(__builtin_fmaf(b, cs.x, a * cs.y));
}

template <class T>
__device__ __forceinline__ void rope_body(const RopeArgs& a) {
    typedef typename T::v8 v8;
    typedef typename T::el el;
    __shared__ __attribute__((aligned(16))) float2 cs[ROPE_TILE_PAIRS]; /* [token][np] cos, sin */
    const int n = a.n_pairs, np = (n + 7) & ~7;
    const int t0 = blockIdx.x * a.tile, tokens = min(a.tile, a.n_tokens - t0);
    for (int i = threadIdx.x; i < tokens * np; i += 256) {
        const int t = i / np, j = i - t * np;
        if (j < n) {
            const int axis = (j >= a.axis_end[0]) + (j >= a.axis_end[1]) + (j >= a.axis_end[2]);
            const double rev = (double)a.pos[axis * a.pos_stride + t0 + t] * a.turns[j];
            float s, c;
            sincospif(2.0f * (float)(rev - rint(rev)), &s, &c);
            cs[i] = float2{c, s};
        }
    }
    __syncthreads();

    /* a head's units: turned pairs, then chunks of channels to copy */
    const int turned = a.adjacent ? (2 * n + 7) / 8 : np / 8;
    const int copy0 = a.adjacent ? turned : 2 * n / 8;
    const int per_head = turned + (a.copy ? a.head_dim / 8 - copy0 : 0);
    const int per_token = per_head * a.n_heads;
    for (int u = threadIdx.x; u < tokens * per_token; u += 256) {
        const int t = u / per_token, r = u - t * per_token, h = r / per_head, k = r - h * per_head;
        const uint16_t* x = a.in + (t0 + t) * a.in_token_stride + h * a.in_head_stride;
        uint16_t* y = a.out + (t0 + t) * a.out_token_stride + h * a.out_head_stride;
        const float2* row = cs + t * np;
        if (k >= turned) {
            const int c = 8 * (copy0 + k - turned);
            if (c >= 2 * n) {
                st8<T>(y + c, ld8<T>(x + c));
            } else {
                for (int e = 2 * n; e < c + 8; ++e) y[e] = x[e];
            }
        } else if (a.adjacent) {
            v8 v = ld8<T>(x + 8 * k);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (4 * k + e < n) {
                    el p = v[2 * e], q = v[2 * e + 1];
                    rope_turn<T>(p, q, row[4 * k + e]);
                    v[2 * e] = p;
                    v[2 * e + 1] = q;
                }
            }
            if (8 * k + 8 <= 2 * n || a.copy) { /* in place, the unturned end of a mixed chunk is not written */
                st8<T>(y + 8 * k, v);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (8 * k + e < 2 * n) reinterpret_cast<el*>(y)[8 * k + e] = v[e];
            }
        } else if (8 * k + 8 <= n) {
            v8 p = ld8<T>(x + 8 * k), q = reinterpret_cast<const Loose8<T>*>(x + 8 * k + n)->v;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                el b = p[e], d = q[e];
                rope_turn<T>(b, d, row[8 * k + e]);
                p[e] = b;
                q[e] = d;
            }
            st8<T>(y + 8 * k, p);
            reinterpret_cast<Loose8<T>*>(y + 8 * k + n)->v = q;
        } else {
            for (int i = 8 * k; i < n; ++i) {
                el b = reinterpret_cast<const el*>(x)[i], d = reinterpret_cast<const el*>(x)[i + n];
                rope_turn<T>(b, d, row[i]);
                reinterpret_cast<el*>(y)[i] = b;
                reinterpret_cast<el*>(y)[i + n] = d;
            }
        }
    }
}

extern "C" __global__ void __launch_bounds__(256) prism_rope_f16(RopeArgs a) { rope_body<F16>(a); }
extern "C" __global__ void __launch_bounds__(256) prism_rope_bf16(RopeArgs a) { rope_body<BF16>(a); }
