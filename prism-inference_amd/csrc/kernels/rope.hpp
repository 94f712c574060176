/*
 * rope.hpp - rotary positions with several axes.
 *
 * Pair i of a head's channels (a, b) turns by phi = pos[axis(i)] * f_i:
 *   a' = a cos phi - b sin phi,  b' = b cos phi + a sin phi
 * The frequencies come from the host in turns (f_i / 2 pi, 64 bits; negated for
 * the inverse). phi is reduced to (-1/2, 1/2] turns in 64 bits, so a position
 * of millions keeps its angle to 1e-9 turns, and sin / cos are taken in fp32.
 */
#pragma once
#include "seq_types.hpp"

template <class T>
__device__ __forceinline__ void rope_body(const RopeArgs& a) {
    /* one thread a (token, head): the simple form */
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= (int64_t)a.n_tokens * a.n_heads) return;
    const int t = (int)(id / a.n_heads), h = (int)(id % a.n_heads);
    const uint16_t* x = a.in + t * a.in_token_stride + h * a.in_head_stride;
    uint16_t* y = a.out + t * a.out_token_stride + h * a.out_head_stride;
    int axis = 0;
    for (int i = 0; i < a.n_pairs; ++i) {
        while (i >= a.axis_end[axis]) ++axis;
        const double rev = (double)a.pos[axis * a.pos_stride + t] * a.turns[i];
        float s, c;
        sincospif(2.0f * (float)(rev - rint(rev)), &s, &c);
        const int ia = a.adjacent ? 2 * i : i, ib = a.adjacent ? 2 * i + 1 : i + a.n_pairs;
        const float u = ld1<T>(x + ia), w = ld1<T>(x + ib);
        st1<T>(y + ia, u * c - w * s);
        st1<T>(y + ib, w * c + u * s);
    }
    for (int i = 2 * a.n_pairs; i < a.head_dim; ++i) y[i] = x[i];
}

extern "C" __global__ void __launch_bounds__(256) prism_rope_f16(RopeArgs a) { rope_body<F16>(a); }
extern "C" __global__ void __launch_bounds__(256) prism_rope_bf16(RopeArgs a) { rope_body<BF16>(a); }
