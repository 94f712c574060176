/*
 * seq_attn.hpp - attention along (ragged) sequences with a sliding window and
 * sinks: query i of a sequence of nq queries and nk keys stands at position
 * p = nk - nq + i and sees keys j <= p + right with j >= p - left or j < sinks.
 *
 * A workgroup takes 128 queries of one head, 32 a wave, and goes once over the
 * keys that any of them sees, 64 at a time, with a running maximum and sum:
 *   S^T = K Q^T           (32x32x16 MFMA: a lane holds one query's scores)
 *   P^T = 2^(c S^T - c m) (registers; c = scale log2 e)
 *   O^T += V^T P^T        (P^T is the B operand as it lies: the MFMA's
 *                          reduction index may be numbered in any order, and
 *                          V^T is read from LDS in that order by transposing
 *                          reads)
 * so a query's maximum, sum and rescaling stay in its lane (two lanes, 32
 * apart, hold halves of its keys). K and V tiles go through LDS, double
 * buffered, the next tile's loads in flight under the current tile's products.
 * Keys that no query of the workgroup sees are staged as zeros. Where only some
 * queries see a tile's key, its weight is zero for the others; should such a
 * V be infinite or NaN (0 * inf), the workgroup does its rows again key by key.
 */
#pragma once
#include "seq_types.hpp"

typedef float f16v __attribute__((ext_vector_type(16)));

#define SEQ_BN 64  /* keys per tile */

__device__ __forceinline__ f16v mfma_32x32x16(h8 a, h8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f16v mfma_32x32x16(b8 a, b8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

/* One query by the whole wave, key after key, a lane per channel: the workgroup's
 * way out where zero weights would meet infinite values. */
template <class T, int HD>
__device__ __forceinline__ void seq_attn_row(const SeqAttnArgs& a, const uint16_t* q, const uint16_t* k, const uint16_t* v,
                                             uint16_t* out, const KeyRange kr) {
    const int lane = lane_id();
    constexpr int E = (HD + 63) / 64;
    float x[E], acc[E] = {}, m = -INFINITY, l = 0.f;
    const bool on = lane < HD;
    for (int e = 0; e < E; ++e) x[e] = on ? ld1<T>(q + lane + 64 * e) : 0.f;
    for (int i = 0; i < kr.sink + kr.hi - kr.lo; ++i) {
        const int64_t j = i < kr.sink ? i : kr.lo + i - kr.sink;
        float d = 0.f;
        for (int e = 0; e < E; ++e) d = __builtin_fmaf(x[e], on ? ld1<T>(k + j * a.k_token_stride + lane + 64 * e) : 0.f, d);
        d = wave_sum(d) * a.scale_log2;
        const float mn = fmaxf(m, d), mu = mn == -INFINITY ? 0.f : mn;
        const float f = fast_exp2(m - mu), p = fast_exp2(d - mu);
        l = __builtin_fmaf(l, f, p);
        for (int e = 0; e < E; ++e)
            acc[e] = __builtin_fmaf(p, on ? ld1<T>(v + j * a.v_token_stride + lane + 64 * e) : 0.f, acc[e] * f);
        m = mn;
    }
    for (int e = 0; e < E; ++e)
        if (on) st1<T>(out + lane + 64 * e, l == 0.f ? 0.f : acc[e] / l);
}

/* The sequence whose query tiles include tile b: sequence s owns the tiles from
 * floor(start / SEQ_BM) + s on, which leaves each enough of them whatever
 * the lengths. 64 candidates a step. */
__device__ __forceinline__ int seq_of_tile(const SeqAttnArgs& a, int b, int& first) {
    int lo = 0, n = a.n_seqs, lane = lane_id();
    first = 0;
    while (true) {
        const int step = (n + 63) / 64;
        const int s = lo + lane * step;
        bool in = false;
        int key = 0;
        if (lane * step < n) {
            key = row_range(a.cu_q, s, a.n_seqs, a.n_q).start / SEQ_BM + s;
            in = key <= b;
        }
        const unsigned long long mask = __ballot(in);
        const int at = mask ? 63 - __builtin_clzll(mask) : 0;
        lo += at * step;
        n = min(step, n - at * step);
        first = __builtin_amdgcn_readlane(key, at);
        if (step == 1) return lo;
    }
}

template <class T, int HD>
__device__ __forceinline__ void seq_attn_body(const SeqAttnArgs& a) {
    typedef typename T::v8 v8;
    constexpr int KS = HD / 16;              /* k-steps of the scores          */
    constexpr int DT = (HD + 31) / 32;       /* 32-channel tiles of the output */
    constexpr int KROW = HD + 8;             /* padded LDS rows (16-bit values): no bank conflicts for  */
    constexpr int VROW = HD + (HD >= 64 ? 32 : 0); /* 16-byte reads down rows; 8 rows of 64 bytes       */
    constexpr int CPR = HD / 8;              /* 16-byte chunks of a row        */
    constexpr int CH = (SEQ_BN * CPR + 255) / 256; /* chunks per thread        */
    __shared__ __attribute__((aligned(16))) uint16_t lk[2][SEQ_BN * KROW];
    __shared__ __attribute__((aligned(16))) uint16_t lv[2][SEQ_BN * VROW];

    /* workgroup -> (query tile, head): an XCD (workgroups b, b + 8, ...) takes a
     * run of neighbouring heads, whose keys its L2 then holds */
    const int tiles = a.n_q / SEQ_BM + a.n_seqs;
    const int total = tiles * a.n_heads, b = blockIdx.x;
    const int big = total & 7, per = total >> 3, xcd = b & 7;
    const int w = xcd * per + min(xcd, big) + (b >> 3);
    const int h = w / tiles, hk = h / (a.n_heads / a.n_kv_heads);
    const int tile = tiles - 1 - (w - h * tiles); /* the last, longest rows first */
    int first;
    const int s = __builtin_amdgcn_readfirstlane(seq_of_tile(a, tile, first));
    const RowRange rq = row_range(a.cu_q, s, a.n_seqs, a.n_q), rk = row_range(a.cu_k, s, a.n_seqs, a.n_k);
    const int nq = rq.end - rq.start, nk = rk.end - rk.start;
    if (tile < first || (int64_t)(tile - first) * SEQ_BM >= nq) return; /* uniform over the workgroup */
    const int q0 = (tile - first) * SEQ_BM, q1 = min(q0 + SEQ_BM, nq);

    const int lane = lane_id(), c32 = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int qa = q0 + 32 * wave, qb = min(qa + 32, q1); /* the wave's queries */
    const int shift = nk - nq;                            /* position - row */
    const bool on = qa < q1;

    const uint16_t* kb = a.k + rk.start * a.k_token_stride + hk * a.k_head_stride;
    const uint16_t* vb = a.v + rk.start * a.v_token_stride + hk * a.v_head_stride;
    const int qi = min(qa + c32, q1 - 1); /* this lane's query; past the end: the last one, never stored */
    const uint16_t* qp = a.q + (rq.start + qi) * a.q_token_stride + h * a.q_head_stride;

    /* keys that the workgroup's, the wave's and the lane's queries see */
    const KeyRange r0 = key_range(shift + q0, nk, a.left, a.right, a.sinks);
    const KeyRange r1 = key_range(shift + q1 - 1, nk, a.left, a.right, a.sinks);
    const KeyRange wa = key_range(shift + qa, nk, a.left, a.right, a.sinks);
    const KeyRange wb = key_range(shift + qb - 1, nk, a.left, a.right, a.sinks);
    const KeyRange me = key_range(shift + qi, nk, a.left, a.right, a.sinks);
    const int sink_end = seq_min(seq_min(a.sinks, r0.lo), r1.hi); /* sinks before the window */
    const int win0 = r0.lo, win1 = r1.hi;
    const int sink_tiles = (sink_end + SEQ_BN - 1) / SEQ_BN;
    const int n_tiles = sink_tiles + (win1 > win0 ? (win1 - win0 + SEQ_BN - 1) / SEQ_BN : 0);

    unsigned bad = 0; /* infinite or NaN V where only some of the queries look */
    v8 qf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = ld8<T>(qp + 16 * ks + 8 * g);

    f16v o[DT] = {};
    float m = -INFINITY, mc = 0.f, l = 0.f; /* mc = c m, or 0 while m is -inf */
    float limit = -INFINITY;
    const float lag = 8.0f / a.scale_log2;
    v8 sk[CH], sv[CH];

    auto key0 = [&](int it) { return it < sink_tiles ? it * SEQ_BN : win0 + (it - sink_tiles) * SEQ_BN; };
    auto end_of = [&](int it) { return it < sink_tiles ? sink_end : win1; };
    /* rows past the end lie past the buffer and read as zeros: no select that would wait for the load */
    int koff[CH], voff[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int id = (threadIdx.x + 256 * c) % (SEQ_BN * CPR), r = id / CPR, e = (id % CPR) * 8;
        koff[c] = 2 * (r * (int)a.k_token_stride + e);
        voff[c] = 2 * (r * (int)a.v_token_stride + e);
    }
    auto fetch = [&](int it) {
        const int k0 = key0(it), rows = seq_min(end_of(it) - k0, SEQ_BN);
        const auto kr = __builtin_amdgcn_make_buffer_rsrc((void*)(kb + k0 * a.k_token_stride), (short)0,
                                                          2 * ((rows - 1) * (int)a.k_token_stride + HD), 0x00020000);
        const auto vr = __builtin_amdgcn_make_buffer_rsrc((void*)(vb + k0 * a.v_token_stride), (short)0,
                                                          2 * ((rows - 1) * (int)a.v_token_stride + HD), 0x00020000);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            sk[c] = __builtin_bit_cast(v8, __builtin_amdgcn_raw_buffer_load_b128(kr, koff[c], 0, 0));
            sv[c] = __builtin_bit_cast(v8, __builtin_amdgcn_raw_buffer_load_b128(vr, voff[c], 0, 0));
        }
    };
    auto put = [&](int it, int buf) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int id = threadIdx.x + 256 * c, r = id / CPR, e = (id % CPR) * 8;
            if (SEQ_BN * CPR >= 256 || id < SEQ_BN * CPR) {
                st8<T>(lk[buf] + r * KROW + e, sk[c]);
                st8<T>(lv[buf] + r * VROW + e, sv[c]);
            }
        }
        /* seen by some queries only: are the values finite? */
        const int k0 = key0(it);
        if ((k0 < r1.lo && k0 + SEQ_BN > a.sinks) || k0 + SEQ_BN > r0.hi) {
            constexpr unsigned E = sizeof(typename T::el) == 2 && __is_same(T, F16) ? 0x7C007C00u : 0x7F807F80u;
            constexpr unsigned U = __is_same(T, F16) ? 0x04000400u : 0x00800080u;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const u4 d = __builtin_bit_cast(u4, sv[c]);
#pragma unroll
                for (int i = 0; i < 4; ++i) bad |= (d[i] & E) + U;
            }
        }
    };

    if (n_tiles > 0) {
        fetch(0);
        put(0, 0);
    }
    /* the queries are in from here on: a wait for them inside the loop would be one for the next tile too */
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = opaque(qf[ks]);
    __syncthreads();
    for (int it = 0; it < n_tiles; ++it) {
        if (it + 1 < n_tiles) fetch(it + 1);
        const int k0 = key0(it), end = end_of(it), buf = it & 1;
        /* not for a tile that none of the wave's queries sees */
        if (on && k0 < wb.hi && (k0 + SEQ_BN > wa.lo || k0 < a.sinks)) {
            /* the scores; a k-step's keys are read two steps ahead */
            const uint16_t* krow = lk[buf] + c32 * KROW + 8 * g;
            f16v sc[2] = {};
            v8 kf[3][2];
#pragma unroll
            for (int ks = 0; ks < KS + 2; ++ks) {
                if (ks < KS) {
#pragma unroll
                    for (int t = 0; t < 2; ++t) kf[ks % 3][t] = ld8<T>(krow + 32 * t * KROW + 16 * ks);
                }
                sched_fence();
                if (ks >= 2) {
#pragma unroll
                    for (int t = 0; t < 2; ++t) sc[t] = mfma_32x32x16(kf[(ks - 2) % 3][t], qf[ks - 2], sc[t]);
                }
            }
            /* V^T of 16 keys: lane's rows are keys 16 t + 4 g ..+3 and 8 more on, its columns by the 16-lane group */
            const uint16_t* vrow = lv[buf] + (4 * g + (lane & 15) / 4) * VROW + (HD >= 32 ? lane & 16 : 0) + 4 * (lane & 3);
            union VFrag {
                s4 h[2];
                v8 v;
            };
            VFrag vf[2][DT];
            auto read_v = [&](int t) {
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    vf[t & 1][d].h[0] = lds_tr4(vrow + 16 * t * VROW + 32 * d);
                    vf[t & 1][d].h[1] = lds_tr4(vrow + (16 * t + 8) * VROW + 32 * d);
                }
            };
            read_v(0);
            const bool whole = k0 + SEQ_BN <= seq_min(wa.hi, end) && (k0 >= wb.lo || k0 + SEQ_BN <= a.sinks);
            if (!whole) {
                const int hi = seq_min(me.hi, end);
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int j = k0 + 32 * t + 8 * (i / 4) + 4 * g + (i & 3);
                        sc[t][i] = j < hi && (j >= me.lo || j < a.sinks) ? sc[t][i] : -INFINITY;
                    }
            }
            float top = sc[0][0];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; i += 2) top = vmax3(top, sc[t][i], sc[t][i + 1]);
            float x, y;
            lanes_x32(top, x, y);
            top = vmax(x, y);
            /* the maximum may lag by 8 powers of two: weights up to 256 cost no precision, rescaling costs much */
            if (__any(top > limit)) {
                top = vmax(top, m);
                const float tc = top == -INFINITY ? 0.f : top * a.scale_log2;
                const float f = fast_exp2(m == -INFINITY ? -INFINITY : mc - tc);
                l *= f;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[d][i] *= f;
                m = top;
                mc = tc;
                limit = top + lag;
            }
            /* 16 keys at a time: the next ones' V is read and their weights computed under the products */
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                if (t < 3) read_v(t + 1);
                v8 p;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float e = fast_exp2(__builtin_fmaf(sc[t / 2][8 * (t & 1) + i], a.scale_log2, -mc));
                    l += e;
                    p[i] = (typename T::el)e;
                }
                sched_fence();
#pragma unroll
                for (int d = 0; d < DT; ++d) o[d] = mfma_32x32x16(vf[t & 1][d].v, p, o[d]);
            }
        }
        if (it + 1 < n_tiles) put(it + 1, buf ^ 1);
        __syncthreads();
    }

    if (__syncthreads_or((bad & 0x80008000u) != 0)) {
        for (int i = qa; i < qb; ++i)
            seq_attn_row<T, HD>(a, a.q + (rq.start + i) * a.q_token_stride + h * a.q_head_stride, kb, vb,
                                a.out + (rq.start + i) * a.out_token_stride + h * a.out_head_stride,
                                key_range(shift + i, nk, a.left, a.right, a.sinks));
        return;
    }
    float x, y;
    lanes_x32(l, x, y);
    l = x + y;
    if (!on || qa + c32 >= qb) return;
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    uint16_t* out = a.out + (rq.start + qi) * a.out_token_stride + h * a.out_head_stride;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int ch = 32 * d + 2 * i + 4 * g;
            if (HD >= 32 || ch < HD) {
                typename T::v4 r;
#pragma unroll
                for (int e = 0; e < 4; ++e) r[e] = (typename T::el)opaque(o[d][i + e] * inv);
                *reinterpret_cast<typename T::v4*>(out + ch) = r;
            }
        }
}

#define SEQ_ATTN(NAME, T, HD) \
    extern "C" __global__ void __launch_bounds__(256, 2) prism_seq_attn_##NAME##_h##HD(SeqAttnArgs a) { seq_attn_body<T, HD>(a); }
SEQ_ATTN(f16, F16, 16) SEQ_ATTN(f16, F16, 32) SEQ_ATTN(f16, F16, 64) SEQ_ATTN(f16, F16, 128)
SEQ_ATTN(bf16, BF16, 16) SEQ_ATTN(bf16, BF16, 32) SEQ_ATTN(bf16, BF16, 64) SEQ_ATTN(bf16, BF16, 128)
#undef SEQ_ATTN
