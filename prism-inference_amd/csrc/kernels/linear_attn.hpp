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
/* decays are e^-rate; rates below 0 and NaN count as 0 */
__device__ __forceinline__ float linear_rate(const LinearAttnArgs& a, int h) {
    return fminf(fmaxf(a.rates[h], 0.f) * 1.4426950408889634f, 1e30f); /* as powers of two; finite: 0 times it is 0 */
}

/* the sequence of segment b: its first segment's number, its rows. Sequence s has those from start / segment + s on, one at
 * least, so the number follows from the starts alone. The wave looks at 64 sequences at a time. */
struct LinearTile {
    int seq, first;
    RowRange rows;
};
__device__ __forceinline__ LinearTile linear_tile(const LinearAttnArgs& a, int b) {
    int lo = 0, n = a.n_seqs;
    const int lane = lane_id();
    while (true) {
        const int step = (n + 63) / 64;
        const int s = lo + min(lane, (n - 1) / step) * step; /* lanes past the end: the last one again */
        const RowRange r = row_range(a.cu, s, a.n_seqs, a.n_tokens);
        const int key = r.start / a.segment + s;
        const unsigned long long mask = __ballot(key <= b);
        const int at = mask ? min(63 - __builtin_clzll(mask), (n - 1) / step) : 0;
        if (step == 1) {
            const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, at); };
            return LinearTile{lo + at, of(key), RowRange{of(r.start), of(r.end)}};
        }
        lo += at * step;
        n = min(step, n - at * step);
    }
}

/* Two fp32 numbers as N pairs of 16-bit ones that add up to them: fp16 11 N bits (of what is above its smallest), bf16 8 N. */
template <class T, int N>
__device__ __forceinline__ void parts(float x, float y, typename T::v2 (&p)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        x = opaque(x);
        y = opaque(y);
        p[i] = typename T::v2{(typename T::el)x, (typename T::el)y};
        if (i + 1 < N) {
            x -= (float)p[i][0];
            y -= (float)p[i][1];
        }
    }
}
/* 2^k that brings the largest magnitude m (of fp16 parts' numbers) to 2^13 .. 2^14; 1 for 0; k from -120 to 60 */
__device__ __forceinline__ float part_scale(float m) {
    const int e = (int)(__builtin_bit_cast(unsigned, m) >> 23); /* m >= 0 */
    return m == 0.f ? 1.f : __builtin_bit_cast(float, (unsigned)seq_clamp(267 - e, 7, 187) << 23);
}
__device__ __forceinline__ float part_unscale(float scale) { /* of a power of two: 1 / scale */
    return __builtin_bit_cast(float, 0x7F000000u - __builtin_bit_cast(unsigned, scale));
}

/* One segment of one head: its chunks in turn, the state in registers. STATES: only the state that the segment adds. */
template <class T, int HD, bool STATES>
__device__ __forceinline__ void linear_segment(const LinearAttnArgs& a) {
    typedef typename T::v8 v8;
    typedef typename T::v4 v4;
    typedef typename T::v2 v2;
    typedef typename T::el el;
    constexpr bool HALF = __is_same(T, F16);
    constexpr int C = LINEAR_CHUNK, QT = C / 16, M = C / 32;
    constexpr int NW = HD >= 64 ? HD / 32 : 1, NT = 64 * NW; /* waves, threads */
    constexpr int DV = HD >= 32 ? 2 : 1, DK = HD / 16;       /* 16-channel tiles of a wave's values, of keys */
    constexpr int KS = (HD + 31) / 32;
    constexpr int RS = HD >= 32 ? HD + 16 : HD; /* LDS row */
    constexpr int CPR = HD / 8, NL = C * CPR / NT; /* 16-byte chunks a row, and a thread's of a matrix */
    constexpr int VP = HALF ? 2 : 3;               /* parts of a decayed value */
    __shared__ __attribute__((aligned(16))) uint16_t lq[STATES ? 8 : C * RS], lk[C * RS], lv[C * RS];
    __shared__ int lbad[2];
    const int lane = lane_id(), l16 = lane & 15, g = lane >> 4, tid = threadIdx.x;
    const int wave = NW == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6);
    const int b = blockIdx.x / a.n_heads, h = blockIdx.x % a.n_heads, hk = h / (a.n_heads / a.n_kv_heads);
    const LinearTile lt = linear_tile(a, b);
    const int seg = b - lt.first;
    if (seg < 0) return; /* only where starts are not in order */
    const int64_t t0 = lt.rows.start + (int64_t)seg * a.segment;
    if (STATES ? t0 + a.segment >= lt.rows.end : seg > 0 && t0 >= lt.rows.end) return;
    const int t1 = (int)min(t0 + a.segment, (int64_t)lt.rows.end);

    const float r2 = linear_rate(a, h);
    const auto decay = [&](int n) { return fast_exp2(-r2 * (float)n); };
    const int number = linear_state(a, lt.seq);
    const int64_t base = ((int64_t)max(number, 0) * a.n_heads + h) * HD * HD + 32 * wave + l16;
    f4* const mine = reinterpret_cast<f4*>(a.ws) + ((int64_t)b * a.n_heads + h) * (HD * HD / 4) + tid; /* + NT * tile */
    f4 S[DK][DV];
    /* the state before the segment */
#pragma unroll
    for (int j = 0; j < DK; ++j)
#pragma unroll
        for (int d = 0; d < DV; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                S[j][d][e] = !STATES && a.state_in && number >= 0 ? a.state_in[base + (16 * j + 4 * g + e) * HD + 16 * d] : 0.f;
    if constexpr (!STATES) {
        const float keep = decay(a.segment);
        for (int s = seg; s > 0; --s) {
            const f4* u = mine - (int64_t)s * a.n_heads * (HD * HD / 4);
#pragma unroll
            for (int j = 0; j < DK; ++j)
#pragma unroll
                for (int d = 0; d < DV; ++d) S[j][d] = S[j][d] * keep + u[NT * (j * DV + d)];
        }
    }
    /* decays: of a key within a query's tile and in the tile before it, of a token up to the chunk's end */
    float within[4], before[4], fade[M][8];
    const float d16 = decay(16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int gap = l16 - 4 * g - e;
        within[e] = gap >= 0 ? decay(max(gap, 0)) * a.scale : 0.f;
        before[e] = decay(16 + gap) * a.scale;
    }

    v8 rq[STATES ? 1 : NL], rk[NL], rv[NL];
    const uint16_t* qb = a.q + h * a.q_head_stride;
    const uint16_t* kb = a.k + hk * a.k_head_stride;
    const uint16_t* vb = a.v + hk * a.v_head_stride;
    const auto load = [&](int64_t c0, int n) {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int id = tid + NT * i, row = id / CPR, c = id % CPR * 8;
            const int64_t t = c0 + min(row, n - 1);
            if constexpr (!STATES) rq[i] = ld8<T>(qb + t * a.q_token_stride + c);
            rk[i] = ld8<T>(kb + t * a.k_token_stride + c);
            rv[i] = ld8<T>(vb + t * a.v_token_stride + c);
            if (row >= n) rk[i] = rv[i] = v8{}; /* behind the segment: no key */
        }
    };
    /* where channel c lies in a row of lq and lk: those that a lane takes of 32 side by side */
    const auto spot = [](int c) { return HD < 32 ? c : (c & ~31) + (c % 16 / 4) * 8 + (c % 32 / 16) * 4 + c % 4; };
    if (t0 < t1) load(t0, min(C, t1 - (int)t0));
    int full = -1; /* the length that fade is for */
    for (int64_t c0 = t0; c0 < t1; c0 += C) {
        const int n = min(C, t1 - (int)c0);
        const int turn = (int)((c0 - t0) / C & 1);
        bool bad = false;
        __syncthreads(); /* the chunk before has been read */
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int id = tid + NT * i, row = id / CPR, c = id % CPR * 8;
            if constexpr (!STATES) {
                *reinterpret_cast<v4*>(lq + row * RS + spot(c)) = v4{rq[i][0], rq[i][1], rq[i][2], rq[i][3]};
                *reinterpret_cast<v4*>(lq + row * RS + spot(c + 4)) = v4{rq[i][4], rq[i][5], rq[i][6], rq[i][7]};
#pragma unroll
                for (int e = 0; e < 8; ++e) bad |= !(__builtin_fabsf((float)rv[i][e]) < INFINITY);
            }
            *reinterpret_cast<v4*>(lk + row * RS + spot(c)) = v4{rk[i][0], rk[i][1], rk[i][2], rk[i][3]};
            *reinterpret_cast<v4*>(lk + row * RS + spot(c + 4)) = v4{rk[i][4], rk[i][5], rk[i][6], rk[i][7]};
            st8<T>(lv + row * RS + c, rv[i]);
        }
        if (tid == 0) lbad[turn ^ 1] = 0; /* for the next chunk */
        if (c0 == t0 && tid == 0) lbad[0] = 0;
        if (c0 == t0) __syncthreads();
        if (bad) lbad[turn] = 1;
        __syncthreads();
        if (c0 + C < t1) load(c0 + C, min(C, t1 - (int)c0 - C));

        /* the wave's values, transposed: lane l16 is a channel, with 8 tokens of each 32 */
        v8 v[DV][M];
#pragma unroll
        for (int d = 0; d < DV; ++d)
#pragma unroll
            for (int m = 0; m < M; ++m) {
                const uint16_t* at = lv + (32 * m + 4 * g + l16 / 4) * RS + 32 * wave + 16 * d + 4 * (l16 & 3);
                union {
                    s4 h[2];
                    v8 v;
                } f;
                f.h[0] = lds_tr4(at);
                f.h[1] = lds_tr4(at + 16 * RS);
                v[d][m] = f.v;
            }
        if constexpr (!STATES) {
            const bool poisoned = __builtin_amdgcn_readfirstlane(lbad[turn]) != 0;
            v8 clean[DV][M];
#pragma unroll
            for (int d = 0; d < DV; ++d)
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    clean[d][m] = v[d][m];
                    if (poisoned)
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            clean[d][m][e] = __builtin_fabsf((float)v[d][m][e]) < INFINITY ? v[d][m][e] : (el)0.f;
                }
            /* the state in 16-bit parts: lane l16 is a channel of the values, with 8 of each 32 channels of the keys */
            v8 sh[KS][DV], sl[KS][DV];
            float back[DV][4]; /* fp16: what takes the scales out of the output's rows 4 g + e */
#pragma unroll
            for (int d = 0; d < DV; ++d) {
                float up = 1.f;
                if constexpr (HALF) {
                    float most = 0.f;
#pragma unroll
                    for (int j = 0; j < DK; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) most = fmaxf(most, __builtin_fabsf(S[j][d][e]));
                    float x, y;
                    lanes_x16(most, x, y);
                    lanes_x32(fmaxf(x, y), x, y);
                    up = part_scale(fmaxf(x, y));
                    const float down = part_unscale(up);
#pragma unroll
                    for (int e = 0; e < 4; ++e) back[d][e] = __shfl(down, 4 * g + e);
                }
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        v2 p[2] = {};
                        const int j = 2 * ks + e / 4;
                        if (j < DK) parts<T, 2>(S[j < DK ? j : 0][d][e % 4] * up, S[j < DK ? j : 0][d][e % 4 + 1] * up, p);
                        sh[ks][d][e] = p[0][0];
                        sh[ks][d][e + 1] = p[0][1];
                        sl[ks][d][e] = p[1][0];
                        sl[ks][d][e + 1] = p[1][1];
                    }
            }
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
                v8 q[KS];
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    if constexpr (HD >= 32) {
                        q[ks] = ld8<T>(lq + (16 * qt + l16) * RS + 32 * ks + 8 * g);
                    } else {
                        const v4 x = *reinterpret_cast<const v4*>(lq + (16 * qt + l16) * RS + 4 * g);
                        q[ks] = v8{x[0], x[1], x[2], x[3], (el)0.f, (el)0.f, (el)0.f, (el)0.f};
                    }
                }
                f4 o[DV] = {};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int d = 0; d < DV; ++d) {
                        o[d] = mfma_16x16x32(sh[ks][d], q[ks], o[d]);
                        o[d] = mfma_16x16x32(sl[ks][d], q[ks], o[d]);
                    }
                /* weights of the chunk's keys: lane l16 is a query, with keys 4 g + e of each 16 */
                f4 w[QT] = {};
                float most = 0.f;
#pragma unroll
                for (int kt = 0; kt <= qt; ++kt) {
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        v8 k;
                        if constexpr (HD >= 32) {
                            k = ld8<T>(lk + (16 * kt + l16) * RS + 32 * ks + 8 * g);
                        } else {
                            const v4 x = *reinterpret_cast<const v4*>(lk + (16 * kt + l16) * RS + 4 * g);
                            k = v8{x[0], x[1], x[2], x[3], (el)0.f, (el)0.f, (el)0.f, (el)0.f};
                        }
                        w[kt] = mfma_16x16x32(k, q[ks], w[kt]);
                    }
                    float far = 1.f;
                    for (int x = kt + 1; x < qt; ++x) far *= d16;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (kt == qt) w[kt][e] = l16 >= 4 * g + e ? w[kt][e] * within[e] : 0.f;
                        else w[kt][e] *= before[e] * far;
                        if (HALF) most = fmaxf(most, __builtin_fabsf(w[kt][e]));
                    }
                }
                const float since = decay(16 * qt + l16 + 1) * a.scale;
                float up = 1.f;
                if constexpr (HALF) {
                    float x, y;
                    lanes_x16(most, x, y);
                    lanes_x32(fmaxf(x, y), x, y);
                    up = part_scale(fmaxf(x, y));
                }
#pragma unroll
                for (int d = 0; d < DV; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[d][e] = HALF ? o[d][e] * back[d][e] * since * up : o[d][e] * since;
#pragma unroll
                for (int m = 0; 2 * m <= qt; ++m) {
                    v8 hi, lo;
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        v2 p[2];
                        const f4 x = w[2 * m + e / 4];
                        parts<T, 2>(HALF ? x[e % 4] * up : x[e % 4], HALF ? x[e % 4 + 1] * up : x[e % 4 + 1], p);
                        hi[e] = p[0][0];
                        hi[e + 1] = p[0][1];
                        lo[e] = p[1][0];
                        lo[e + 1] = p[1][1];
                    }
#pragma unroll
                    for (int d = 0; d < DV; ++d) {
                        o[d] = mfma_16x16x32(clean[d][m], hi, o[d]);
                        o[d] = mfma_16x16x32(clean[d][m], lo, o[d]);
                    }
                }
                const float down = HALF ? part_unscale(up) : 1.f;
                const int i = 16 * qt + l16;
                if (poisoned) /* queries from a value on that is not finite */
                    for (int d = 0; d < DV; ++d)
                        for (int e = 0; e < 4; ++e)
                            for (int t = 0; t <= i; ++t)
                                if (!(__builtin_fabsf(ld1<T>(lv + t * RS + 32 * wave + 16 * d + 4 * g + e)) < INFINITY))
                                    o[d][e] = __builtin_nanf("");
                if (i < n) {
                    uint16_t* out = a.out + (c0 + i) * a.out_token_stride + h * a.out_head_stride + 32 * wave + 4 * g;
#pragma unroll
                    for (int d = 0; d < DV; ++d) {
                        v4 r;
#pragma unroll
                        for (int e = 0; e < 4; ++e) r[e] = (el)opaque(HALF ? o[d][e] * down : o[d][e]);
                        *reinterpret_cast<v4*>(out + 16 * d) = r;
                    }
                }
            }
        }
        /* the next state */
        if (n != full) {
            full = n;
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int e = 0; e < 8; ++e) fade[m][e] = decay(max(n - 1 - (32 * m + e / 4 * 16 + 4 * g + e % 4), 0));
        }
        const float keep = decay(n);
        v8 vp[DV][M][VP];
        float down[DV];
#pragma unroll
        for (int d = 0; d < DV; ++d) {
            float up = 1.f;
            if constexpr (HALF) {
                float most = 0.f;
#pragma unroll
                for (int m = 0; m < M; ++m)
#pragma unroll
                    for (int e = 0; e < 8; ++e) most = fmaxf(most, __builtin_fabsf((float)v[d][m][e] * fade[m][e]));
                float x, y;
                lanes_x16(most, x, y);
                lanes_x32(fmaxf(x, y), x, y);
                up = part_scale(fmaxf(x, y));
                down[d] = part_unscale(up);
            }
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    v2 p[VP];
                    const float x = (float)v[d][m][e] * fade[m][e], y = (float)v[d][m][e + 1] * fade[m][e + 1];
                    parts<T, VP>(HALF ? x * up : x, HALF ? y * up : y, p);
#pragma unroll
                    for (int i = 0; i < VP; ++i) {
                        vp[d][m][i][e] = p[i][0];
                        vp[d][m][i][e + 1] = p[i][1];
                    }
                }
        }
#pragma unroll
        for (int j = 0; j < DK; ++j) {
            v8 k[M];
#pragma unroll
            for (int m = 0; m < M; ++m) {
                const uint16_t* at = lk + (32 * m + 4 * g + l16 / 4) * RS + spot(16 * j + 4 * (l16 & 3));
                union {
                    s4 h[2];
                    v8 v;
                } f;
                f.h[0] = lds_tr4(at);
                f.h[1] = lds_tr4(at + 16 * RS);
                k[m] = f.v;
            }
#pragma unroll
            for (int d = 0; d < DV; ++d) {
                f4 u = HALF ? f4{} : S[j][d] * keep;
#pragma unroll
                for (int m = 0; m < M; ++m)
#pragma unroll
                    for (int i = 0; i < VP; ++i) u = mfma_16x16x32(k[m], vp[d][m][i], u);
                if constexpr (HALF) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) S[j][d][e] = __builtin_fmaf(u[e], down[d], S[j][d][e] * keep);
                } else {
                    S[j][d] = u;
                }
            }
        }
    }
    if constexpr (STATES) {
#pragma unroll
        for (int j = 0; j < DK; ++j)
#pragma unroll
            for (int d = 0; d < DV; ++d) mine[NT * (j * DV + d)] = S[j][d];
    } else if (number >= 0 && a.state_out && t1 == lt.rows.end) {
#pragma unroll
        for (int j = 0; j < DK; ++j)
#pragma unroll
            for (int d = 0; d < DV; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) a.state_out[base + (16 * j + 4 * g + e) * HD + 16 * d] = S[j][d][e];
    }
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
    extern "C" __global__ void __launch_bounds__(HD >= 64 ? 2 * HD : 64) prism_linear_attn_##NAME##_h##HD(LinearAttnArgs a) { linear_segment<T, HD, false>(a); } \
    extern "C" __global__ void __launch_bounds__(HD >= 64 ? 2 * HD : 64) prism_linear_states_##NAME##_h##HD(LinearAttnArgs a) { linear_segment<T, HD, true>(a); } \
    extern "C" __global__ void __launch_bounds__(256) prism_linear_step_##NAME##_h##HD(LinearAttnArgs a) { linear_step<T, HD>(a); }
LINEAR(f16, F16, 16) LINEAR(f16, F16, 32) LINEAR(f16, F16, 64) LINEAR(f16, F16, 128)
LINEAR(bf16, BF16, 16) LINEAR(bf16, BF16, 32) LINEAR(bf16, BF16, 64) LINEAR(bf16, BF16, 128)
#undef LINEAR
