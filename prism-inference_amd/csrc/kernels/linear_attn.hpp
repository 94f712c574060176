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

/* Two fp32 numbers as N pairs of bf16 numbers that add up to them, to 2^-9N (rounded to nearest, so that what is left has a sign and half a bit
 * more). bf16's exponents are fp32's: the bits do not depend on what else is in a product. */
template <int N>
__device__ __forceinline__ void parts(float x, float y, uint32_t (&p)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const b2 v = __builtin_convertvector((f2{x, y}), b2);
        p[i] = __builtin_bit_cast(uint32_t, v);
        if (i + 1 < N) {
            x -= (float)v[0];
            y -= (float)v[1];
        }
    }
}
/* 8 values as numbers of bf16 that add up to them, exactly: fp16's 11 bits are two. Products of two inputs take fp16 as it is; weights,
 * states and decayed values, which differ by more than fp16's powers of two beside each other, meet them in bf16. The product of both second
 * numbers, 2^-18 of a term at most, is not taken where the other factor has two numbers, which hold it to 2^-18. */
__device__ __forceinline__ void numbers(b8 v, b8 (&n)[1]) { n[0] = v; }
__device__ __forceinline__ void numbers(h8 v, b8 (&n)[2]) {
    u4 w[2];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        uint32_t p[2];
        parts<2>((float)v[2 * e], (float)v[2 * e + 1], p);
        w[0][e] = p[0];
        w[1][e] = p[1];
    }
    n[0] = __builtin_bit_cast(b8, w[0]);
    n[1] = __builtin_bit_cast(b8, w[1]);
}
/* The larger of each half of two words of 16-bit values, as whole numbers. */
typedef unsigned short us2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t most2(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2, a), __builtin_bit_cast(us2, b)));
}
/* The largest magnitude of 8 values, its bits; 2 words side by side */
template <class V>
__device__ __forceinline__ uint32_t most8(V v) {
    const u4 w = __builtin_bit_cast(u4, v) & 0x7FFF7FFFu;
    return most2(most2(w[0], w[1]), most2(w[2], w[3]));
}
template <class T>
__device__ __forceinline__ bool infinite(uint32_t most) { /* bits of magnitudes, two of them */
    constexpr uint32_t inf = __is_same(T, F16) ? 0x7C00 : 0x7F80;
    return (most & 0xFFFF) >= inf || most >> 16 >= inf;
}

/* What bounds it. Few short sequences: a chain of launch, starts, tokens and products; 9 up to 130, 8 x 16, 8 us. 8,160 tokens,
 * 8 x 32, fp16: 19 us behind 6 for the segments' states, of which each chunk is 1 and the rest latency. 23,000 tokens of 5 sequences, 32 x 128,
 * bf16: 212 us behind 88 (805 MB: 3.8 TB/s); matrix cores 30 %, vector units 39 % busy. Without any product the kernel still takes 0.8 of
 * that: loads, staging in LDS, barriers and stores, with two workgroups a CU (256 registers, 67 KB of LDS).
 * fp16's second numbers are products 3 for 2 and 5 for 3, and made anew by each wave from what it reads: 5 x 4,500, 32 x 128 415 us for bf16's 285.
 * In fp16 with a power of two for each chunk, row of the state or channel it took 297, but numbers far below the largest lost their bits. fp16
 * keys split once, into LDS, took 409 (of 32 channels 104 for 109) for a barrier more.
 *
 * One segment of one head: its chunks of 64 tokens in turn,
 *   o_i = scale (e^(-r (i+1)) q_i S + sum_{j <= i} e^(-r (i-j)) (q_i k_j) v_j),  S' = e^(-r n) S + sum_j k_j^T e^(-r (n-1-j)) v_j
 * A wave has 16 channels of the values, so its part of the state is its own and stays in registers: 16 x 16 tiles as the
 * product leaves them, which are at the same time what the next chunk's product q S takes.
 * From 64 channels on a wave has all queries (WQ = 1) and the weights (q_i k_j) are all waves' work and go through LDS.
 * Below, where that is few waves, each has one or two of the four query tiles with weights of its own, and the
 * state's update is done again by the waves of other tiles. STATES: only the state that the segment adds. */
template <class T, int HD, bool STATES>
__device__ __forceinline__ void linear_segment(const LinearAttnArgs& a) {
    typedef typename T::v8 v8;
    typedef typename T::v4 v4;
    typedef typename T::el el;
    constexpr int IN = __is_same(T, F16) ? 2 : 1; /* numbers of bf16 that an input is */
    constexpr int C = LINEAR_CHUNK, QT = C / 16, M = C / 32;
    constexpr int DV = HD >= 128 ? 2 : 1;          /* a wave's 16-channel tiles of the values */
    constexpr int WD = HD / 16 / DV, WQ = STATES || HD >= 64 ? 1 : QT / WD, QN = QT / WQ; /* waves by channels, by query tiles; a wave's */
    constexpr bool SHARED = WQ == 1;
    constexpr int NT = 64 * WD * WQ;
    constexpr int DK = HD / 16; /* 16-channel tiles of the keys */
    /* of row or column r of a wave's tile d: a lane's 4 outputs of two tiles lie side by side, 16 bytes a store */
    const auto channel = [](int d, int r) { return 4 * DV * (r / 4) + 4 * d + r % 4; };
    constexpr int KS = (HD + 31) / 32;
    constexpr int RS = HD >= 32 ? HD + 16 : HD;    /* LDS row: 4 rows' parts of a transposed read lie in different banks */
    constexpr int CPR = HD / 8, NL = (C * CPR + NT - 1) / NT; /* 16-byte chunks a row, and a thread's of a matrix */
    constexpr int TILES = QT * (QT + 1) / 2;       /* of weights */
    __shared__ __attribute__((aligned(16))) uint16_t lq[STATES ? 8 : C * RS], lk[C * RS], lv[C * RS];
    __shared__ __attribute__((aligned(16))) uint16_t lw[!STATES && SHARED ? 6 * 2 * 64 * 8 : 8]; /* weights [query tile, 32 keys][part] */
    __shared__ uint32_t lbad[2][WD * WQ]; /* of a chunk, by waves: a value that is not finite */
    const int lane = lane_id(), l16 = lane & 15, g = lane >> 4, tid = threadIdx.x;
    const int wave = NT == 64 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6), wd = wave % WD, wq = wave / WD;
    const int b = blockIdx.x / a.n_heads, h = blockIdx.x % a.n_heads, hk = h / (a.n_heads / a.n_kv_heads);
    const LinearTile lt = linear_tile(a, b);
    const int seg = b - lt.first;
    if (seg < 0) return; /* only where starts are not in order */
    const int64_t t0 = lt.rows.start + (int64_t)seg * a.segment;
    const bool last = t0 + a.segment >= lt.rows.end;
    if (STATES ? last && (seg == 0 || t0 >= lt.rows.end) : seg > 0 && t0 >= lt.rows.end) return;
    const int t1 = (int)min(t0 + a.segment, (int64_t)lt.rows.end);

    /* The first chunk is asked for before anything else is waited for. A chunk's tokens lie at its end: a short one, the segment's last, has rows of zeros before them, so that decays up to
       the end are always the same. Token strides are at most 2^22: 32-bit offsets from a base that is the same for all. */
    v8 rq[STATES ? 1 : NL], rk[NL], rv[NL];
    const int row0 = min(tid / CPR, C - 1), col0 = tid % CPR * 8;
    const auto load = [&](const uint16_t* m, int64_t first, uint32_t stride, uint32_t offset, v8 (&r)[NL]) { /* bytes */
#pragma unroll
        for (int i = 0; i < NL; ++i)
            r[i] = *reinterpret_cast<const v8*>(reinterpret_cast<const char*>(m) + first + (int64_t)(NT / CPR * i) * stride + offset);
    };
    const uint32_t sq = 2 * (uint32_t)a.q_token_stride, sk = 2 * (uint32_t)a.k_token_stride, sv = 2 * (uint32_t)a.v_token_stride;
    const uint32_t oq = row0 * sq + 2 * col0, ok = row0 * sk + 2 * col0, ov = row0 * sv + 2 * col0;
    const auto load_chunk = [&](int64_t first) { /* 64 tokens from there on */
        if constexpr (!STATES) load(a.q + h * a.q_head_stride, first * sq, sq, oq, rq);
        load(a.k + hk * a.k_head_stride, first * sk, sk, ok, rk);
        load(a.v + hk * a.v_head_stride, first * sv, sv, ov, rv);
    };
    const auto no_keys = [&](int rows) { /* the first ones are not the chunk's */
#pragma unroll
        for (int i = 0; i < NL; ++i)
            if (row0 + NT / CPR * i < rows) rk[i] = rv[i] = v8{};
    };
    const int len = t1 > t0 && !(STATES && last) ? t1 - (int)t0 : 0;
    if (len >= C) {
        load_chunk(t0);
    } else if (len > 0) { /* nothing before it is the segment's, or need exist */
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int64_t t = t0 + max(row0 + NT / CPR * i - (C - len), 0);
            if constexpr (!STATES) rq[i] = ld8<T>(a.q + t * a.q_token_stride + h * a.q_head_stride + col0);
            rk[i] = ld8<T>(a.k + t * a.k_token_stride + hk * a.k_head_stride + col0);
            rv[i] = ld8<T>(a.v + t * a.v_token_stride + hk * a.v_head_stride + col0);
        }
    }

    const float r2 = linear_rate(a, h);
    const auto decay = [&](int n) { return fast_exp2(-r2 * (float)n); };
    const float d1 = decay(1), d2 = decay(2), d3 = decay(3);
    const int number = linear_state(a, lt.seq);
    const int64_t base = ((int64_t)max(number, 0) * a.n_heads + h) * HD * HD + 16 * DV * wd;
    f4* const mine = reinterpret_cast<f4*>(a.ws) + ((int64_t)b * a.n_heads + h) * (HD * HD / 4) + wd * 64 + lane; /* + 64 WD * (tile DV + d) */
    f4 S[DK][DV]; /* rows 16 j + 4 g + e, channels 16 DV wd + channel(d, l16) of the values */
    /* state_out may be state_in, and a sequence's last segment may end before the first one begins: where there are
       several, the launch before this one has read state_in. Its first segment goes on from there, and the last, which
       adds to nothing, leaves a copy for the first. */
    const bool begins = number >= 0 && a.state_in && (STATES ? seg == 0 || last : seg == 0 && last);
#pragma unroll
    for (int j = 0; j < DK; ++j)
#pragma unroll
        for (int d = 0; d < DV; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[j][d][e] = begins ? a.state_in[base + (16 * j + 4 * g + e) * HD + channel(d, l16)] : 0.f;
    if constexpr (!STATES)
        if (seg == 0 && !last) {
            const f4* const copy = mine + (int64_t)((lt.rows.end - lt.rows.start - 1) / a.segment) * a.n_heads * (HD * HD / 4);
#pragma unroll
            for (int j = 0; j < DK * DV; ++j) S[j / DV][j % DV] = copy[64 * WD * j];
        }
    if constexpr (!STATES) {
        constexpr int DEPTH = DK <= 2 ? 16 : DK <= 4 ? 4 : 2; /* segments asked for at once */
        const float keep = decay(a.segment);
        for (int s = seg; s > 0; s -= DEPTH) {
            f4 u[DEPTH][DK * DV];
#pragma unroll
            for (int i = 0; i < DEPTH; ++i)
#pragma unroll
                for (int j = 0; j < DK * DV; ++j) u[i][j] = mine[64 * WD * j - (int64_t)max(s - i, 1) * a.n_heads * (HD * HD / 4)];
#pragma unroll
            for (int i = 0; i < DEPTH; ++i)
                if (i < s)
#pragma unroll
                    for (int j = 0; j < DK * DV; ++j) S[j / DV][j % DV] = S[j / DV][j % DV] * keep + u[i][j];
        }
    }
    if constexpr (!STATES && SHARED) /* keys behind a tile's queries, in the 32 that it has a part of */
        for (int x = tid; x < 256; x += NT)
            *reinterpret_cast<uint64_t*>(lw + ((x / 128 * 6 + x / 64 % 2) * 64 + x % 64) * 8 + 4) = 0;
    const auto weights_at = [](int qt, int m) { return (qt + (qt == 3) + m) * 2 * 64 * 8; }; /* 0, 1, 2 3, 4 5 */

    /* where channel c lies in a row of lq and lk: those that a lane takes of 32 side by side */
    const auto spot = [](int c) { return HD < 32 ? c : (c & ~31) + (c % 16 / 4) * 8 + (c % 32 / 16) * 4 + c % 4; };
    const auto row_of = [&](const uint16_t* m, int row, int ks) {
        if constexpr (HD >= 32) {
            return ld8<T>(m + row * RS + 32 * ks + 8 * g);
        } else {
            const v4 x = *reinterpret_cast<const v4*>(m + row * RS + 4 * g);
            return v8{x[0], x[1], x[2], x[3], (el)0.f, (el)0.f, (el)0.f, (el)0.f};
        }
    };
    const auto transposed = [&](const uint16_t* m, int t, int c) { /* lane l16: channel c + l16, tokens t + 4 g.. and t + 16 + 4 g.. */
        const uint16_t* at = m + (t + 4 * g + l16 / 4) * RS + c;
        union {
            s4 h[2];
            v8 v;
        } f;
        f.h[0] = lds_tr4(at);
        f.h[1] = lds_tr4(at + 16 * RS);
        return f.v;
    };
    if (len < C) no_keys(C - len);
    for (int c0 = 0; c0 < len; c0 += C) {
        const int n = min(C, len - c0), skip = C - n, turn = c0 / C & 1;
        __syncthreads(); /* the chunk before has been read */
        uint32_t mv = 0;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int id = tid + NT * i, row = id / CPR, c = id % CPR * 8;
            if (C * CPR % NT != 0 && row >= C) break;
            if constexpr (!STATES) {
                *reinterpret_cast<v4*>(lq + row * RS + spot(c)) = v4{rq[i][0], rq[i][1], rq[i][2], rq[i][3]};
                *reinterpret_cast<v4*>(lq + row * RS + spot(c + 4)) = v4{rq[i][4], rq[i][5], rq[i][6], rq[i][7]};
                mv = most2(mv, most8(rv[i]));
            }
            *reinterpret_cast<v4*>(lk + row * RS + spot(c)) = v4{rk[i][0], rk[i][1], rk[i][2], rk[i][3]};
            *reinterpret_cast<v4*>(lk + row * RS + spot(c + 4)) = v4{rk[i][4], rk[i][5], rk[i][6], rk[i][7]};
            st8<T>(lv + row * RS + c, rv[i]);
        }
        if constexpr (!STATES) {
            const bool bad = __any(infinite<T>(mv));
            if (lane == 0) lbad[turn][wave] = bad;
        }
        __syncthreads();

        if (c0 + C < len) {
            const int early = max(2 * C - (len - c0), 0);
            load_chunk(t0 + c0 + C - early);
            if (early > 0) no_keys(early);
        }
        v8 v[DV][M]; /* lane l16 is a channel */
        const auto values = [&] {
#pragma unroll
            for (int d = 0; d < DV; ++d)
#pragma unroll
                for (int m = 0; m < M; ++m) v[d][m] = transposed(lv, 32 * m, 16 * DV * wd + channel(d, 4 * (l16 & 3)));
        };
        if constexpr (!STATES) {
            uint32_t bad = 0;
#pragma unroll
            for (int i = 0; i < WD * WQ; ++i) bad |= lbad[turn][i];
            /* weights of 16 queries and 16 keys: lane l16 is a query, with keys 4 g + e; as two numbers of bf16 */
            const auto weigh = [&](int qt, int kt, uint32_t (&hi)[2], uint32_t (&lo)[2]) {
                f4 w = {};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) w = mfma_16x16x32(row_of(lk, 16 * kt + l16, ks), row_of(lq, 16 * qt + l16, ks), w);
                const int gap = 16 * (qt - kt) + l16 - 4 * g;
                if (kt < qt) { /* gap is 4 or more */
                    const float far = decay(gap - 3) * a.scale;
                    w[0] *= far * d3;
                    w[1] *= far * d2;
                    w[2] *= far * d1;
                    w[3] *= far;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = gap >= e ? w[e] * (decay(max(gap - e, 0)) * a.scale) : 0.f;
                }
                uint32_t p[2][2];
                parts<2>(w[0], w[1], p[0]);
                parts<2>(w[2], w[3], p[1]);
                hi[0] = p[0][0];
                hi[1] = p[1][0];
                lo[0] = p[0][1];
                lo[1] = p[1][1];
            };
            const auto tile_of = [&](int i) { return WQ == 1 ? i : WQ == QT ? wq : i == 0 ? wq : QT - 1 - wq; };
            if constexpr (SHARED) {
                for (int x = wave; x < TILES; x += WD) {
                    const int qt = (x >= 1) + (x >= 3) + (x >= 6), kt = x - qt * (qt + 1) / 2;
                    uint32_t hi[2], lo[2];
                    weigh(qt, kt, hi, lo);
                    uint16_t* to = lw + weights_at(qt, kt / 2) + lane * 8 + kt % 2 * 4;
                    *reinterpret_cast<uint64_t*>(to) = hi[0] | (uint64_t)hi[1] << 32;
                    *reinterpret_cast<uint64_t*>(to + 64 * 8) = lo[0] | (uint64_t)lo[1] << 32;
                }
            }
            f4 o[QN][DV] = {};
            /* q S, the state as two numbers of bf16: lane l16 is a channel of the values, with 8 of each 32 channels of the keys */
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                b8 s[DV][2];
#pragma unroll
                for (int d = 0; d < DV; ++d) {
                    u4 hi = {}, lo = {};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = 2 * ks + e / 2;
                        if (j >= DK) continue;
                        uint32_t p[2];
                        const float x = S[j < DK ? j : 0][d][e % 2 * 2], y = S[j < DK ? j : 0][d][e % 2 * 2 + 1];
                        parts<2>(x, y, p);
                        hi[e] = p[0];
                        lo[e] = p[1];
                    }
                    s[d][0] = __builtin_bit_cast(b8, hi);
                    s[d][1] = __builtin_bit_cast(b8, lo);
                }
                b8 q[QN][IN];
#pragma unroll
                for (int i = 0; i < QN; ++i) numbers(row_of(lq, 16 * tile_of(i) + l16, ks), q[i]);
#pragma unroll
                for (int part = 0; part < 2; ++part)
#pragma unroll
                    for (int x = 0; x < IN - part * (IN - 1); ++x)
#pragma unroll
                        for (int i = 0; i < QN; ++i)
#pragma unroll
                            for (int d = 0; d < DV; ++d) o[i][d] = mfma_16x16x32(s[d][part], q[i][x], o[i][d]);
            }
#pragma unroll
            for (int i = 0; i < QN; ++i) {
                const float far = decay(max(16 * tile_of(i) + l16 + 1 - skip, 0)) * a.scale;
#pragma unroll
                for (int d = 0; d < DV; ++d) o[i][d] *= far;
            }
            /* values that are not finite must not meet weights of zero: queries before them */
            const bool poisoned = __builtin_amdgcn_readfirstlane(bad) != 0;
            if constexpr (SHARED) __syncthreads(); /* the weights are in */
            values();
            if (poisoned)
#pragma unroll
                for (int d = 0; d < DV; ++d)
#pragma unroll
                    for (int m = 0; m < M; ++m)
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[d][m][e] = __builtin_fabsf((float)v[d][m][e]) < INFINITY ? v[d][m][e] : (el)0.f;
            b8 vb[DV][M][IN];
#pragma unroll
            for (int d = 0; d < DV; ++d)
#pragma unroll
                for (int m = 0; m < M; ++m) numbers(v[d][m], vb[d][m]);
            if constexpr (SHARED) {
#pragma unroll
                for (int m = 0; m < M; ++m)
#pragma unroll
                    for (int part = 0; part < 2; ++part)
#pragma unroll
                        for (int qt = 2 * m; qt < QT; ++qt) {
                            const b8 w = ld8<BF16>(lw + weights_at(qt, m) + (part * 64 + lane) * 8);
#pragma unroll
                            for (int i = 0; i < IN - part * (IN - 1); ++i)
#pragma unroll
                                for (int d = 0; d < DV; ++d) o[qt][d] = mfma_16x16x32(vb[d][m][i], w, o[qt][d]);
                        }
            } else {
#pragma unroll
                for (int i = 0; i < QN; ++i) {
                    const int qt = tile_of(i);
#pragma unroll
                    for (int m = 0; m < M; ++m) {
                        if (2 * m > qt) break;
                        uint32_t hi[2][2], lo[2][2] = {};
                        weigh(qt, 2 * m, hi[0], lo[0]);
                        if (2 * m < qt) weigh(qt, 2 * m + 1, hi[1], lo[1]);
                        else hi[1][0] = hi[1][1] = 0;
                        const b8 first = __builtin_bit_cast(b8, u4{hi[0][0], hi[0][1], hi[1][0], hi[1][1]});
                        const b8 second = __builtin_bit_cast(b8, u4{lo[0][0], lo[0][1], lo[1][0], lo[1][1]});
#pragma unroll
                        for (int d = 0; d < DV; ++d) {
#pragma unroll
                            for (int x = 0; x < IN; ++x) o[i][d] = mfma_16x16x32(vb[d][m][x], first, o[i][d]);
                            o[i][d] = mfma_16x16x32(vb[d][m][0], second, o[i][d]);
                        }
                    }
                }
            }
            if (poisoned) /* what sees one of them */
#pragma unroll
                for (int d = 0; d < DV; ++d) {
                    int from[4] = {C, C, C, C}; /* the first in channel 4 g + e */
                    for (int t = C - 1; t >= 0; --t)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (!(__builtin_fabsf(ld1<T>(lv + t * RS + 16 * DV * wd + channel(d, 4 * g + e))) < INFINITY)) from[e] = t;
#pragma unroll
                    for (int i = 0; i < QN; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[i][d][e] = 16 * tile_of(i) + l16 >= from[e] ? __builtin_nanf("") : o[i][d][e];
                }
#pragma unroll
            for (int i = 0; i < QN; ++i) {
                const int row = 16 * tile_of(i) + l16;
                if (row < skip) continue;
                uint16_t* first = a.out + (t0 + c0) * a.out_token_stride + h * a.out_head_stride + 16 * DV * wd;
                first += (uint32_t)(row - skip) * (uint32_t)a.out_token_stride + channel(0, 4 * g);
                el r[4 * DV];
#pragma unroll
                for (int x = 0; x < 4 * DV; ++x) r[x] = (el)opaque(o[i][x / 4][x % 4]);
                __builtin_memcpy(__builtin_assume_aligned(first, 8 * DV), r, sizeof(r));
            }
        }
        /* the next state */
        values();
        const float keep = decay(n);
        float fade[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) fade[i] = decay(15 - 4 * g - i);
        const auto faded = [&](int d, int m, float (&x)[8]) {
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const float far = decay(C - 16 - 32 * m - 4 * e);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[e + i] = (float)v[d][m][e + i] * (fade[i] * far);
            }
        };
        const auto key = [&](int m, int j) { return transposed(lk, 32 * m, spot(16 * j + 4 * (l16 & 3))); };
        constexpr int J = DK < 4 / DV ? DK : 4 / DV; /* tiles side by side: their products do not wait for each other */
        /* decayed values as three numbers of bf16, which leave 2^-27 of them; keys' second numbers (fp16) do without the third */
#pragma unroll
        for (int j = 0; j < DK; ++j)
#pragma unroll
            for (int d = 0; d < DV; ++d) S[j][d] *= keep;
#pragma unroll
        for (int m = 0; m < M; ++m) {
            u4 w[DV][3];
#pragma unroll
            for (int d = 0; d < DV; ++d) {
                float x[8];
                faded(d, m, x);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t p[3];
                    parts<3>(x[2 * e], x[2 * e + 1], p);
#pragma unroll
                    for (int i = 0; i < 3; ++i) w[d][i][e] = p[i];
                }
            }
#pragma unroll
            for (int j0 = 0; j0 < DK; j0 += J) {
                b8 k[J][IN];
#pragma unroll
                for (int j = 0; j < J; ++j) numbers(key(m, j0 + j), k[j]);
#pragma unroll
                for (int i = 0; i < 3; ++i)
#pragma unroll
                    for (int x = 0; x < (i < 2 ? IN : 1); ++x)
#pragma unroll
                        for (int j = 0; j < J; ++j)
#pragma unroll
                            for (int d = 0; d < DV; ++d) S[j0 + j][d] = mfma_16x16x32(k[j][x], __builtin_bit_cast(b8, w[d][i]), S[j0 + j][d]);
            }
        }
    }
    if (wq > 0) return; /* the same state */
    if constexpr (STATES) {
#pragma unroll
        for (int j = 0; j < DK * DV; ++j) mine[64 * WD * j] = S[j / DV][j % DV];
    } else if (number >= 0 && a.state_out && t1 == lt.rows.end) {
#pragma unroll
        for (int j = 0; j < DK; ++j)
#pragma unroll
            for (int d = 0; d < DV; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) a.state_out[base + (16 * j + 4 * g + e) * HD + channel(d, l16)] = S[j][d][e];
    }
}

/* One token of a sequence and head, in fp32: a wave (128 channels: four), whose lanes have four columns of R rows of the state
 * each, 16 bytes a load; sums over the rows meet across lanes. Bound by HBM: the state read and written once, 8,160 x 8 x 32 x 32
 * 95 us (551 MB, 5.8 TB/s; a copy of as much 108). A lane a column, 4 bytes a load, took 129. */
template <class T, int HD>
__device__ __forceinline__ void linear_step(const LinearAttnArgs& a) {
    typedef typename T::v4 v4;
    constexpr int WPI = HD == 128 ? 4 : 1, COLS = HD / 4, R = HD / (64 / COLS) / WPI; /* waves a head; lanes a row; rows of a lane */
    __shared__ f4 part[WPI > 1 ? 4 * 32 : 1];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t item = WPI > 1 ? blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
    if (item >= (int64_t)a.n_seqs * a.n_heads) return;
    const int s = (int)(item / a.n_heads), h = (int)(item % a.n_heads), hk = h / (a.n_heads / a.n_kv_heads);
    const int c = lane % COLS * 4, r0 = ((WPI > 1 ? wave : 0) * (64 / COLS) + lane / COLS) * R;
    const int number = linear_state(a, s);
    uint16_t* out = a.out + s * a.out_token_stride + h * a.out_head_stride + c;
    const bool first = lane < COLS && (WPI == 1 || wave == 0);
    if (number < 0) {
        if (first) *reinterpret_cast<v4*>(out) = v4{};
        return;
    }
    const int64_t at = ((int64_t)number * a.n_heads + h) * HD * HD + r0 * HD + c;
    f4 S[R];
#pragma unroll
    for (int i = 0; i < R; ++i) S[i] = *reinterpret_cast<const f4*>(a.state_in + at + i * HD);
    const float keep = fast_exp2(-linear_rate(a, h));
    const uint16_t* q = a.q + s * a.q_token_stride + h * a.q_head_stride + r0;
    const uint16_t* k = a.k + s * a.k_token_stride + hk * a.k_head_stride + r0;
    const v4 vv = *reinterpret_cast<const v4*>(a.v + s * a.v_token_stride + hk * a.v_head_stride + c);
    const f4 v = __builtin_convertvector(vv, f4);
    typename T::el kr[R], qr[R];
    __builtin_memcpy(kr, k, 2 * R);
    __builtin_memcpy(qr, q, 2 * R);
    f4 o = {};
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            S[i][e] = __builtin_fmaf((float)kr[i], v[e], S[i][e] * keep);
            o[e] = __builtin_fmaf((float)qr[i], S[i][e], o[e]);
        }
        *reinterpret_cast<f4*>(a.state_out + at + i * HD) = S[i];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float x, y;
        if constexpr (COLS <= 4) o[e] += dpp<0x141>(dpp<0x1B>(o[e])); /* lane ^ 4: quads mirrored in eights, and back within */
        if constexpr (COLS <= 8) o[e] += dpp<0x128>(o[e]);            /* lane ^ 8 */
        if constexpr (COLS <= 16) {
            lanes_x16(o[e], x, y);
            o[e] = x + y;
        }
        lanes_x32(o[e], x, y);
        o[e] = x + y;
    }
    if constexpr (WPI > 1) {
        if (lane < COLS) part[wave * 32 + lane] = o;
        __syncthreads();
        if (first) o = (part[lane] + part[32 + lane]) + (part[64 + lane] + part[96 + lane]);
    }
    if (first) {
        v4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = (typename T::el)opaque(o[e] * a.scale);
        *reinterpret_cast<v4*>(out) = r;
    }
}

#define LINEAR(NAME, T, HD)                                                                                                   \
    extern "C" __global__ void __launch_bounds__(256, HD < 32 ? 4 : HD < 128 ? 3 : 2) prism_linear_attn_##NAME##_h##HD(LinearAttnArgs a) { linear_segment<T, HD, false>(a); } \
    extern "C" __global__ void __launch_bounds__(HD < 128 ? 4 * HD : 256, HD < 128 ? 3 : 2) prism_linear_states_##NAME##_h##HD(LinearAttnArgs a) { linear_segment<T, HD, true>(a); } \
    extern "C" __global__ void __launch_bounds__(256) prism_linear_step_##NAME##_h##HD(LinearAttnArgs a) { linear_step<T, HD>(a); }
LINEAR(f16, F16, 16) LINEAR(f16, F16, 32) LINEAR(f16, F16, 64) LINEAR(f16, F16, 128)
LINEAR(bf16, BF16, 16) LINEAR(bf16, BF16, 32) LINEAR(bf16, BF16, 64) LINEAR(bf16, BF16, 128)
#undef LINEAR
