/*
 * seq_attn.hpp - attention along (ragged) sequences with a sliding window and
 * sinks: query i of a sequence of nq queries and nk keys stands at position
 * p = nk - nq + i and sees keys j <= p + right with j >= p - left or j < sinks.
 *
 * A workgroup takes 128 or 64 rows, 32 a wave: a row is a query of one head, the heads
 * that share a key head side by side (so the workgroup's queries are fewer, and the keys that they see
 * together too). It goes once over the keys that any of them sees, in tiles of 64,
 * 128 or 256, with a running maximum and sum; with few workgroups, 2 or 4 waves
 * take the same rows, each some keys of every tile, and are joined at the end:
 *   S^T = K Q^T           (32x32x16 MFMA: a lane holds one query's scores)
 *   P^T = 2^(c S^T - c m) (registers; c = scale log2 e)
 *   O^T += V^T P^T        (P^T is the B operand as it lies: the MFMA's
 *                          reduction index may be numbered in any order, and
 *                          V^T is read from LDS in that order by transposing
 *                          reads)
 * The weights are rounded to the type of the values, which is what the products
 * take: each by half a step, as the output is, so that the two together err 1.2 to
 * 1.4 times as much as the output's rounding alone (rms 1.73e-5 and 1.28e-5 at 8,160
 * queries x 32 channels in fp16, 1.11e-4 and 7.9e-5 at 128 channels in bf16). Two 16-bit numbers a
 * weight, as paged_attn.hpp has them where they are free, leave the output's rounding alone and
 * took, in us: 8,160, 8 x 32, window 1,023: 41.6 instead of 29.2; 4,000, 32 x 64: 146 instead of
 * 91; two of 4,501 and 5,800, 32/8 x 128: 404 instead of 310. With this order
 * a query's maximum, sum and rescaling stay in its lane (two lanes, 32
 * apart, hold halves of its keys). K and V tiles go through LDS, double
 * buffered, the next tile's loads in flight under the current tile's products.
 * Keys that no query of the workgroup sees are staged as zeros. Where only some
 * queries see a tile's key, its weight is zero for the others; should such a
 * V be infinite or NaN (0 * inf), the workgroup does its rows again one by one,
 * and so it does where scaled scores pass 2^22.
 */
#pragma once
#include "seq_types.hpp"

typedef float f16v __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f16v mfma_32x32x16(h8 a, h8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f16v mfma_32x32x16(b8 a, b8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

template <class T>
__device__ __forceinline__ typename T::v8 splat_one() {
    typename T::v8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (typename T::el)1.0f;
    return v;
}

/* 16 bytes a lane from a buffer straight to LDS, 1 KiB in a row from byte address `to` (the same in every
 * lane) on; lanes past the buffer's end write zeros. In assembly because the compiler would wait for it before
 * the next LDS read, whichever: the caller waits (vm_wait) before the barrier behind which the data is read. */
typedef int i4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i4 buffer_of(const void* p, int bytes) {
    const uint64_t at = (uint64_t)p;
    return i4{(int)at, (int)(at >> 32) & 0xFFFF, bytes, 0x00020000};
}
__device__ __forceinline__ void load_to_lds(i4 buffer, int offset, unsigned to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 ::"s"(to), "v"(offset), "s"(buffer)
                 : "memory", "m0");
}
/* Computed here and not nearer to its use: keeps what goes beside the matrix products there. */
template <class T>
__device__ __forceinline__ T pinned(T v) {
    asm volatile("" : "+v"(v));
    return v;
}
__device__ __forceinline__ void vm_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

/* One query by the whole wave, a step for every 64 keys that it sees: a lane per key for the scores, then a lane per
 * channel for the values, key after key. The workgroup's way out where zero weights would meet infinite values, and for
 * huge scores. One infinite value near the end of 20,000 queries that see all before them, 8 heads x 128: 58 ms, and 0.8
 * without it; with a step for every key it was 256. */
template <class T, int HD>
__device__ __forceinline__ void seq_attn_row(const SeqAttnArgs& a, const uint16_t* q, const uint16_t* k, const uint16_t* v,
                                             uint16_t* out, const KeyRange kr) {
    constexpr int E = (HD + 63) / 64, U = 16;
    const int lane = lane_id(), n = kr.sink + kr.hi - kr.lo;
    const bool on = lane < HD;
    const auto key = [&](int i) -> int64_t { return i < kr.sink ? i : kr.lo + i - kr.sink; };
    float acc[E] = {}, m = -INFINITY, l = 0.f; /* l: of the lane's keys */
    for (int i0 = 0; i0 < n; i0 += 64) {
        const uint16_t* kp = k + key(seq_min(i0 + lane, n - 1)) * a.k_token_stride;
        float d = 0.f;
#pragma unroll 8
        for (int c = 0; c < HD; c += 8) {
            const typename T::v8 x = ld8<T>(q + c), y = ld8<T>(kp + c);
#pragma unroll
            for (int e = 0; e < 8; ++e) d = __builtin_fmaf((float)x[e], (float)y[e], d);
        }
        d = i0 + lane < n ? d * a.scale_log2 : -INFINITY;
        float top = fmaxf(m, d);
        for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
        const float mu = top == -INFINITY ? 0.f : top, f = fast_exp2(m - mu), p = fast_exp2(d - mu);
        l = __builtin_fmaf(l, f, p);
        m = top;
        for (int e = 0; e < E; ++e) acc[e] *= f;
        for (int i = i0; i < seq_min(i0 + 64, n); i += U) {
            float w[U], x[U][E];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                w[u] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, p), i - i0 + u));
                const uint16_t* vp = v + key(seq_min(i + u, n - 1)) * a.v_token_stride;
                for (int e = 0; e < E; ++e) x[u][e] = on ? ld1<T>(vp + lane + 64 * e) : 0.f;
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                for (int e = 0; e < E; ++e) acc[e] = i + u < n ? __builtin_fmaf(w[u], x[u][e], acc[e]) : acc[e];
        }
    }
    l = wave_sum(l);
    for (int e = 0; e < E; ++e)
        if (on) st1<T>(out + lane + 64 * e, l == 0.f ? 0.f : acc[e] / l);
}

/* The sequence whose query tiles include tile b, and its rows: sequence s owns the
 * tiles from floor(start / tile_q) + s on, which leaves each enough of them
 * whatever the lengths. 64 candidates a step; the last step's loads bring the
 * rows along. */
struct SeqTile {
    int first;     /* the sequence's first tile */
    RowRange q, k;
};
__device__ __forceinline__ SeqTile seq_of_tile(const SeqAttnArgs& a, int b) {
    int lo = 0, n = a.n_seqs;
    const int lane = lane_id();
    while (true) {
        const int step = (n + 63) / 64;
        const int s = lo + min(lane, (n - 1) / step) * step; /* lanes past the end: the last one again */
        const RowRange q = row_range(a.cu_q, s, a.n_seqs, a.n_q);
        RowRange k{0, 0};
        if (step == 1) k = row_range(a.cu_k, s, a.n_seqs, a.n_k);
        const int key = q.start / a.tile_q + s;
        const unsigned long long mask = __ballot(key <= b);
        const int at = mask ? min(63 - __builtin_clzll(mask), (n - 1) / step) : 0;
        if (step == 1) {
            const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, at); };
            return SeqTile{of(key), RowRange{of(q.start), of(q.end)}, RowRange{of(k.start), of(k.end)}};
        }
        lo += at * step;
        n = min(step, n - at * step);
    }
}

/* RW: waves, 32 rows each; KW: groups of them, which share the rows, each taking its keys of every tile. */
template <class T, int HD, int RW, int KW>
__device__ __forceinline__ void seq_attn_body(const SeqAttnArgs& a) {
    typedef typename T::v8 v8;
    constexpr int NP = HD <= 32 && KW == 1 ? 4 : 2; /* parts of 32 keys that a wave has of a tile */
    constexpr int NTHR = 64 * RW * KW, BN = 32 * NP * KW; /* threads; keys per tile */
    constexpr int KS = HD / 16;              /* k-steps of the scores          */
    constexpr int DT = (HD + 31) / 32;       /* 32-channel tiles of the output */
    constexpr bool ONES = HD == 16 || (HD <= 64 && KW == 1); /* sums of weights on the matrix cores, see below */
    constexpr int NS = KS > 2 * DT ? KS : 2 * DT; /* steps of a part           */
    constexpr int EL = 16 / NS;              /* scores per lane and step       */
    constexpr int CPR = HD / 8;              /* 16-byte chunks of a row        */
    constexpr int CHUNKS = BN * CPR, CH = (CHUNKS + NTHR - 1) / NTHR; /* per tile, per thread */
    constexpr int TILE = 2 * BN * HD;        /* bytes of a tile of K or V      */
    constexpr int KRING = (NP == 2 ? 2 : 3) * TILE, KVBYTES = KRING + 2 * TILE, MERGE = (KW - 1) * RW * 64 * (16 * DT + 2) * 4;
    __shared__ __attribute__((aligned(16))) uint8_t lds[KVBYTES > MERGE ? KVBYTES : MERGE]; /* a ring of K tiles, two V tiles */
    const auto uni = [](int v) { return __builtin_amdgcn_readfirstlane(v); };

    /* workgroup -> (query tile, head): an XCD (workgroups b, b + 8, ...) takes a
     * run of neighbouring heads, whose keys its L2 then holds; the last tiles, whose
     * queries may see the most keys, come first, so the launch ends with short ones
     * (with whole groups of heads per XCD, over all of them). Measured together with LDS addresses in
     * registers and 16-byte stores: 2 of 5,000 queries, 32 heads x 128, 409 -> 374 us. */
    const int tiles = a.n_q / a.tile_q + a.n_seqs, groups = a.n_heads / a.tile_heads, b = blockIdx.x, xcd = b & 7;
    int hg, tile; /* group of heads, tile of queries */
    if (groups % 8 == 0) {
        const int some = groups / 8, i = b >> 3;
        tile = tiles - 1 - i / some;
        hg = xcd * some + i % some;
    } else {
        const int total = tiles * groups, w = xcd * (total >> 3) + min(xcd, total & 7) + (b >> 3);
        hg = w / tiles;
        tile = tiles - 1 - (w - hg * tiles);
    }
    const int hk = hg * a.tile_heads / (a.n_heads / a.n_kv_heads);
    const SeqTile st = seq_of_tile(a, tile);
    const RowRange rq = st.q, rk = st.k;
    const int first = st.first;
    const int nq = rq.end - rq.start, nk = rk.end - rk.start;
    if (tile < first || (int64_t)(tile - first) * a.tile_q >= nq) return; /* uniform over the workgroup */
    const int q0 = (tile - first) * a.tile_q, q1 = min(q0 + a.tile_q, nq);

    /* A SIMD's turns go first to waves outside of the products: what they do there is one chain, maximum, exchange,
       branch, and products are behind it. 8,160 queries, 8 heads x 32, window 1,023: 27.4 -> 25.2 us; 2,000 x 16,
       all keys: 14.5 -> 13.2; x 64: 18.4 -> 17.7; 4,000, 32 heads x 128: 139.5 -> 136.7, x 64: 85.7 -> 87.3 (at 64
       it gains with few workgroups and costs with many; one rule for all widths). */
    __builtin_amdgcn_s_setprio(3);
    const int lane = lane_id(), c32 = lane & 31, g = lane >> 5;
    const int wave8 = uni(threadIdx.x >> 6), wave = wave8 % RW, kgroup = wave8 / RW;
    const int row = 32 * wave + c32; /* this lane's; the wave's queries: qa .. qb - 1 */
    const int qa = q0 + 32 * wave / a.tile_heads, qb = min(q0 + (32 * wave + 31) / a.tile_heads + 1, q1);
    const int shift = nk - nq;                            /* position - row */
    const bool on = qa < q1;

    const uint16_t* kb = a.k + rk.start * a.k_token_stride + hk * a.k_head_stride;
    const uint16_t* vb = a.v + rk.start * a.v_token_stride + hk * a.v_head_stride;
    const int qrow = q0 + row / a.tile_heads, h = hg * a.tile_heads + row % a.tile_heads;
    const int qi = min(qrow, q1 - 1); /* past the end: the last one, never stored */
    const uint16_t* qp = a.q + (rq.start + qi) * a.q_token_stride + h * a.q_head_stride;

    /* Keys that the workgroup's, the wave's and the lane's queries see. Tiles go over
     * the sinks first (if a window begins behind them), then over the rest of the
     * window, so a tile needs no more than one comparison per end. */
    const KeyRange r0 = key_range(shift + q0, nk, a.left, a.right, a.sinks);
    const KeyRange r1 = key_range(shift + q1 - 1, nk, a.left, a.right, a.sinks);
    const KeyRange me = key_range(shift + qi, nk, a.left, a.right, a.sinks);
    const int sink_end = r1.lo > 0 ? seq_min(a.sinks, r1.hi) : 0;
    const int win0 = seq_max(r0.lo, sink_end), win1 = r1.hi;
    const int sink_tiles = (sink_end + BN - 1) / BN;
    const int n_tiles = sink_tiles + (win1 > win0 ? (win1 - win0 + BN - 1) / BN : 0);
    const KeyRange ra = key_range(shift + qa, nk, a.left, a.right, a.sinks);
    const KeyRange rb = key_range(shift + qb - 1, nk, a.left, a.right, a.sinks);
    const int a_lo = uni(ra.lo), a_hi = uni(ra.hi), b_lo = uni(rb.lo), b_hi = uni(rb.hi);

    const int see_hi = on ? b_hi : INT32_MIN, see_sink = seq_min(see_hi, sink_end);
    unsigned bad = 0; /* infinite or NaN V where only some of the queries look, or scores too large for mc */
    /* c s - mc is one FMA with the rounded mc, which leaves weights a factor of up to half a step of mc: it cancels in
       the division, but has to fit the weights' type: 2^(1/4) at 2^22, 2^64 at 2^30. */
    constexpr float MAX_FAST = 0x1p22f;
    v8 qf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = ld8<T>(qp + 16 * ks + 8 * g);

    f16v o[DT] = {};
    /* fp16 weights are 2^UP times as large, with which the lag (see limit) stays below 2^16: what is lost of a weight
       is below 2^-32 of the largest, not 2^-25. Many keys behind one strong key may matter. */
    constexpr float UP = __is_same(T, F16) ? 7.f : 0.f;
    float m = -INFINITY, mc = 0.f, l = 0.f; /* mc = c m - UP, or 0 while m is -inf */
    /* The sum of a query's weights: as many additions as weights on the vector units, or products with ones on
       the matrix cores, which wait for the vector units up to 64 channels (5 sequences of 243 to 3,788 queries, 20
       heads x 32: 113 us and, added, 129; 8 waves have no registers for it). 16 channels leave half of the
       output's rows free: there V's unused rows are the ones. The weights summed are then the rounded ones. */
    f16v lsum = {};
    const v8 ones = splat_one<T>();
    float limit = -INFINITY;
    const float lag = fminf(8.0f / a.scale_log2, 0x1.fffffep127f); /* finite: -inf + lag has to stay -inf, the limit of who saw no key */

    /* k0 of tile t + 1, from tile t's; where a tile's keys end */
    auto step = [&](int t, int k0) { return t + 1 == sink_tiles ? win0 : k0 + BN; };
    auto end_of = [&](int t) { return t < sink_tiles ? sink_end : win1; };
    /* Tiles go from memory to LDS directly, 64 chunks of 16 bytes in a row per wave and load. A lane may choose
       which chunk it brings, so chunk c of row r lies at place c ^ swizzle(r): for K, 16 rows' chunks of one
       column then lie in different banks; for V, 4 rows' groups of 64 bytes. Rows past the end lie past the
       buffer and are written as zeros. */
    auto swizzle_k = [](int r) { return CPR < 16 ? r / (16 / CPR) & (CPR - 1) : r & 15; };
    auto swizzle_v = [](int r) { return HD == 128 ? (r & 3) * 4 : HD == 64 ? (r >> 1 & 1) * 4 : 0; };
    int koff[CH], voff[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int id = (threadIdx.x + NTHR * c) % CHUNKS, r = id / CPR, e = id % CPR;
        koff[c] = 2 * (r * (int)a.k_token_stride + (e ^ swizzle_k(r)) * 8);
        voff[c] = 2 * (r * (int)a.v_token_stride + (e ^ swizzle_v(r)) * 8);
    }
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) uint8_t*)lds;
    auto fetch = [&](int to, const uint16_t* base, int stride, const int (&off)[CH], int t, int k0) {
        if (t >= n_tiles) return;
        const int rows = seq_min(end_of(t) - k0, BN);
        const i4 buffer = buffer_of(base + (int64_t)k0 * stride, 2 * ((rows - 1) * stride + HD));
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int id0 = 64 * wave8 + NTHR * c; /* the wave's first chunk */
            if (CHUNKS % NTHR == 0 || id0 < CHUNKS) load_to_lds(buffer, off[c], lds0 + to + 16 * id0);
        }
    };
    auto check_v = [&](int at, int t, int k0) { /* a tile that some queries see only in part: finite? (Rows past the
                                                    end are zeros where V's rows do not overlap.) */
        if ((t >= sink_tiles && k0 < r1.lo) || k0 + BN > seq_min(r0.hi, end_of(t))) {
            constexpr unsigned E = __is_same(T, F16) ? 0x7C007C00u : 0x7F807F80u;
            constexpr unsigned U = __is_same(T, F16) ? 0x04000400u : 0x00800080u;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int id = (threadIdx.x + NTHR * c) % CHUNKS;
                const u4 d = *reinterpret_cast<const u4*>(lds + KRING + at + 16 * id);
#pragma unroll
                for (int i = 0; i < 4; ++i) bad |= (d[i] & E) + U;
            }
        }
    };

    /* The wave's keys go in parts of 32. In the body for part i three parts are under way: the scores of
       part i + 1 and the products of part i - 1 on the matrix cores, the weights of part i on the vector
       units, a few of each at a time. */
    union VFrag {
        s4 h[2];
        v8 v;
    };
    /* this lane's places (bytes from the rings on), to be xored with 32 per k-step and 64 per 32 channels */
    const int krow = 2 * (32 * NP * kgroup + c32) * HD + 16 * (g ^ swizzle_k(c32));
    const int vrow = 2 * (32 * NP * kgroup + 4 * g + (lane & 15) / 4) * HD +
                     ((HD >= 32 ? 2 * (lane & 16) : 0) ^ 16 * swizzle_v((lane & 15) / 4)) + 8 * (lane & 3);
    int kat[KS], vat[DT];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kat[ks] = opaque(krow ^ 32 * ks);
#pragma unroll
    for (int d = 0; d < DT; ++d) vat[d] = opaque(KRING + (vrow ^ 64 * d));
    auto read_k = [&](int off, int ks) { return *reinterpret_cast<const v8*>(lds + kat[ks] + off); };
    /* does the wave see any of the part of tile t that starts at k0? (whole numbers: scalar code) */
    auto active = [&](int t, int k0) -> int {
        const int hi = t < n_tiles ? (t < sink_tiles ? see_sink : see_hi) : INT32_MIN;
        const int lo = t < sink_tiles ? INT32_MIN : a_lo - 32;
        return (int)(k0 < hi) & (int)(k0 > lo);
    };
    auto read_v = [&](VFrag& f, int off, int j) { /* 16 keys j / DT, channels 32 (j % DT) ..: V^T as
                                                    lane's rows keys 4 g ..+3 and 8 more on */
        const uint8_t* v = lds + vat[j % DT] + (off + 32 * (j / DT) * HD);
        f.h[0] = lds_tr4(v);
        f.h[1] = lds_tr4(v + 16 * HD);
        if constexpr (HD == 16) { /* every lane takes part in the transposing read */
            f.v = opaque(f.v);
            f.v = c32 >= 16 ? ones : f.v;
        }
    };
    auto weights = [](const unsigned (&p)[8], int i) { return __builtin_bit_cast(v8, u4{p[4 * i], p[4 * i + 1], p[4 * i + 2], p[4 * i + 3]}); };
    auto none = [](unsigned (&p)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = 0;
    };
    /* sc, p: scores and weights of the part at k0 of tile t; sn: scores of the next part (keys at ka); pl: weights
       of the last one (values at va). A part that the wave does not see gets zero weights. */
    auto body = [&](int t, int k0, int ka, int va, f16v& sc, f16v& sn, unsigned (&p)[8], const unsigned (&pl)[8]) {
        v8 kf[3];
        VFrag vf[3];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (j < KS) kf[j] = read_k(ka, j);
            if (j < 2 * DT) read_v(vf[j], va, j);
        }
        const int end = end_of(t);
        const bool cut_lo = t >= sink_tiles && k0 < b_lo;
        if (k0 + 32 > seq_min(a_hi, end) || cut_lo) {
            const int hi = seq_clamp(seq_min(me.hi, end) - k0, 0, 32), lo = cut_lo ? seq_clamp(me.lo - k0, 0, 32) : 0;
            const unsigned seen = ((unsigned)(((uint64_t)1 << hi) - ((uint64_t)1 << seq_min(lo, hi)))) >> (4 * g);
#pragma unroll
            for (int e = 0; e < 16; ++e) { /* a bit field and a bit select: no compare to wait for */
                const int all = (int)(seen << (31 - 8 * (e / 4) - (e & 3))) >> 31;
                const float x = sc[e];
                sc[e] = __builtin_bit_cast(float, (__builtin_bit_cast(int, x) & all) | ((int)0xFF800000 & ~all));
            }
        }
        float top = vmax(sc[0], sc[1]), x, y;
#pragma unroll
        for (int e = 2; e < 16; e += 2) top = vmax3(top, sc[e], sc[e + 1]);
        lanes_x32(top, x, y);
        top = vmax(x, y);
        /* the maximum may lag by 8 powers of two: weights up to 256 (fp16: 2^15) cost no precision, rescaling
           costs much */
        float f = 1.f;
        const bool scale = __any(top > limit);
        if (scale) {
            top = vmax(top, m);
            const float tc = top == -INFINITY ? 0.f : top * a.scale_log2 - UP;
            if (__builtin_fabsf(tc) >= MAX_FAST) bad = ~0u;
            f = fast_exp2(m == -INFINITY ? -INFINITY : mc - tc);
            if (!ONES) l *= f;
            m = top;
            mc = tc;
            limit = top + lag;
        }
        __builtin_amdgcn_s_setprio(0);
        sn = f16v{};
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            if (j + 2 < KS) kf[(j + 2) % 3] = read_k(ka, j + 2);
            if (j + 2 < 2 * DT) read_v(vf[(j + 2) % 3], va, j + 2);
            if (j < KS) sn = mfma_32x32x16(kf[j % 3], qf[j], sn);
#pragma unroll
            for (int e = EL * j; e < EL * (j + 1); e += 2) {
                const float z0 = fast_exp2(__builtin_fmaf(sc[e], a.scale_log2, -mc));
                const float z1 = fast_exp2(__builtin_fmaf(sc[e + 1], a.scale_log2, -mc));
                if (!ONES) {
                    l += z0;
                    l += z1;
                }
                p[e / 2] = pinned(__builtin_bit_cast(unsigned, typename T::v2{(typename T::el)z0, (typename T::el)z1}));
            }
            if (!ONES) l = pinned(l);
            if (j < 2 * DT) o[j % DT] = mfma_32x32x16(vf[j % 3].v, weights(pl, j / DT), o[j % DT]);
            if (ONES && HD > 16 && j < 2) lsum = mfma_32x32x16(ones, weights(pl, j), lsum);
            sched_fence();
        }
        __builtin_amdgcn_s_setprio(3);
        if (scale) {
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[d][e] *= f;
            if (ONES && HD > 16) lsum[0] *= f; /* every row holds the sum: one is kept up */
        }
    };

    const int ks_ = (int)a.k_token_stride, vs_ = (int)a.v_token_stride;
    int k0 = sink_tiles > 0 ? 0 : win0, k1 = step(0, k0), k2 = step(1, k1); /* of tiles t, t + 1, t + 2 */
    fetch(0, kb, ks_, koff, 0, k0);
    /* there is no part before the first: its weights are zero, and so is its V */
    for (int i = threadIdx.x; i < TILE / 16; i += NTHR) *reinterpret_cast<v8*>(lds + KRING + TILE + 16 * i) = v8{};
    vm_wait();
    /* the queries are in from here on: the compiler would wait for them, and the tiles on the way, in the loop */
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = opaque(qf[ks]);
    __syncthreads();
    fetch(TILE, kb, ks_, koff, 1, k1);
    fetch(KRING, vb, vs_, voff, 0, k0);
    f16v s0 = {}, s1 = {};
    unsigned p0[8] = {}, p1[8] = {};
    int last = 0, now0 = active(0, k0 + 32 * NP * kgroup);
    if (now0) {
#pragma unroll
        for (int j = 0; j < KS; ++j) s0 = mfma_32x32x16(read_k(0, j), qf[j], s0);
    }
    /* Tile t's V and tile t + 1's K have come to LDS at the barrier behind the tile's first body; the next V and
       the K after that go where the body before the barrier read last, or nobody for a tile. */
    auto pass = [&](int t, auto kbuf, auto knext, auto kfree, auto vbuf, auto vother) { /* places in the rings */
        const int at = k0 + 32 * NP * kgroup;
        int now1 = active(t, at + 32);
        const int next0 = active(t + 1, k1 + 32 * NP * kgroup);
        if (last | now0 | now1) {
            body(t, at, kbuf + 64 * HD, vother + (NP - 1) * 64 * HD, s0, s1, p0, p1);
        } else {
            none(p0);
        }
        vm_wait();
        __syncthreads();
        fetch(kfree, kb, ks_, koff, t + 2, k2);
        fetch(KRING + vother, vb, vs_, voff, t + 1, k1);
        check_v(vbuf, t, k0);
#pragma unroll
        for (int i = 1; i < NP; ++i) {
            const int now2 = i + 1 < NP ? active(t, at + 32 * (i + 1)) : next0;
            f16v &sc = i & 1 ? s1 : s0, &sn = i & 1 ? s0 : s1;
            unsigned(&p)[8] = i & 1 ? p1 : p0;
            if (now0 | now1 | now2) {
                body(t, at + 32 * i, i + 1 < NP ? kbuf + 64 * HD * (i + 1) : knext, vbuf + 64 * HD * (i - 1), sc, sn, p,
                     i & 1 ? p0 : p1);
            } else {
                none(p);
            }
            now0 = now1;
            now1 = now2;
        }
        last = now0;
        now0 = now1;
        k0 = k1;
        k1 = k2;
        k2 = step(t + 2, k2);
    };
    int vlast = 0; /* place of the last tile's V */
    if constexpr (KRING == 2 * TILE) { /* two tiles a turn: every LDS address a register of its own plus a constant */
        for (int t = 0; t < n_tiles; t += 2) {
            pass(t, 0, TILE, 0, 0, TILE);
            vlast = 0;
            if (t + 1 == n_tiles) break;
            pass(t + 1, TILE, 0, TILE, TILE, 0);
            vlast = TILE;
        }
    } else {
        for (int t = 0, k = 0; t < n_tiles; ++t) {
            const int knext = k + TILE < KRING ? k + TILE : 0, kfree = KRING - k - knext;
            vlast = (t & 1) * TILE;
            pass(t, k, knext, kfree, vlast, TILE - vlast);
            k = knext;
        }
    }
    if (last) { /* the last part's products */
        const int va = vlast + (NP - 1) * 64 * HD;
#pragma unroll
        for (int j = 0; j < 2 * DT; ++j) {
            VFrag vf;
            read_v(vf, va, j);
            o[j % DT] = mfma_32x32x16(vf.v, weights(p1, j / DT), o[j % DT]);
            if (ONES && HD > 16 && j % DT == 0) lsum = mfma_32x32x16(ones, weights(p1, j / DT), lsum);
        }
    }

    if (__syncthreads_or((bad & 0x80008000u) != 0)) {
        for (int r = 32 * wave + kgroup; r < 32 * wave + 32; r += KW) {
            const int i = q0 + r / a.tile_heads, head = hg * a.tile_heads + r % a.tile_heads;
            if (i >= q1) break;
            seq_attn_row<T, HD>(a, a.q + (rq.start + i) * a.q_token_stride + head * a.q_head_stride, kb, vb,
                                a.out + (rq.start + i) * a.out_token_stride + head * a.out_head_stride,
                                key_range(shift + i, nk, a.left, a.right, a.sinks));
        }
        return;
    }
    if constexpr (ONES) {
        l = HD == 16 ? o[0][8] : lsum[0];
    } else {
        float x, y;
        lanes_x32(l, x, y);
        l = x + y;
    }
    if constexpr (KW > 1) { /* the other groups' results through LDS (everyone is done with the tiles) */
        constexpr int ST = 64 * RW, PART = (16 * DT + 2) * ST;
        float* red = reinterpret_cast<float*>(lds) + (wave * 64 + lane);
        if (kgroup > 0) {
            float* mine = red + (kgroup - 1) * PART;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) mine[(16 * d + e) * ST] = o[d][e];
            mine[16 * DT * ST] = m == -INFINITY ? m : mc;
            mine[(16 * DT + 1) * ST] = l;
        }
        __syncthreads();
        if (kgroup > 0) return;
        float m0 = m == -INFINITY ? m : mc;
#pragma unroll
        for (int k = 0; k < KW - 1; ++k) {
            const float* other = red + k * PART;
            const float m1 = other[16 * DT * ST], top = vmax(m0, m1);
            const float f0 = m0 == -INFINITY ? 0.f : fast_exp2(m0 - top), f1 = m1 == -INFINITY ? 0.f : fast_exp2(m1 - top);
            l = l * f0 + other[(16 * DT + 1) * ST] * f1;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[d][e] = o[d][e] * f0 + other[(16 * d + e) * ST] * f1;
            m0 = top;
        }
    }
    const bool store = qrow < q1;
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    uint16_t* out = a.out + (rq.start + qi) * a.out_token_stride + h * a.out_head_stride;
    /* a lane has 4 channels of every 8; its partner 32 lanes on, the others: 8 and 8 after an exchange */
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 8) {
            if (32 * d + 2 * i >= HD) break;
            u4 r;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                unsigned w[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const float a0 = o[d][i + 4 * x + 2 * e], a1 = o[d][i + 4 * x + 2 * e + 1];
                    w[x] = __builtin_bit_cast(unsigned, typename T::v2{(typename T::el)opaque(a0 * inv), (typename T::el)opaque(a1 * inv)});
                }
                const auto sw = __builtin_amdgcn_permlane32_swap(w[0], w[1], false, false);
                r[e] = sw[0];
                r[2 + e] = sw[1];
            }
            if (store) *reinterpret_cast<u4*>(out + 32 * d + 2 * i + 8 * g) = r;
        }
}

/* Which of them: seq_rules.h's seq_plan. W4, W8: waves per SIMD that the registers have to allow. 8 waves with up to
 * 32 channels: two workgroups per CU (8,160 queries, 8 heads x 32, window 1,023: 30 us; one, 36). */
#define SEQ_ATTN(NAME, T, HD, W4, W8)                                                                                                    \
    extern "C" __global__ void __launch_bounds__(256, W4) prism_seq_attn_##NAME##_h##HD(SeqAttnArgs a) { seq_attn_body<T, HD, 4, 1>(a); } \
    extern "C" __global__ void __launch_bounds__(512, W8) prism_seq_attn_##NAME##_h##HD##_w8(SeqAttnArgs a) { seq_attn_body<T, HD, 4, 2>(a); }
#define SEQ_ATTN_NARROW(NAME, T, HD, W8) \
    extern "C" __global__ void __launch_bounds__(512, W8) prism_seq_attn_##NAME##_h##HD##_narrow(SeqAttnArgs a) { seq_attn_body<T, HD, 2, 4>(a); }
SEQ_ATTN(f16, F16, 16, 4, 4) SEQ_ATTN(f16, F16, 32, 3, 4) SEQ_ATTN(f16, F16, 64, 3, 2) SEQ_ATTN(f16, F16, 128, 2, 2)
SEQ_ATTN(bf16, BF16, 16, 4, 4) SEQ_ATTN(bf16, BF16, 32, 3, 4) SEQ_ATTN(bf16, BF16, 64, 3, 2) SEQ_ATTN(bf16, BF16, 128, 2, 2)
SEQ_ATTN_NARROW(f16, F16, 16, 4) SEQ_ATTN_NARROW(f16, F16, 32, 4) SEQ_ATTN_NARROW(f16, F16, 64, 2)
SEQ_ATTN_NARROW(bf16, BF16, 16, 4) SEQ_ATTN_NARROW(bf16, BF16, 32, 4) SEQ_ATTN_NARROW(bf16, BF16, 64, 2)
#undef SEQ_ATTN
#undef SEQ_ATTN_NARROW
