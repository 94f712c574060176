/*
 * paged_attn4.hpp - attention of one new token per sequence over a paged cache
 * of 4 bits: paged_attn.hpp's formula, work and join; keys and values become 16-bit
 * numbers, exactly, on their way into the products (a conversion instruction makes two,
 * and takes the block's power of two along).
 *
 *   paged4_few   one or two heads a key head, 16 or 32 channels: a lane holds 8 or 16 channels of a key;
 *   paged4_many  S^T = K Q^T and O^T += V^T P^T on 16x16x32 MFMAs with the heads as columns. A lane
 *                takes a quarter of a key's row: the products only ask that queries' channels are in the
 *                same order. V goes through a wave's own LDS, as 16-bit numbers, for transposed reads.
 *
 * A key and a value are 17/16 of a byte a channel, a quarter of 16-bit ones, so that the vector units come close to memory:
 *   paged4_few   8,160 streams of 52 keys, 8 x 32: 32 us for 117 MB, vector units 96 % busy. One maximum for the wave: 40 us with one a lane,
 *                whose sums are scaled once more at the end.
 *   paged4_many  24 streams of 1,000 to 20,001, 32 over 8 x 128: 65 us for 276 MB (4.2 TB/s), its loads alone 53; one of 131,075: 34 for 143 MB.
 *                Keys through LDS in whole lines, and the next step's asked for ahead of the softmax, were slower or equal.
 */
#pragma once
#include "cache4.hpp"
#include "paged_work.hpp"

/* What a wave has to do, as paged_work, but with the splits of a length as long as those of the longest expected: workgroups are
 * alike, short sequences have fewer, and those without keys leave at once. */
__device__ __forceinline__ bool paged4_work(const PagedAttnArgs& a, int wave, PagedWork& w) {
    const unsigned items = (unsigned)a.n_seqs * a.n_kv_heads * a.head_tiles; /* 32 bits: a launch has fewer than 2^24 workgroups */
    unsigned item = blockIdx.x;
    int part = 0;
    w.split = 0;
    if (a.waves == 1) {
        item = item * 4 + wave;
    } else {
        const unsigned x = divide(item, a.splits, a.by_splits);
        w.split = (int)(item - x * a.splits);
        item = x;
        part = w.split * 4 + wave;
    }
    if (item >= items) return false;
    const unsigned both = divide(item, a.head_tiles, a.by_tiles);
    const int ht = (int)(item - both * a.head_tiles);
    w.seq = (int)divide(both, a.n_kv_heads, a.by_kv);
    w.hk = (int)(both - w.seq * a.n_kv_heads);
    w.head = w.hk * a.group + ht * PAGED_TILE_HEADS;
    w.heads = min(a.group - ht * PAGED_TILE_HEADS, PAGED_TILE_HEADS);
    const int n = seq_clamp(a.lengths[w.seq], 0, a.table_pages << a.page_log2);
    w.kr = key_range(n - 1, n, a.left, 0, a.sinks);
    const int seen = w.kr.sink + w.kr.hi - w.kr.lo;
    if (a.waves == 1) {
        w.i0 = 0;
        w.i1 = seen;
        return true;
    }
    const int parts = 4 * a.splits;
    int each = a.each;
    if ((int64_t)each * parts < seen) each = ((seen - 1) / parts + 16) & ~15; /* longer than expected */
    const int64_t at = (int64_t)part * each;
    w.i0 = at < seen ? (int)at : seen;
    w.i1 = seq_min(seen - w.i0, each) + w.i0;
    return true;
}

/* Key i of those that the wave sees, of which there are some: its table entry, past the end the last one's. A load for every lane, and
 * nothing that waits for it: the entries of several keys are asked for together. */
__device__ __forceinline__ int paged4_entry(const PagedAttnArgs& a, const PagedWork& w, int i) {
    const int32_t* row = a.table + (int64_t)w.seq * a.table_pages; /* of 2^30 entries at most: 32-bit offsets */
    const uint32_t page = (uint32_t)w.key(min(i, w.i1 - 1)) >> a.page_log2;
    return *reinterpret_cast<const int32_t*>(reinterpret_cast<const char*>(row) + 4 * page);
}
/* ... and where it lies, its slot's number in [page][head][slot]; a slot of the first page if it is not seen. */
struct Paged4Key {
    int64_t at;
    bool seen;
};
__device__ __forceinline__ Paged4Key paged4_key(const PagedAttnArgs& a, const PagedWork& w, int i, int entry) {
    const bool seen = i < w.i1 && page_ok(entry, a.n_pages);
    const int slot = w.key(min(i, w.i1 - 1)) & ((1 << a.page_log2) - 1);
    return Paged4Key{(int64_t)((((uint64_t)(uint32_t)(seen ? entry : 0) * (uint32_t)a.n_kv_heads + (uint32_t)w.hk) << a.page_log2) + (uint32_t)slot), seen};
}

template <class T, int HD, int G>
__device__ __forceinline__ void paged4_few(const PagedAttnArgs& a) {
    constexpr int CH = HD / 2 < 16 ? HD / 2 : 16; /* channels of a lane */
    constexpr int W = CH / 8;                     /* words of codes     */
    constexpr int LPK = HD / CH, KPS = 64 / LPK;  /* lanes a key, keys a step of the wave */
    constexpr int U = 2;                          /* steps in flight    */
    typedef typename T::v8 v8;
    __shared__ float lacc[4 * G * HD], lm[4 * G], ll[4 * G];
    const int lane = lane_id(), slot = lane / LPK, ch = lane % LPK * CH;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint8_t* kp = reinterpret_cast<const uint8_t*>(a.k_pages);
    const uint8_t* vp = reinterpret_cast<const uint8_t*>(a.v_pages);
    PagedWork w;
    if (!paged4_work(a, wave, w)) return; /* only where waves work alone */

    v8 q[G][W];
    float acc[G][CH] = {}, m[G], l[G];
#pragma unroll
    for (int h = 0; h < G; ++h) {
#pragma unroll
        for (int x = 0; x < W; ++x) q[h][x] = ld8<T>(a.q + w.seq * a.q_seq_stride + (w.head + h) * a.q_head_stride + ch + 8 * x);
        m[h] = -INFINITY;
        l[h] = 0.f;
    }
    const auto add = [](float x, float y) { return x + y; };
    const auto most = [](float x, float y) { return vmax(x, y); };
    const auto steps = [&](auto count, int i) {
        constexpr int U = decltype(count)::value;
        int entry[U];
        uint32_t k[U][W], v[U][W];
        uint8_t ks[U], vs[U];
        bool ok[U];
#pragma unroll
        for (int u = 0; u < U; ++u) entry[u] = paged4_entry(a, w, i + u * KPS + slot);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const Paged4Key key = paged4_key(a, w, i + u * KPS + slot, entry[u]);
            ok[u] = key.seen;
            __builtin_memcpy(k[u], kp + key.at * (HD / 2) + ch / 2, 4 * W);
            __builtin_memcpy(v[u], vp + key.at * (HD / 2) + ch / 2, 4 * W);
            ks[u] = a.k_scales[key.at];
            vs[u] = a.v_scales[key.at];
        }
        v8 kk[U][W];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int x = 0; x < W; ++x) kk[u][x] = fp4_values<T>(k[u][x], fp4_scale(ks[u]));
        float s[G][U];
#pragma unroll
        for (int h = 0; h < G; ++h) {
            float top = -INFINITY;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float d = 0.f;
#pragma unroll
                for (int x = 0; x < W; ++x) d = dot8(q[h][x], kk[u][x], d);
                if constexpr (LPK == 2) d = lanes_sum<2>(d);
                s[h][u] = ok[u] ? d * a.scale_log2 : -INFINITY;
                top = vmax(top, s[h][u]);
            }
            top = across<LPK>(top, most);
            if (__builtin_amdgcn_readfirstlane(top > m[h])) { /* the same for all lanes; not where a score is NaN: weights are then */
                if (i > w.i0) {
                    const float f = fast_exp2(m[h] - top);
                    l[h] *= f;
#pragma unroll
                    for (int e = 0; e < CH; ++e) acc[h][e] *= f;
                }
                m[h] = top;
            }
            const float mu = m[h] == -INFINITY ? 0.f : m[h];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                s[h][u] = fast_exp2(s[h][u] - mu);
                l[h] += s[h][u];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int x = 0; x < W; ++x) {
                const uint32_t word = v[u][x];
                const auto two = [&](auto byte) {
                    constexpr int B = decltype(byte)::value;
                    const f2 y = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, ok[u] ? fp4_scale(vs[u]) : 1.f, B);
#pragma unroll
                    for (int h = 0; h < G; ++h) {
                        acc[h][8 * x + 2 * B] = __builtin_fmaf(y[0], s[h][u], acc[h][8 * x + 2 * B]);
                        acc[h][8 * x + 2 * B + 1] = __builtin_fmaf(y[1], s[h][u], acc[h][8 * x + 2 * B + 1]);
                    }
                };
                two(Count<0>{});
                two(Count<1>{});
                two(Count<2>{});
                two(Count<3>{});
            }
    };
    int i = w.i0;
    for (; w.i1 - i > KPS; i += KPS * U) steps(Count<U>{}, i);
    if (i < w.i1) steps(Count<1>{}, i);
    /* The wave's 32 key slots together, halving what a lane holds: each step pairs lanes that differ in one bit, and one
       takes the sum of one half of the channels, the other of the other. In the end lane bits 5, 4, 3 (and 2) name a
       channel, bit 0 the lane's half of the row. */
    static_assert(LPK == 2, "lane bit 0: channels; 1 to 5: keys");
    const bool b3 = lane & 8, b2 = lane & 4;
    const int mine = (lane >> 5 & 1) * (CH / 2) + (lane >> 4 & 1) * (CH / 4) + (lane >> 3 & 1) * (CH / 8) + (CH == 16 ? lane >> 2 & 1 : 0);
#pragma unroll
    for (int h = 0; h < G; ++h) {
        l[h] = across<LPK>(l[h], add);
        float (&x)[CH] = acc[h];
#pragma unroll
        for (int e = 0; e < CH / 2; ++e) {
            const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x[e]), __builtin_bit_cast(unsigned, x[e + CH / 2]), false, false);
            x[e] = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
        }
#pragma unroll
        for (int e = 0; e < CH / 4; ++e) {
            const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x[e]), __builtin_bit_cast(unsigned, x[e + CH / 4]), false, false);
            x[e] = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
        }
#pragma unroll
        for (int e = 0; e < CH / 8; ++e) { /* row_ror 8 */
            const float keep = b3 ? x[e + CH / 8] : x[e], give = b3 ? x[e] : x[e + CH / 8];
            x[e] = keep + dpp<0x128>(give);
        }
        if constexpr (CH == 16) { /* quads mirrored in eights: lane ^ 7, and back within quads below */
            const float keep = b2 ? x[1] : x[0], give = b2 ? x[0] : x[1];
            const float there = dpp<0x1B>(give); /* quad_perm [3,2,1,0] */
            x[0] = keep + dpp<0x141>(there);     /* row_half_mirror: lane ^ 7; together lane ^ 4 */
        } else {
            x[0] += dpp<0x141>(dpp<0x1B>(x[0]));
        }
        x[0] += dpp<0x4E>(x[0]); /* lane ^ 2 */
    }
    const int c = ch + mine;
    if (a.waves == 1) {
        if ((lane & (CH == 16 ? 2 : 6)) == 0) {
#pragma unroll
            for (int h = 0; h < G; ++h)
                st1<T>(a.out + w.seq * a.out_seq_stride + (w.head + h) * a.out_head_stride + c, acc[h][0] * (l[h] == 0.f ? 0.f : 1.0f / l[h]));
        }
        return;
    }
#pragma unroll
    for (int h = 0; h < G; ++h) {
        if ((lane & (CH == 16 ? 2 : 6)) == 0) lacc[(wave * G + h) * HD + c] = acc[h][0];
        if (lane == 0) {
            lm[wave * G + h] = m[h];
            ll[wave * G + h] = l[h];
        }
    }
    __syncthreads();
    paged_join_waves<T, HD>(a, w, G, lacc, lm, ll, G);
}

template <class T, int HD>
__device__ __forceinline__ void paged4_many(const PagedAttnArgs& a) {
    typedef typename T::v8 v8;
    constexpr int KT = HD >= 128 ? 2 : 4, KEYS = 16 * KT; /* tiles of 16 keys a step */
    constexpr int KS = (HD + 31) / 32;                    /* k-steps of the scores (16 channels: half a step, zeros) */
    constexpr int QUARTER = HD >= 32 ? HD / 4 : 8;        /* channels of a lane (16: two lanes have them all) */
    constexpr int BL = KS;                                /* blocks of a row */
    constexpr int DT = HD / 16;                           /* 16-channel tiles of the output */
    constexpr int VROW = HD + (HD >= 32 ? 16 : 0);        /* LDS row (values): 8 rows of 32 bytes without conflicts */
    constexpr int VBYTES = 4 * KEYS * VROW * 2, ABYTES = 4 * PAGED_TILE_HEADS * HD * 4;
    __shared__ __attribute__((aligned(16))) uint8_t lds[VBYTES > ABYTES ? VBYTES : ABYTES];
    __shared__ float lm[4 * PAGED_TILE_HEADS], ll[4 * PAGED_TILE_HEADS];
    const int lane = lane_id(), l16 = lane & 15, g = lane >> 4, part = HD >= 32 ? g : g & 1;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint16_t* lv = reinterpret_cast<uint16_t*>(lds) + wave * KEYS * VROW; /* this wave's rows */
    const uint8_t* kp = reinterpret_cast<const uint8_t*>(a.k_pages) + part * (QUARTER / 2);
    const uint8_t* vp = reinterpret_cast<const uint8_t*>(a.v_pages) + part * (QUARTER / 2);
    const uint8_t* kx = a.k_scales + part * QUARTER / 32;
    const uint8_t* vx = a.v_scales + part * QUARTER / 32;
    PagedWork w;
    if (!paged4_work(a, wave, w)) return; /* only where waves work alone */

    v8 q[KS];
    const uint16_t* qp = a.q + w.seq * a.q_seq_stride + (w.head + min(l16, w.heads - 1)) * a.q_head_stride;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const v8 x = ld8<T>(qp + part * QUARTER + 8 * ks);
        q[ks] = HD >= 32 || g < 2 ? x : v8{};
    }
    /* Weights as the sum of two 16-bit numbers, as in paged_attn.hpp: what a matrix product takes. bf16's leave 2^-16 of a weight, so that some
       four outputs of a thousand round to the other side than with fp32 weights; the error against 64 bits is the same, the output's rounding. */
    constexpr bool HALF = __is_same(T, F16);
    constexpr float UP = HALF ? 15.f : 0.f, LEAST = HALF ? 0x1p-24f : 0x1p-133f; /* the type's smallest */
    f4 o[DT] = {};
    float m = -INFINITY, mu = 0.f, l = 0.f;

    const int key = lane & (KEYS - 1); /* a lane's of the step */
    int entry = w.i0 < w.i1 ? paged4_entry(a, w, w.i0 + key) : -1;
    for (int i = w.i0; i < w.i1; i += KEYS) {
        const Paged4Key own = paged4_key(a, w, i + key, entry);
        const uint64_t seen = __ballot(own.seen);
        /* every lane's own keys, l16 of each tile */
        int64_t at[KT];
        {
            const int64_t x = own.at;
            int lo[2], hi[2];
            lanes_x16((int)x, lo[0], lo[1]);
            lanes_x16((int)(x >> 32), hi[0], hi[1]);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if constexpr (KT == 2) {
                    at[t] = (int64_t)hi[t] << 32 | (uint32_t)lo[t];
                } else {
                    int l0, l1, h0, h1;
                    lanes_x32(lo[t], l0, l1);
                    lanes_x32(hi[t], h0, h1);
                    at[t] = (int64_t)h0 << 32 | (uint32_t)l0;
                    at[t + 2] = (int64_t)h1 << 32 | (uint32_t)l1;
                }
            }
        }
        uint32_t k[KT][KS], v[KT][KS];
        uint8_t ksc[KT], vsc[KT];
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            __builtin_memcpy(k[t], __builtin_assume_aligned(kp + at[t] * (HD / 2), QUARTER / 2), QUARTER / 2);
            ksc[t] = kx[at[t] * BL];
        }
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            __builtin_memcpy(v[t], __builtin_assume_aligned(vp + at[t] * (HD / 2), QUARTER / 2), QUARTER / 2);
            vsc[t] = vx[at[t] * BL];
        }
        entry = paged4_entry(a, w, i + KEYS + key);

        f4 s[KT] = {};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                v8 x = fp4_values<T>(k[t][ks], fp4_scale(ksc[t]));
                if (HD < 32 && g >= 2) x = v8{}; /* channels 16.. do not exist */
                s[t] = mfma_16x16x32(x, q[ks], s[t]);
            }
        const bool all = seen == ~0ull; /* two tiles: lanes 32.. have the same keys again */
        float top = m;
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (!all) s[t][e] = seen >> (16 * t + 4 * g + e) & 1 ? s[t][e] : -INFINITY;
                top = fmaxf(top, s[t][e]);
            }
        float x, y;
        lanes_x16(top, x, y);
        lanes_x32(fmaxf(x, y), x, y);
        top = fmaxf(x, y);
        if (__any(top > m)) {
            const float f = fast_exp2(m == -INFINITY ? -INFINITY : (m - top) * a.scale_log2);
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= f;
            m = top;
            mu = top == -INFINITY ? 0.f : top;
        }
        v8 p[KT / 2], rest[KT / 2];
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const float z0 = fast_exp2(__builtin_fmaf(s[t][e] - mu, a.scale_log2, UP));
                const float z1 = fast_exp2(__builtin_fmaf(s[t][e + 1] - mu, a.scale_log2, UP));
                l += z0;
                l += z1;
                typename T::v2 hi, lo;
                two_numbers(z0, z1, LEAST, hi, lo);
                p[t / 2][4 * (t & 1) + e] = hi[0];
                p[t / 2][4 * (t & 1) + e + 1] = hi[1];
                rest[t / 2][4 * (t & 1) + e] = lo[0];
                rest[t / 2][4 * (t & 1) + e + 1] = lo[1];
            }
        /* V into the wave's rows and back transposed. The LDS works a wave's accesses off in order; the
           fences keep the compiler from changing it. */
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            uint32_t word[KS];
            float scale = fp4_scale(vsc[t]);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) word[ks] = v[t][ks];
            if (!all && !(seen >> (16 * t + l16) & 1)) { /* zeros, not what may be NaN */
                scale = 1.f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) word[ks] = 0;
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                if (HD >= 32 || g < 2) st8<T>(lv + (16 * t + l16) * VROW + part * QUARTER + 8 * ks, fp4_values<T>(word[ks], scale));
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int n = 0; n < KT / 2; ++n)
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const uint16_t* from = lv + (32 * n + 4 * g + l16 / 4) * VROW + 16 * d + 4 * (l16 & 3);
                union {
                    s4 h[2];
                    v8 v;
                } vf;
                vf.h[0] = lds_tr4(from);
                vf.h[1] = lds_tr4(from + 16 * VROW);
                o[d] = mfma_16x16x32(vf.v, p[n], o[d]);
                o[d] = mfma_16x16x32(vf.v, rest[n], o[d]);
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    l = sum_groups(l);
    if (a.waves == 1) {
        if (l16 < w.heads) {
            const float inv = l == 0.f ? 0.f : 1.0f / l;
            uint16_t* out = a.out + w.seq * a.out_seq_stride + (w.head + l16) * a.out_head_stride + 4 * g;
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                typename T::v4 r;
#pragma unroll
                for (int e = 0; e < 4; ++e) r[e] = (typename T::el)opaque(o[d][e] * inv);
                *reinterpret_cast<typename T::v4*>(out + 16 * d) = r;
            }
        }
        return;
    }
    __syncthreads(); /* every wave is done with its V rows */
    float* acc = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int d = 0; d < DT; ++d)
        *reinterpret_cast<f4*>(acc + (wave * PAGED_TILE_HEADS + l16) * HD + 16 * d + 4 * g) = o[d];
    if (g == 0) {
        lm[wave * PAGED_TILE_HEADS + l16] = m * a.scale_log2;
        ll[wave * PAGED_TILE_HEADS + l16] = l;
    }
    __syncthreads();
    paged_join_waves<T, HD>(a, w, w.heads, acc, lm, ll, PAGED_TILE_HEADS);
}

/* The splits of one (sequence, head) together: their weights by the threads of the workgroup, then HD channels by
 * 256 / HD groups of splits. */
template <class T, int HD>
__device__ __forceinline__ void paged4_join(const PagedAttnArgs& a) {
    static_assert(PAGED4_MAX_SPLITS <= 256, "a thread per split");
    __shared__ float weight[256], part[256], tops[4], sums[4];
    const int tid = threadIdx.x, wave = tid >> 6;
    const float* ws = a.ws + (int64_t)blockIdx.x * a.splits * (HD + 2);
    const bool in = tid < a.splits;
    const float m = in ? ws[tid * (HD + 2) + HD] : -INFINITY, l = in ? ws[tid * (HD + 2) + HD + 1] : 0.f;
    float top = m;
    for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
    if (lane_id() == 0) tops[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    const float f = m == -INFINITY ? 0.f : fast_exp2(m - top);
    weight[tid] = f;
    const float mine = wave_sum(l * f);
    if (lane_id() == 0) sums[wave] = mine;
    __syncthreads();
    const float sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    const int c = tid % HD;
    float o = 0.f;
#pragma unroll 8 /* that many loads at once: the launch is as long as their latency */
    for (int s = tid / HD; s < a.splits; s += 256 / HD) o = __builtin_fmaf(ws[s * (HD + 2) + c], weight[s], o);
    part[tid] = o;
    __syncthreads();
    if (tid < HD) {
        o = 0.f;
#pragma unroll
        for (int k = 0; k < 256 / HD; ++k) o += part[k * HD + tid];
        const int seq = blockIdx.x / a.n_heads, head = blockIdx.x % a.n_heads;
        st1<T>(a.out + seq * a.out_seq_stride + head * a.out_head_stride + tid, sum == 0.f ? 0.f : o / sum);
    }
}

#define PAGED4(NAME, T, HD) \
    extern "C" __global__ void __launch_bounds__(256, 3) prism_paged_attn4_##NAME##_h##HD##_many(PagedAttnArgs a) { paged4_many<T, HD>(a); } \
    extern "C" __global__ void __launch_bounds__(256) prism_paged_attn4_join_##NAME##_h##HD(PagedAttnArgs a) { paged4_join<T, HD>(a); }
PAGED4(f16, F16, 16) PAGED4(f16, F16, 32) PAGED4(f16, F16, 64) PAGED4(f16, F16, 128)
PAGED4(bf16, BF16, 16) PAGED4(bf16, BF16, 32) PAGED4(bf16, BF16, 64) PAGED4(bf16, BF16, 128)
#undef PAGED4
#define PAGED4_FEW(NAME, T, HD) \
    extern "C" __global__ void __launch_bounds__(256) prism_paged_attn4_##NAME##_h##HD##_g1(PagedAttnArgs a) { paged4_few<T, HD, 1>(a); } \
    extern "C" __global__ void __launch_bounds__(256) prism_paged_attn4_##NAME##_h##HD##_g2(PagedAttnArgs a) { paged4_few<T, HD, 2>(a); }
PAGED4_FEW(f16, F16, 16) PAGED4_FEW(f16, F16, 32) PAGED4_FEW(bf16, BF16, 16) PAGED4_FEW(bf16, BF16, 32)
#undef PAGED4_FEW
