/*
 * paged_attn.hpp - attention of one new token per sequence over its paged cache.
 *
 * The token is the last of its sequence (position L - 1, L = lengths[s]); it
 * sees the `left` keys before it, itself and the first `sinks` ones:
 *   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c (q.k_j) - m),  c = scale log2 e
 * with a running maximum m, so the keys are read once: bound by HBM reads. Keys
 * of a page that the table does not name properly are not seen; values of keys
 * that are not seen are replaced by zeros before any product.
 *
 * An item is a sequence and the heads that share a key head (16 at most). Its
 * keys are dealt to `parts` waves: one, four of a workgroup, or four in each of
 * `splits` workgroups, whose results (maximum, sum, output) are joined in LDS
 * and, for splits, through the workspace by prism_paged_attn_join. The parts
 * follow from the length on the device; the host only chooses how many
 * (seq_rules.h).
 *
 * Two kernels by the heads of a group:
 *   paged_few   1 or 2: a lane holds 8 channels of a key; products are
 *               dot2 / FMA, scores meet over a key's HD / 8 lanes, and every key
 *               slot of the wave keeps a softmax of its own until the end;
 *   paged_many  more: S^T = K Q^T and O^T += V^T P^T on 16x16x32 MFMAs with the
 *               heads as columns, V through a wave's own LDS for transposed reads.
 */
#pragma once
#include "paged_work.hpp"

template <class T, int HD, int G>
__device__ __forceinline__ void paged_few(const PagedAttnArgs& a) {
    typedef typename T::v8 v8;
    constexpr int LPK = HD / 8;   /* lanes per key              */
    constexpr int KPS = 64 / LPK; /* keys per step of the wave  */
    constexpr int U = 4;          /* steps in flight            */
    __shared__ float lacc[4 * G * HD], lm[4 * G], ll[4 * G];
    const int lane = lane_id(), slot = lane / LPK, ch = lane % LPK * 8;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    PagedWork w;
    if (!paged_work(a, wave, w)) return; /* only where waves work alone */

    v8 q[G];
    float acc[G][8] = {}, m[G], l[G];
#pragma unroll
    for (int h = 0; h < G; ++h) {
        q[h] = ld8<T>(a.q + w.seq * a.q_seq_stride + (w.head + h) * a.q_head_stride + ch);
        m[h] = -INFINITY;
        l[h] = 0.f;
    }
    const auto steps = [&](auto count, int i) {
        constexpr int U = decltype(count)::value;
        int page[U];
        v8 k[U], v[U];
        bool ok[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int x = i + u * KPS + slot;
            page[u] = x < w.i1 ? paged_page(a, w, w.key(x)) : -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int x = i + u * KPS + slot;
            ok[u] = page[u] >= 0;
            const int64_t at = (ok[u] ? paged_at<HD>(a, w, page[u], w.key(x)) : 0) + ch;
            k[u] = ld8<T>(a.k_pages + at);
            v[u] = ld8<T>(a.v_pages + at);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = ok[u] ? v[u] : v8{};
#pragma unroll
        for (int h = 0; h < G; ++h) {
            float s[U], top = m[h];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                s[u] = lanes_sum<LPK>(dot8(q[h], k[u], 0.f)) * a.scale_log2;
                s[u] = ok[u] ? s[u] : -INFINITY;
                top = fmaxf(top, s[u]);
            }
            const float mu = top == -INFINITY ? 0.f : top;
            const float f = fast_exp2(m[h] - mu);
            l[h] *= f;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[h][e] *= f;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float p = fast_exp2(s[u] - mu);
                l[h] += p;
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[h][e] = __builtin_fmaf((float)v[u][e], p, acc[h][e]);
            }
            m[h] = top;
        }
    };
    /* the last keys, or few: without the loads of the steps behind them (8,160 sequences of 1 to 9 tokens, 8 heads x 32:
       40.7 -> 30.1 us) */
    for (int i = w.i0; i < w.i1; i += KPS * U)
        if (w.i1 - i > KPS) steps(Count<U>{}, i);
        else steps(Count<1>{}, i);
    /* the wave's key slots together */
    const auto add = [](float x, float y) { return x + y; };
    const auto most = [](float x, float y) { return fmaxf(x, y); };
#pragma unroll
    for (int h = 0; h < G; ++h) {
        const float top = across<LPK>(m[h], most);
        const float f = m[h] == -INFINITY ? 0.f : fast_exp2(m[h] - top);
        l[h] = across<LPK>(l[h] * f, add);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[h][e] = across<LPK>(acc[h][e] * f, add);
        m[h] = top;
    }
    if (a.waves == 1) {
        if (slot == 0) {
#pragma unroll
            for (int h = 0; h < G; ++h) {
                const float inv = l[h] == 0.f ? 0.f : 1.0f / l[h];
                v8 r;
#pragma unroll
                for (int e = 0; e < 8; ++e) r[e] = (typename T::el)opaque(acc[h][e] * inv);
                st8<T>(a.out + w.seq * a.out_seq_stride + (w.head + h) * a.out_head_stride + ch, r);
            }
        }
        return;
    }
    if (slot == 0) {
#pragma unroll
        for (int h = 0; h < G; ++h) {
#pragma unroll
            for (int e = 0; e < 8; ++e) lacc[(wave * G + h) * HD + ch + e] = acc[h][e];
            if (lane == 0) {
                lm[wave * G + h] = m[h];
                ll[wave * G + h] = l[h];
            }
        }
    }
    __syncthreads();
    paged_join_waves<T, HD>(a, w, G, lacc, lm, ll, G);
}

template <class T, int HD>
__device__ __forceinline__ void paged_many(const PagedAttnArgs& a) {
    typedef typename T::v8 v8;
    constexpr int KS = (HD + 31) / 32;             /* k-steps of the scores (16 channels: half a step, zeros) */
    constexpr int DT = HD / 16;                    /* 16-channel tiles of the output */
    constexpr int VROW = HD + (HD >= 32 ? 16 : 0); /* LDS row (values): 8 rows of 32 bytes without conflicts */
    constexpr int CPR = HD / 8, RPI = 64 / CPR, NV = 32 / RPI; /* V: chunks a row, rows a load, loads for 32 keys */
    constexpr int VBYTES = 4 * 32 * VROW * 2, ABYTES = 4 * PAGED_TILE_HEADS * HD * 4;
    __shared__ __attribute__((aligned(16))) uint8_t lds[VBYTES > ABYTES ? VBYTES : ABYTES];
    __shared__ float lm[4 * PAGED_TILE_HEADS], ll[4 * PAGED_TILE_HEADS];
    const int lane = lane_id(), l16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint16_t* lv = reinterpret_cast<uint16_t*>(lds) + wave * 32 * VROW; /* this wave's 32 rows */
    PagedWork w;
    if (!paged_work(a, wave, w)) return; /* only where waves work alone */

    v8 q[KS];
    const uint16_t* qp = a.q + w.seq * a.q_seq_stride + (w.head + min(l16, w.heads - 1)) * a.q_head_stride;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const bool in = HD >= 32 || g < 2;
        const v8 x = ld8<T>(qp + (in ? 32 * ks + 8 * g : 0));
        q[ks] = in ? x : v8{};
    }
    /* A weight meets V as the sum of two 16-bit numbers (2^-15 of it off at most, where the output is rounded by 2^-8; fp16
       2^-20), fp16's from 2^15 down, so what is lost is below 2^-39 of the largest: many keys behind one strong key may matter.
       The first is cut off and the second held above zero, so an infinite V meets no zero beside a weight and no other
       sign. The outputs' errors are those of paged_few, which has 32-bit weights; rounded to one 16-bit number they were 1.3
       times as large. us with one number and with two: 24 sequences to 20,001, 32/8 x 128: 207.8, 208.9; one of 131,075: 108.2, 108.8; 64 to 1,000, 32/8 x 64:
       21.3, 21.6; 34, 40/8 x 16, window 2,820: 22.1, 24.1. */
    constexpr bool HALF = __is_same(T, F16);
    constexpr float UP = HALF ? 15.f : 0.f, LEAST = HALF ? 0x1p-24f : 0x1p-133f; /* the type's smallest */
    f4 o[DT] = {};
    float m = -INFINITY, mu = 0.f, l = 0.f; /* mu = m, or 0 while m is -inf; l as the weights, 2^UP times too large */

    const auto page_of = [&](int i) { /* lane's key of the 32 from i on */
        const int x = i + (lane & 31);
        return x < w.i1 ? paged_page(a, w, w.key(x)) : -1;
    };
    int page = w.i0 < w.i1 ? page_of(w.i0) : -1;
    for (int i = w.i0; i < w.i1; i += 32) {
        const unsigned seen = (unsigned)__ballot(page >= 0);
        v8 k[2][KS], v[NV];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int r = 16 * t + l16, p = __shfl(page, r);
            const int64_t at = p >= 0 ? paged_at<HD>(a, w, p, w.key(i + r)) : 0;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) k[t][ks] = ld8<T>(a.k_pages + at + (HD >= 32 ? 32 * ks + 8 * g : 8 * (g & 1)));
        }
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int r = n * RPI + lane / CPR, p = __shfl(page, r);
            const int64_t at = p >= 0 ? paged_at<HD>(a, w, p, w.key(i + r)) : 0;
            v[n] = ld8<T>(a.v_pages + at + lane % CPR * 8);
        }
        const int next = i + 32 < w.i1 ? page_of(i + 32) : -1;

        f4 s[2] = {};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if (HD < 32 && g >= 2) k[t][ks] = v8{}; /* channels 16.. do not exist */
                s[t] = mfma_16x16x32(k[t][ks], q[ks], s[t]);
            }
        float top = m;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (seen != 0xFFFFFFFFu) s[t][e] = seen >> (16 * t + 4 * g + e) & 1 ? s[t][e] : -INFINITY;
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
        /* The maximum is subtracted before the scaling: the largest weight is then 2^UP whatever the scores, where an FMA with
           the rounded product c m leaves half a step of it, 2^64 at scores of 2^30. */
        v8 p, rest;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const float z0 = fast_exp2(__builtin_fmaf(s[t][e] - mu, a.scale_log2, UP));
                const float z1 = fast_exp2(__builtin_fmaf(s[t][e + 1] - mu, a.scale_log2, UP));
                l += z0;
                l += z1;
                typename T::v2 hi, lo;
                two_numbers(z0, z1, LEAST, hi, lo);
                p[4 * t + e] = hi[0];
                p[4 * t + e + 1] = hi[1];
                rest[4 * t + e] = lo[0];
                rest[4 * t + e + 1] = lo[1];
            }
        /* V into the wave's rows and back transposed. The LDS works a wave's accesses off in order; the
           fences keep the compiler from changing it. */
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int r = n * RPI + lane / CPR;
            st8<T>(lv + r * VROW + lane % CPR * 8, seen >> r & 1 ? v[n] : v8{});
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const uint16_t* at = lv + (4 * g + l16 / 4) * VROW + 16 * d + 4 * (l16 & 3);
            union {
                s4 h[2];
                v8 v;
            } vf;
            vf.h[0] = lds_tr4(at);
            vf.h[1] = lds_tr4(at + 16 * VROW);
            o[d] = mfma_16x16x32(vf.v, p, o[d]);
            o[d] = mfma_16x16x32(vf.v, rest, o[d]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        page = next;
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
__device__ __forceinline__ void paged_join(const PagedAttnArgs& a) {
    static_assert(PAGED_MAX_SPLITS == 64, "a lane per split");
    __shared__ float weight[PAGED_MAX_SPLITS], part[256], total;
    const int tid = threadIdx.x;
    const float* ws = a.ws + (int64_t)blockIdx.x * a.splits * (HD + 2);
    const bool in = tid < a.splits; /* all in the first wave */
    const float m = in ? ws[tid * (HD + 2) + HD] : -INFINITY, l = in ? ws[tid * (HD + 2) + HD + 1] : 0.f;
    if (tid < 64) {
        float top = m;
        for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
        const float f = m == -INFINITY ? 0.f : fast_exp2(m - top);
        weight[tid] = f;
        const float sum = wave_sum(l * f);
        if (tid == 0) total = sum;
    }
    __syncthreads();
    const float sum = total;
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

#define PAGED_ATTN(NAME, T, HD)                                                                                             \
    extern "C" __global__ void __launch_bounds__(256) prism_paged_attn_##NAME##_h##HD##_g1(PagedAttnArgs a) { paged_few<T, HD, 1>(a); } \
    extern "C" __global__ void __launch_bounds__(256) prism_paged_attn_##NAME##_h##HD##_g2(PagedAttnArgs a) { paged_few<T, HD, 2>(a); } \
    extern "C" __global__ void __launch_bounds__(256, 3) prism_paged_attn_##NAME##_h##HD##_many(PagedAttnArgs a) { paged_many<T, HD>(a); } \
    extern "C" __global__ void __launch_bounds__(256) prism_paged_attn_join_##NAME##_h##HD(PagedAttnArgs a) { paged_join<T, HD>(a); }
PAGED_ATTN(f16, F16, 16) PAGED_ATTN(f16, F16, 32) PAGED_ATTN(f16, F16, 64) PAGED_ATTN(f16, F16, 128)
PAGED_ATTN(bf16, BF16, 16) PAGED_ATTN(bf16, BF16, 32) PAGED_ATTN(bf16, BF16, 64) PAGED_ATTN(bf16, BF16, 128)
#undef PAGED_ATTN
