/*
 * paged_attn4.hpp - attention of one new token per sequence over a paged cache
 * of 4 bits: paged_attn.hpp's formula, work and join; keys and values become 16-bit
 * numbers, exactly, on their way into the products.
 */
#pragma once
#include "cache4.hpp"
#include "paged_work.hpp"

template <class T, int HD>
__device__ __forceinline__ void paged4_many(const PagedAttnArgs& a) {
    typedef typename T::v8 v8;
    constexpr int KS = (HD + 31) / 32;             /* k-steps of the scores (16 channels: half a step, zeros) */
    constexpr int BL = KS;                         /* blocks of a row */
    constexpr int DT = HD / 16;                    /* 16-channel tiles of the output */
    constexpr int VROW = HD + (HD >= 32 ? 16 : 0); /* LDS row (values) */
    constexpr int CPR = HD / 8, RPI = 64 / CPR, NV = 32 / RPI; /* V: chunks a row, rows a load, loads for 32 keys */
    constexpr int VBYTES = 4 * 32 * VROW * 2, ABYTES = 4 * PAGED_TILE_HEADS * HD * 4;
    __shared__ __attribute__((aligned(16))) uint8_t lds[VBYTES > ABYTES ? VBYTES : ABYTES];
    __shared__ float lm[4 * PAGED_TILE_HEADS], ll[4 * PAGED_TILE_HEADS];
    const int lane = lane_id(), l16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint16_t* lv = reinterpret_cast<uint16_t*>(lds) + wave * 32 * VROW; /* this wave's 32 rows */
    const uint8_t* kp = reinterpret_cast<const uint8_t*>(a.k_pages);
    const uint8_t* vp = reinterpret_cast<const uint8_t*>(a.v_pages);
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
    /* weights as the sum of two 16-bit numbers, as in paged_attn.hpp */
    constexpr bool HALF = __is_same(T, F16);
    constexpr float UP = HALF ? 15.f : 0.f, LEAST = HALF ? 0x1p-24f : 0x1p-133f; /* the type's smallest */
    f4 o[DT] = {};
    float m = -INFINITY, mu = 0.f, l = 0.f;

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
            const int64_t at = p >= 0 ? paged_at<1>(a, w, p, w.key(i + r)) : 0;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                k[t][ks] = fp4_values<T>(*reinterpret_cast<const uint32_t*>(kp + at * (HD / 2) + (HD >= 32 ? 16 * ks + 4 * g : 4 * (g & 1))),
                                         fp4_scale(a.k_scales[at * BL + ks]));
        }
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int r = n * RPI + lane / CPR, p = __shfl(page, r), c = lane % CPR;
            const int64_t at = p >= 0 ? paged_at<1>(a, w, p, w.key(i + r)) : 0;
            v[n] = fp4_values<T>(*reinterpret_cast<const uint32_t*>(vp + at * (HD / 2) + 4 * c), fp4_scale(a.v_scales[at * BL + c / 4]));
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
                s[t][e] = seen >> (16 * t + 4 * g + e) & 1 ? s[t][e] : -INFINITY;
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

#define PAGED4(NAME, T, HD) \
    extern "C" __global__ void __launch_bounds__(256, 3) prism_paged_attn4_##NAME##_h##HD##_many(PagedAttnArgs a) { paged4_many<T, HD>(a); }
PAGED4(f16, F16, 16) PAGED4(f16, F16, 32) PAGED4(f16, F16, 64) PAGED4(f16, F16, 128)
PAGED4(bf16, BF16, 16) PAGED4(bf16, BF16, 32) PAGED4(bf16, BF16, 64) PAGED4(bf16, BF16, 128)
#undef PAGED4
