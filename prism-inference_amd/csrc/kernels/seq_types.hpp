/*
 * seq_types.hpp - the element types of the sequence operators. Values are 16
 * bits, fp16 or bf16; every sum, softmax statistic and angle is fp32 or wider,
 * rounded once (to nearest, ties to even) at the store.
 */
#pragma once
#include "../seq_index.h"
#include "common.hpp"

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef unsigned int u4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));

struct F16 {
    typedef f16 el;
    typedef h8 v8;
    typedef h4 v4;
    typedef h2 v2;
};
struct BF16 {
    typedef __bf16 el;
    typedef b8 v8;
    typedef b4 v4;
    typedef b2 v2;
};

template <int N>
struct Count {
    static constexpr int value = N;
};

template <class T>
__device__ __forceinline__ typename T::v8 ld8(const uint16_t* p) {
    return *reinterpret_cast<const typename T::v8*>(p);
}
template <class T>
__device__ __forceinline__ void st8(uint16_t* p, typename T::v8 v) {
    *reinterpret_cast<typename T::v8*>(p) = v;
}
template <class T>
__device__ __forceinline__ float ld1(const uint16_t* p) {
    return (float)*reinterpret_cast<const typename T::el*>(p);
}
template <class T>
__device__ __forceinline__ void st1(uint16_t* p, float v) {
    *reinterpret_cast<typename T::el*>(p) = (typename T::el)opaque(v);
}

/* Sum over the 64 lanes; every lane gets the same bits. */
__device__ __forceinline__ float wave_sum(float v) { return sum_groups(group_sum<16>(v)); }

__device__ __forceinline__ f4 mfma_16x16x32(b8 a, b8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

/* Transposing LDS read: 16 lanes read 4 rows of 16 values (lane i: row i / 4,
 * values 4 (i % 4) ..+3) and lane i gets column i's 4 values. */
typedef short s4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ s4 lds_tr4(const void* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)p);
}
