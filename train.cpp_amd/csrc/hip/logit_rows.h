// Rows of logits in F32, F16 or BF16 as the losses read and write them: 16 bytes at a time.
#pragma once

#include "common.h"

namespace trc_hip {
namespace {

// 16 bytes of a row whose address is only as aligned as one element
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t h8u __attribute__((ext_vector_type(8), aligned(2)));

template <int TYPE>
struct Row;
template <>
struct Row<TRC_HIP_TYPE_F32> {
    typedef float Elem;
    static constexpr int VEC = 4;
    static __device__ __forceinline__ float get(float x) { return x; }
    static __device__ __forceinline__ float put(float x) { return x; }
    static __device__ __forceinline__ void load(const Elem* p, float* x) {
        const f4u v = *(const f4u*) p;
#pragma unroll
        for (int k = 0; k < VEC; ++k) x[k] = v[k];
    }
    static __device__ __forceinline__ void store(Elem* p, const float* x) {
        f4u v;
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = x[k];
        __builtin_nontemporal_store(v, (f4u*) p);
    }
};
template <int TYPE>
struct Row16 {
    typedef uint16_t Elem;
    static constexpr int VEC = 8;
    static __device__ __forceinline__ float get(uint16_t x) {
        return TYPE == TRC_HIP_TYPE_F16 ? half_bits_to_float(x) : __builtin_bit_cast(float, (uint32_t) x << 16);
    }
    // rounded to nearest, once, from 32 bits
    static __device__ __forceinline__ uint16_t put(float x) {
        if (TYPE == TRC_HIP_TYPE_F16) return __builtin_bit_cast(uint16_t, (_Float16) x);
        return __builtin_bit_cast(uint16_t, (__bf16) x);
    }
    static __device__ __forceinline__ void load(const Elem* p, float* x) {
        const h8u v = *(const h8u*) p;
#pragma unroll
        for (int k = 0; k < VEC; ++k) x[k] = get(v[k]);
    }
    static __device__ __forceinline__ void store(Elem* p, const float* x) {
        h8u v;
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = put(x[k]);
        __builtin_nontemporal_store(v, (h8u*) p);
    }
};
template <>
struct Row<TRC_HIP_TYPE_F16> : Row16<TRC_HIP_TYPE_F16> {};
template <>
struct Row<TRC_HIP_TYPE_BF16> : Row16<TRC_HIP_TYPE_BF16> {};

}  // namespace
}  // namespace trc_hip
