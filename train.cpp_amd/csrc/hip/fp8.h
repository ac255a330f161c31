// Matrices in 8-bit floating point (e4m3: sign, 4 bits of exponent, 3 of fraction, no infinities, largest
// value 448) with a scale for each block of 128: what the quantizer, the products and the single-token
// product share.
//
// A value is code x scale. Activations have a scale for each 128 neighbours of a row, a power
// of two held as its exponent's byte (127 added); weights one for each 128 x 128, such a byte or a float. A
// power of two costs an e4m3 value nothing but range (its spacing is relative), and makes quantizing exact but
// for the code's own rounding.
#pragma once

#include "common.h"

namespace trc_hip {
namespace {

constexpr int F8_BLOCK = 128;

typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));
typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));

// What a lane holds of a 16 x 128 operand: row lane % 16, the 16 bytes of chunk lane / 16 and those of chunk
// lane / 16 + 4 of the row's eight. Both operands hold the same k in the same place, and the order of a sum's
// terms is free, so this need not be the order in which the instructions count k.
union F8Frag {
    u4v half[2];
    u2v quarter[4];
};

// Eight codes in binary16, which holds every e4m3 value.
__device__ __forceinline__ h8v f8_half8(u2v c) {
    union {
        h2v h[4];
        h8v all;
    } o;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        o.h[2 * w] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[w], 1.f, false);
        o.h[2 * w + 1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[w], 1.f, true);
    }
    return o.all;
}
__device__ __forceinline__ float f8_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// A block's exponent byte from its largest finite magnitude: the smallest power of two by which it falls to 448 =
// 1.75 2^8 or less, 2^-126 at least; 1 for a block of zeros.
__device__ __forceinline__ uint32_t f8_exponent(float amax) {
    const uint32_t b = __builtin_bit_cast(uint32_t, amax);
    if (b == 0) return 127;
    const int e = (int) (b >> 23) - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return (uint32_t) (e < 1 ? 1 : e);
}
// 2^-(byte - 127)
__device__ __forceinline__ float f8_inverse(uint32_t byte) { return __builtin_bit_cast(float, (254u - byte) << 23); }
// a value that is not finite takes no part in its block's scale; its code is NaN
__device__ __forceinline__ float f8_finite(float a) { return a < INFINITY ? a : 0.f; }
// Eight values as codes, to nearest even. (What is not finite stays so times a power of two, and the conversion
// makes it NaN.)
__device__ __forceinline__ u2v f8_codes(const float (&x)[8], float inv) {
    u2v r;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * w] * inv, x[4 * w + 1] * inv, 0, false);
        c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * w + 2] * inv, x[4 * w + 3] * inv, c, true);
        r[w] = (uint32_t) c;
    }
    return r;
}

// Element types of activations and results.
typedef float f4a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t h8a2 __attribute__((ext_vector_type(8), aligned(2)));
__device__ __forceinline__ float f8_float(int type, uint16_t b) {
    return type == TRC_HIP_TYPE_F16 ? half_bits_to_float(b) : __builtin_bit_cast(float, (uint32_t) b << 16);
}
__device__ __forceinline__ uint16_t f8_bits(int type, float x) {
    return type == TRC_HIP_TYPE_F16 ? __builtin_bit_cast(uint16_t, (_Float16) x) : __builtin_bit_cast(uint16_t, (__bf16) x);
}
// Elements i .. i + 7 of a row of n (zeros past it), whose address is as aligned as an element.
template <int TYPE>
__device__ __forceinline__ void f8_load8(const uint8_t* row, int64_t i, int64_t n, float (&x)[8]) {
    if (i + 8 <= n) {
        if constexpr (TYPE == TRC_HIP_TYPE_F32) {
            const f4a4 a = *(const f4a4*) (row + 4 * i), b = *(const f4a4*) (row + 4 * i + 16);
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = a[k], x[4 + k] = b[k];
        } else {
            const h8a2 a = *(const h8a2*) (row + 2 * i);
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = f8_float(TYPE, a[k]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            x[k] = 0.f;
            if (i + k < n) {
                if constexpr (TYPE == TRC_HIP_TYPE_F32) x[k] = ((const float*) row)[i + k];
                else x[k] = f8_float(TYPE, ((const uint16_t*) row)[i + k]);
            }
        }
    }
}
__device__ __forceinline__ float f8_amax8(const float (&x)[8]) {
    float m = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = fmaxf(m, f8_finite(fabsf(x[k])));
    return m;
}
// the largest of a group of 16 lanes
__device__ __forceinline__ float f8_max16(float m) {
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    return m;
}

}  // namespace

// The products' arguments. The weight's rows are M, the codes' K columns; `out` is rows x N.
struct F8Args {
    const uint8_t* w;
    int64_t w_nb1;      // bytes from row to row, a multiple of 128
    int64_t K, M, N;
    const uint8_t* ws;  // the weight's scales
    int64_t ws_nb1;
    int ws_float;       // floats, or bytes
    const uint8_t* x;   // codes, rows of whole blocks
    int64_t x_nb1;
    const uint8_t* xs;
    int64_t xs_nb1;
    uint8_t* y;
    int64_t y_nb1;
    int y_type;
};
// fp8.hip: the quantizer; the products of few tokens that are still floats; those of up to 64 in 8 bits, without a
// workspace
int launch_f8_quantize(const trc_hip_tensor& x, const trc_hip_fp8& q, hipStream_t s);
int launch_f8_matvec(const F8Args& a, const trc_hip_tensor& x, hipStream_t s);
int launch_f8_skinny(const F8Args& a, hipStream_t s);
// fp8_mm.hip: W x, or W^T x with `back`, of operands in 8 bits. Up to 64 tokens the first f8_held bytes of the stream's
// workspace are left as they are.
int launch_f8_product(const F8Args& a, bool back, hipStream_t s);

constexpr int F8_FUSED = 2;  // most tokens whose activations a product's workgroups quantize for themselves
// bytes of the workspace with N tokens' codes and exponents
constexpr size_t f8_held(int64_t K, int64_t N) {
    const int64_t kb = (K + 127) / 128;
    return (size_t) (N * (kb * 128 + (kb + 3) / 4 * 4));
}

}  // namespace trc_hip
