// 8-bit floating point with a scale for each block of 128: the quantizer, and the product for up to 64 tokens.
//
//   e = the smallest exponent with amax_block 2^-e <= 448      code = e4m3(x 2^-e)
//   y[m,n] = sum_b ws[m/128,b] 2^e[n,b] sum_{k in block b} w[m,k] x[n,k]
#include "fp8.h"

namespace trc_hip {

namespace {

constexpr int Q_THREADS = 256;

// Rows. A wave takes four blocks of a row: 16 lanes each, 8 elements a lane, and writes their exponents as one word.
// Bound by memory. UNITS such pieces of a wave are under way together.
template <int TYPE, int UNITS>
__global__ __launch_bounds__(Q_THREADS) void k_f8_rows(const uint8_t* __restrict__ x, size_t x_nb1, int64_t K, int64_t units,
                                                        FastDiv groups, uint8_t* __restrict__ q, size_t q_nb1,
                                                        uint8_t* __restrict__ sc, size_t sc_nb1) {
    const int lane = (int) threadIdx.x & 63;
    const int64_t u0 = ((int64_t) blockIdx.x * (Q_THREADS / 64) + (threadIdx.x >> 6)) * UNITS;
    float v[UNITS][8];
    uint32_t row[UNITS], g[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const uint32_t unit = (uint32_t) min(u0 + u, units - 1);  // (a piece may be done twice, with the same result)
        row[u] = div_by(unit, groups);
        g[u] = unit - row[u] * groups.d;
        f8_load8<TYPE>(x + row[u] * x_nb1, (int64_t) g[u] * 512 + lane * 8, K, v[u]);
    }
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const uint32_t e = f8_exponent(f8_max16(f8_amax8(v[u])));
        const int64_t at = (int64_t) g[u] * 512 + lane * 8;
        if (at / F8_BLOCK * F8_BLOCK < K) *(u2v*) (q + row[u] * q_nb1 + at) = f8_codes(v[u], f8_inverse(e));
        const uint32_t word = __builtin_amdgcn_readlane(e, 0) | __builtin_amdgcn_readlane(e, 16) << 8 |
                              __builtin_amdgcn_readlane(e, 32) << 16 | __builtin_amdgcn_readlane(e, 48) << 24;
        if (lane == 0) *(uint32_t*) (sc + row[u] * sc_nb1 + 4 * g[u]) = word;
    }
}

// Blocks of 128 x 128: a workgroup holds one in registers.
template <int TYPE>
__global__ __launch_bounds__(Q_THREADS) void k_f8_blocks(const uint8_t* __restrict__ x, size_t x_nb1, int64_t K, int64_t R,
                                                          uint32_t kb, uint8_t* __restrict__ q, size_t q_nb1,
                                                          uint8_t* __restrict__ sc, size_t sc_nb1) {
    const uint32_t bj = blockIdx.x / kb, bi = blockIdx.x - bj * kb;
    const int64_t at = (int64_t) bi * F8_BLOCK + (threadIdx.x & 15) * 8, row0 = (int64_t) bj * F8_BLOCK + (threadIdx.x >> 4);
    float v[8][8], m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t row = row0 + 16 * i;
        f8_load8<TYPE>(x + min(row, R - 1) * x_nb1, at, row < R ? K : 0, v[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, f8_amax8(v[i]));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    __shared__ float w[Q_THREADS / 64];
    if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]));
    const uint32_t e = f8_exponent(m);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t row = row0 + 16 * i;
        if (row < R) *(u2v*) (q + row * q_nb1 + at) = f8_codes(v[i], f8_inverse(e));
    }
    if (threadIdx.x == 0) sc[bj * sc_nb1 + bi] = (uint8_t) e;
}

constexpr int SK_WAVES = 8;
constexpr int SK_FUSED = 4;             // tokens whose activations a wave quantizes for itself
constexpr int SK_PITCH = 512 + 16;      // of their codes in LDS: 8 rows' 16 bytes fall on different banks
constexpr uint32_t SK_RSRC = 0x00027000;

// Up to 16 NT tokens: a workgroup takes 16 of the weight's rows, its waves share K out in groups of four blocks and
// join their sums in LDS. The weight goes from memory to registers; bound by its bytes, of which as many are under way as
// waves fit a CU: they are held to few registers, operands turned to binary16 a quarter at a time.
// FUSED: x holds floats (of type XTYPE), and every wave quantizes what it multiplies: N <= SK_FUSED.
template <int NT, int XTYPE>
__global__ __launch_bounds__(SK_WAVES * 64, NT == 1 ? 6 : 4) void k_f8_skinny(F8Args a, const uint8_t* __restrict__ xf, size_t xf_nb1) {
    constexpr bool FUSED = XTYPE >= 0;
    const int lane = (int) threadIdx.x & 63, wave = (int) threadIdx.x >> 6, waves = (int) blockDim.x >> 6;
    const int r16 = lane & 15, chunk = lane >> 4;
    const int64_t row0 = (int64_t) blockIdx.x * 16;
    const int kb = (int) ((a.K + F8_BLOCK - 1) / F8_BLOCK), groups = (kb + 3) / 4;
    const int rows = (int) min((int64_t) 16, a.M - row0);
    const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(
        (void*) (a.w + row0 * a.w_nb1), (short) 0, (int) ((rows - 1) * a.w_nb1 + (int64_t) kb * F8_BLOCK), SK_RSRC);
    const uint32_t w_off = (uint32_t) (r16 * a.w_nb1) + chunk * 16;
    const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(
        (void*) a.x, (short) 0, FUSED ? 0 : (int) ((a.N - 1) * a.x_nb1 + (int64_t) kb * F8_BLOCK), SK_RSRC);
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        (void*) a.xs, (short) 0, FUSED ? 0 : (int) ((a.N - 1) * a.xs_nb1 + (int64_t) groups * 4), SK_RSRC);
    __shared__ __attribute__((aligned(16))) uint8_t codes[FUSED ? SK_WAVES * SK_FUSED * SK_PITCH : 16];
    __shared__ uint32_t words[FUSED ? SK_WAVES * SK_FUSED : 1];
    __shared__ __attribute__((aligned(16))) float red[SK_WAVES * 16 * NT * 16];
    const uint8_t* const wsr = a.ws + (row0 / F8_BLOCK) * a.ws_nb1;

    f4 acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = {0.f, 0.f, 0.f, 0.f};
    for (int g = wave; g < groups; g += waves) {
        F8Frag w[4];
        float ws[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            // (past K the last block again, which is not used)
            const int at = min(4 * g + b, kb - 1);
            w[b].half[0] = __builtin_bit_cast(u4v, __builtin_amdgcn_raw_buffer_load_b128(rw, w_off, (uint32_t) at * F8_BLOCK, 0));
            w[b].half[1] = __builtin_bit_cast(u4v, __builtin_amdgcn_raw_buffer_load_b128(rw, w_off + 64, (uint32_t) at * F8_BLOCK, 0));
            ws[b] = a.ws_float ? ((const float*) wsr)[at] : f8_scale(wsr[at]);
        }
        uint32_t scale[NT];
        if constexpr (FUSED) {
            uint8_t* const mine = codes + wave * SK_FUSED * SK_PITCH;
            for (int t = 0; t < a.N; ++t) {
                float v[8];
                f8_load8<XTYPE>(xf + t * xf_nb1, (int64_t) g * 512 + lane * 8, a.K, v);
                const uint32_t e = f8_exponent(f8_max16(f8_amax8(v)));
                *(u2v*) (mine + t * SK_PITCH + lane * 8) = f8_codes(v, f8_inverse(e));
                if (r16 == 0) ((uint8_t*) (words + wave * SK_FUSED + t))[chunk] = (uint8_t) e;
            }
            // a wave's own LDS accesses are carried out in their order
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            scale[0] = words[wave * SK_FUSED + min(r16, (int) a.N - 1)];
        } else {
#pragma unroll
            for (int j = 0; j < NT; ++j)
                scale[j] = __builtin_amdgcn_raw_buffer_load_b32(rs, (uint32_t) ((16 * j + r16) * a.xs_nb1) + 4 * g, 0, 0);
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            if (4 * g + b >= kb) break;
            F8Frag x[NT];
            f4 part[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                if constexpr (FUSED) {
                    const uint8_t* const p = codes + (wave * SK_FUSED + min(r16, (int) a.N - 1)) * SK_PITCH + b * F8_BLOCK + chunk * 16;
                    x[j].half[0] = *(const u4v*) p;
                    x[j].half[1] = *(const u4v*) (p + 64);
                } else {
                    const uint32_t at = (uint32_t) ((16 * j + r16) * a.x_nb1) + (4 * g + b) * F8_BLOCK + chunk * 16;
                    x[j].half[0] = __builtin_bit_cast(u4v, __builtin_amdgcn_raw_buffer_load_b128(rx, at, 0, 0));
                    x[j].half[1] = __builtin_bit_cast(u4v, __builtin_amdgcn_raw_buffer_load_b128(rx, at + 64, 0, 0));
                }
                part[j] = {0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const h8v wq = f8_half8(w[b].quarter[q]);
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    part[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wq, f8_half8(x[j].quarter[q]), part[j], 0, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const float s = f8_scale((scale[j] >> (8 * b)) & 255u);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[j][i] = fmaf(part[j][i] * s, ws[b], acc[j][i]);
            }
        }
        if constexpr (FUSED) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) *(f4*) (red + ((wave * NT + j) * 16 + r16) * 16 + chunk * 4) = acc[j];
    __syncthreads();
    for (int e = (int) threadIdx.x; e < 256 * NT; e += (int) blockDim.x) {
        const int token = e >> 4, r = e & 15;
        if (token >= a.N || r >= rows) continue;
        float s = 0.f;
        for (int w = 0; w < waves; ++w) s += red[w * NT * 256 + e];
        uint8_t* const y = a.y + token * a.y_nb1;
        if (a.y_type == TRC_HIP_TYPE_F32) ((float*) y)[row0 + r] = s;
        else ((uint16_t*) y)[row0 + r] = f8_bits(a.y_type, s);
    }
}

template <int TYPE>
int rows_of(const trc_hip_tensor& x, const trc_hip_fp8& q, hipStream_t s) {
    const int64_t K = x.ne[0], R = x.ne[1], groups = (K + 4 * F8_BLOCK - 1) / (4 * F8_BLOCK), units = R * groups;
    // four pieces a wave from 16 waves a SIMD on
    const int n = units >= (int64_t) device_cus() * 64 * 4 ? 4 : 1;
    const int64_t per = (Q_THREADS / 64) * n, wgs = (units + per - 1) / per;
    hipLaunchKernelGGL(n == 4 ? (k_f8_rows<TYPE, 4>) : (k_f8_rows<TYPE, 1>), dim3((unsigned) wgs), dim3(Q_THREADS), 0, s,
                       (const uint8_t*) x.data, x.nb[1], K, units, fast_div(groups), (uint8_t*) q.q.data, q.q.nb[1],
                       (uint8_t*) q.scale.data, q.scale.nb[1]);
    return check_launch("fp8_quantize");
}

template <int TYPE>
int blocks_of(const trc_hip_tensor& x, const trc_hip_fp8& q, hipStream_t s) {
    const int64_t K = x.ne[0], R = x.ne[1], kb = (K + F8_BLOCK - 1) / F8_BLOCK, rb = (R + F8_BLOCK - 1) / F8_BLOCK;
    hipLaunchKernelGGL(k_f8_blocks<TYPE>, dim3((unsigned) (kb * rb)), dim3(Q_THREADS), 0, s, (const uint8_t*) x.data, x.nb[1], K, R,
                       (uint32_t) kb, (uint8_t*) q.q.data, q.q.nb[1], (uint8_t*) q.scale.data, q.scale.nb[1]);
    return check_launch("fp8_quantize (blocks)");
}

template <int XTYPE>
int skinny(const F8Args& a, const uint8_t* xf, size_t xf_nb1, hipStream_t s) {
    const int64_t wgs = (a.M + 15) / 16, groups = (a.K + 4 * F8_BLOCK - 1) / (4 * F8_BLOCK);
    const unsigned threads = 64 * (unsigned) (groups < SK_WAVES ? groups : SK_WAVES);
    auto* k = k_f8_skinny<1, XTYPE>;
    if constexpr (XTYPE < 0) {
        if (a.N > 16) k = a.N <= 32 ? k_f8_skinny<2, -1> : a.N <= 48 ? k_f8_skinny<3, -1> : k_f8_skinny<4, -1>;
    }
    hipLaunchKernelGGL(k, dim3((unsigned) wgs), dim3(threads), 0, s, a, xf, xf_nb1);
    return check_launch("fp8 (few tokens)");
}

}  // namespace

int launch_f8_quantize(const trc_hip_tensor& x, const trc_hip_fp8& q, hipStream_t s) {
    const bool rows = q.scale.ne[1] == x.ne[1];
    if (x.type == TRC_HIP_TYPE_F32) return rows ? rows_of<TRC_HIP_TYPE_F32>(x, q, s) : blocks_of<TRC_HIP_TYPE_F32>(x, q, s);
    if (x.type == TRC_HIP_TYPE_F16) return rows ? rows_of<TRC_HIP_TYPE_F16>(x, q, s) : blocks_of<TRC_HIP_TYPE_F16>(x, q, s);
    return rows ? rows_of<TRC_HIP_TYPE_BF16>(x, q, s) : blocks_of<TRC_HIP_TYPE_BF16>(x, q, s);
}

// x: activations to be quantized on the way, or null where a holds codes.
int launch_f8_skinny(const F8Args& a, const trc_hip_tensor* x, hipStream_t s) {
    if (x == nullptr) return skinny<-1>(a, nullptr, 0, s);
    if (a.N <= SK_FUSED) {
        const uint8_t* const p = (const uint8_t*) x->data;
        if (x->type == TRC_HIP_TYPE_F32) return skinny<TRC_HIP_TYPE_F32>(a, p, x->nb[1], s);
        if (x->type == TRC_HIP_TYPE_F16) return skinny<TRC_HIP_TYPE_F16>(a, p, x->nb[1], s);
        return skinny<TRC_HIP_TYPE_BF16>(a, p, x->nb[1], s);
    }
    // codes and exponents in the stream's workspace
    const int64_t kb = (a.K + F8_BLOCK - 1) / F8_BLOCK, pitch = kb * F8_BLOCK, words = (kb + 3) / 4 * 4;
    if ((size_t) (a.N * (pitch + words)) > qm_workspace_bytes()) {
        return fail(TRC_HIP_E_SHAPE, "trc_hip_fp8_matvec: %lld tokens of %lld do not fit the workspace", (long long) a.N,
                    (long long) a.K);
    }
    uint8_t* wsp = nullptr;
    int rc = qm_stream_workspace(s, &wsp);
    if (rc != TRC_HIP_OK) return rc;
    trc_hip_fp8 q{};
    q.q.data = wsp;
    q.q.nb[1] = (size_t) pitch;
    q.scale.data = wsp + a.N * pitch;
    q.scale.nb[1] = (size_t) words;
    q.scale.ne[1] = a.N;
    rc = launch_f8_quantize(*x, q, s);
    if (rc != TRC_HIP_OK) return rc;
    F8Args b = a;
    b.x = wsp;
    b.x_nb1 = pitch;
    b.xs = wsp + a.N * pitch;
    b.xs_nb1 = words;
    return skinny<-1>(b, nullptr, 0, s);
}

}  // namespace trc_hip
