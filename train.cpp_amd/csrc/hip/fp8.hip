// 8-bit floating point with a scale for each block of 128: the quantizer, and the product for up to 64 tokens.
//
//   e = the smallest exponent with amax_block 2^-e <= 448      code = e4m3(x 2^-e)
//   y[m,n] = sum_b ws[m/128,b] 2^e[n,b] sum_{k in block b} w[m,k] x[n,k]
#include "fp8.h"

namespace trc_hip {

namespace {

constexpr int Q_THREADS = 256;

// Rows. A wave takes four blocks of a row: 16 lanes each, 8 elements a lane, and writes their exponents as one word.
// Bound by memory: 4096 x 4096 of bfloat16 10 us (4.9 TB/s), 14336 x 8192 64 (5.5). Two or four such pieces a wave, their loads
// under way together, were slower (13 and 16 us where one took 12, 71 and 95 where it took 65): fewer waves hide less.
template <int TYPE>
__global__ __launch_bounds__(Q_THREADS) void k_f8_rows(const uint8_t* __restrict__ x, size_t x_nb1, int64_t K, int64_t units,
                                                        FastDiv groups, uint8_t* __restrict__ q, size_t q_nb1,
                                                        uint8_t* __restrict__ sc, size_t sc_nb1) {
    const int lane = (int) threadIdx.x & 63;
    // (the last piece may be done more than once, with the same result)
    const uint32_t unit = (uint32_t) min((int64_t) blockIdx.x * (Q_THREADS / 64) + (threadIdx.x >> 6), units - 1);
    const uint32_t row = div_by(unit, groups), g = unit - row * groups.d;
    const int64_t at = (int64_t) g * 512 + lane * 8;
    float v[8];
    f8_load8<TYPE>(x + row * x_nb1, at, K, v);
    const uint32_t e = f8_exponent(f8_max16(f8_amax8(v)));
    if (at / F8_BLOCK * F8_BLOCK < K) *(u2v*) (q + row * q_nb1 + at) = f8_codes(v, f8_inverse(e));
    const uint32_t word = __builtin_amdgcn_readlane(e, 0) | __builtin_amdgcn_readlane(e, 16) << 8 |
                          __builtin_amdgcn_readlane(e, 32) << 16 | __builtin_amdgcn_readlane(e, 48) << 24;
    if (lane == 0) *(uint32_t*) (sc + row * sc_nb1 + 4 * g) = word;
}

// Blocks of 128 x 128: a workgroup holds one in registers, so that the matrix is read once; one a workgroup keeps every CU
// busy from 4 M elements on. Bound by memory: 4096 x 4096 of bfloat16 11 us (4.6 TB/s), 14336 x 8192 70 (5.0), of floats 102 (5.7);
// smaller ones have few workgroups (1999 x 2050: 272, 7.6 us where rows take 4.7).
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

constexpr int SK_WAVES = 16;            // most of a workgroup
constexpr int SK_LDS = 48 * 1024;       // most bytes of tokens that it holds (with its waves' sums two workgroups fit a CU)
constexpr uint32_t SK_RSRC = 0x00027000;

// The 16 rows of the weight that a workgroup takes, as its waves read them: groups of four blocks of K in turn, from memory to
// registers.
struct SkWeight {
    const F8Args& a;
    const int lane, wave, waves;
    const int kb, groups;
    __device__ __forceinline__ explicit SkWeight(const F8Args& args)
        : a(args), lane((int) threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6)),
          waves((int) blockDim.x >> 6), kb((int) ((args.K + F8_BLOCK - 1) / F8_BLOCK)), groups((kb + 3) / 4) {}
    // (rows past the weight are read as zeros; past K the last block again, which is not used)
    __device__ __forceinline__ void load(int64_t tile, int g, F8Frag (&w)[4]) const {
        const int64_t row0 = tile * 16;
        const int64_t rows = min((int64_t) 16, a.M - row0);
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
            (void*) (a.w + row0 * a.w_nb1), (short) 0, (int) ((rows - 1) * a.w_nb1 + (int64_t) kb * F8_BLOCK), SK_RSRC);
        const uint32_t off = (uint32_t) ((lane & 15) * a.w_nb1) + (lane >> 4) * 16;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const uint32_t at = (uint32_t) min(4 * g + b, kb - 1) * F8_BLOCK;
            w[b].half[0] = __builtin_bit_cast(u4v, __builtin_amdgcn_raw_buffer_load_b128(r, off, at, 0));
            w[b].half[1] = __builtin_bit_cast(u4v, __builtin_amdgcn_raw_buffer_load_b128(r, off + 64, at, 0));
        }
    }
    // a group's scales, by the scalar unit (a byte within its word; a vector load would wait for the weight's before it)
    __device__ __forceinline__ void scales(int64_t tile, int g, float (&s)[4]) const {
        typedef const __attribute__((address_space(4))) uint32_t scalar_word;
        const uint64_t row = (uint64_t) (a.ws + tile / 8 * a.ws_nb1);
        if (a.ws_float) {
#pragma unroll
            for (int b = 0; b < 4; ++b) s[b] = __builtin_bit_cast(float, ((scalar_word*) row)[min(4 * g + b, kb - 1)]);
        } else {
            const uint32_t word = ((scalar_word*) row)[g];
#pragma unroll
            for (int b = 0; b < 4; ++b) s[b] = f8_scale(word >> (8 * b) & 255u);
        }
    }
};

// A block's products of one fragment of the weight with NT of tokens, added to acc.
template <int NT>
__device__ __forceinline__ void sk_block(const F8Frag& w, float ws, const F8Frag (&x)[NT], const float (&xs)[NT], f4 (&acc)[NT]) {
    f4 part[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) part[j] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const h8v h = f8_half8(w.quarter[q]);
#pragma unroll
        for (int j = 0; j < NT; ++j) part[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h, f8_half8(x[j].quarter[q]), part[j], 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = fmaf(part[j][i], xs[j] * ws, acc[j][i]);
}

// The waves' sums of a tile, joined in their order and stored.
template <int NT>
__device__ __forceinline__ void sk_store(const SkWeight& w, int64_t tile, const f4 (&acc)[NT], float* red) {
    const int r16 = w.lane & 15, chunk = w.lane >> 4;
#pragma unroll
    for (int j = 0; j < NT; ++j) *(f4*) (red + ((w.wave * NT + j) * 16 + r16) * 16 + chunk * 4) = acc[j];
    // (a bare barrier: loads from memory stay under way)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    for (int e = (int) threadIdx.x; e < 256 * NT; e += (int) blockDim.x) {
        const int token = e >> 4;
        const int64_t r = tile * 16 + (e & 15);
        if (token >= w.a.N || r >= w.a.M) continue;
        float s = 0.f;
        for (int k = 0; k < w.waves; ++k) s += red[k * NT * 256 + e];
        uint8_t* const y = w.a.y + token * w.a.y_nb1;
        if (w.a.y_type == TRC_HIP_TYPE_F32) ((float*) y)[r] = s;
        else ((uint16_t*) y)[r] = f8_bits(w.a.y_type, s);
    }
}

// N tokens, up to F8_FUSED, whose activations are still floats (of type XTYPE): every wave first quantizes what it will
// multiply, into LDS, while its first weights come. DEEP: several groups a wave, two of them under way in turn; else one, in as
// few registers as let four workgroups share a CU (of two tokens three). A workgroup a tile: fewer that take several each were slower
// (14336 rows of 4096: 16.4 us, 15.4 so), what is under way from the start counts for more. Bound by the weight's way from
// memory: 14336 rows of 4096 for one token 13.5 us (4.4 TB/s with the launch), products in binary16 as they need nothing else.
template <int N, int XTYPE, bool DEEP>
__global__ __launch_bounds__(DEEP ? SK_WAVES * 64 : 512, DEEP ? 4 : 6) void k_f8_few(F8Args a, const uint8_t* __restrict__ xf, size_t xf_nb1) {
    extern __shared__ __attribute__((aligned(16))) uint8_t codes[];  // tokens' rows, then their exponents' words
    __shared__ __attribute__((aligned(16))) float red[(DEEP ? SK_WAVES : 8) * 256];
    const SkWeight w(a);
    const int lane = w.lane, r16 = lane & 15, chunk = lane >> 4;
    const int pitch = w.groups * 512 + 16;
    uint32_t* const words = (uint32_t*) (codes + N * pitch);
    auto load_x = [&](int g, float (&x)[N][8]) {
#pragma unroll
        for (int t = 0; t < N; ++t) f8_load8<XTYPE>(xf + t * xf_nb1, (int64_t) g * 512 + lane * 8, a.K, x[t]);
    };
    // (the activations before the weight: loads arrive in their order)
    float v[N][8];
    load_x(w.wave, v);
    struct Group {
        F8Frag w[4];
        float scale[4];
    } even, odd;
    auto load_w = [&](int g, Group& into) {
        w.load(blockIdx.x, g, into.w);
        w.scales(blockIdx.x, g, into.scale);
    };
    load_w(w.wave, even);
    if (DEEP && w.wave + w.waves < w.groups) load_w(w.wave + w.waves, odd);
    for (int g = w.wave; g < w.groups; g += w.waves) {
#pragma unroll
        for (int t = 0; t < N; ++t) {
            const uint32_t e = f8_exponent(f8_max16(f8_amax8(v[t])));
            *(u2v*) (codes + t * pitch + g * 512 + lane * 8) = f8_codes(v[t], f8_inverse(e));
            if (r16 == 0) ((uint8_t*) (words + t * w.groups + g))[chunk] = (uint8_t) e;
        }
        if (!DEEP) break;
        if (g + w.waves < w.groups) load_x(g + w.waves, v);
    }
    // a wave's own LDS accesses are carried out in their order
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int token = min(r16, N - 1);
    f4 acc[1] = {{0.f, 0.f, 0.f, 0.f}};
    auto multiply = [&](int g, const Group& f) {
        const uint32_t word = words[token * w.groups + g];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            if (4 * g + b >= w.kb) break;
            F8Frag x[1];
            const uint8_t* const p = codes + token * pitch + g * 512 + b * F8_BLOCK + chunk * 16;
            x[0].half[0] = *(const u4v*) p;
            x[0].half[1] = *(const u4v*) (p + 64);
            const float xs[1] = {f8_scale(word >> (8 * b) & 255u)};
            sk_block<1>(f.w[b], f.scale[b], x, xs, acc);
        }
    };
    if (!DEEP) {
        multiply(w.wave, even);
    } else {
        for (int g = w.wave; g < w.groups; g += 2 * w.waves) {
            multiply(g, even);
            if (g + 2 * w.waves < w.groups) load_w(g + 2 * w.waves, even);
            if (g + w.waves >= w.groups) break;
            multiply(g + w.waves, odd);
            if (g + 3 * w.waves < w.groups) load_w(g + 3 * w.waves, odd);
        }
    }
    sk_store<1>(w, blockIdx.x, acc, red);
}

// Up to 16 NT tokens in 8 bits: a workgroup a tile, a wave a group of four blocks of K at a time, so that few tokens and
// rows fill the chip. Bound by memory at 16 tokens (4096 rows of 4096: 7.2 us), then by every workgroup's reading all
// tokens from the L2 (64 tokens: 13.7).
template <int NT>
__global__ __launch_bounds__(SK_WAVES * 64, 4) void k_f8_skinny(F8Args a) {
    __shared__ __attribute__((aligned(16))) float red[SK_WAVES * 256 * NT];
    const SkWeight w(a);
    const int r16 = w.lane & 15, chunk = w.lane >> 4;
    const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(
        (void*) a.x, (short) 0, (int) ((a.N - 1) * a.x_nb1 + (int64_t) w.kb * F8_BLOCK), SK_RSRC);
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        (void*) a.xs, (short) 0, (int) ((a.N - 1) * a.xs_nb1 + (int64_t) w.groups * 4), SK_RSRC);
    const int64_t tile = blockIdx.x;
    f4 acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = {0.f, 0.f, 0.f, 0.f};
    for (int g = w.wave; g < w.groups; g += w.waves) {
        auto token = [&](int b, int j) {
            F8Frag x;
            const uint32_t at = (uint32_t) ((16 * j + r16) * a.x_nb1) + min(4 * g + b, w.kb - 1) * F8_BLOCK + chunk * 16;
            x.half[0] = __builtin_bit_cast(u4v, __builtin_amdgcn_raw_buffer_load_b128(rx, at, 0, 0));
            x.half[1] = __builtin_bit_cast(u4v, __builtin_amdgcn_raw_buffer_load_b128(rx, at + 64, 0, 0));
            return x;
        };
        // (the tokens before the weight: loads arrive in their order)
        uint32_t words[NT];
        F8Frag x[NT], now[4];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            words[j] = __builtin_amdgcn_raw_buffer_load_b32(rs, (uint32_t) ((16 * j + r16) * a.xs_nb1) + 4 * g, 0, 0);
            x[j] = token(0, j);
        }
        w.load(tile, g, now);
        float ws[4];
        w.scales(tile, g, ws);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            if (4 * g + b >= w.kb) break;
            F8Frag more[NT];
            float xs[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                if (b < 3) more[j] = token(b + 1, j);
                xs[j] = f8_scale(words[j] >> (8 * b) & 255u);
            }
            sk_block<NT>(now[b], ws[b], x, xs, acc);
#pragma unroll
            for (int j = 0; j < NT; ++j) x[j] = more[j];
        }
    }
    sk_store<NT>(w, tile, acc, red);
}

template <int TYPE>
int rows_of(const trc_hip_tensor& x, const trc_hip_fp8& q, hipStream_t s) {
    const int64_t K = x.ne[0], R = x.ne[1], groups = (K + 4 * F8_BLOCK - 1) / (4 * F8_BLOCK), units = R * groups;
    hipLaunchKernelGGL(k_f8_rows<TYPE>, dim3((unsigned) ((units + Q_THREADS / 64 - 1) / (Q_THREADS / 64))), dim3(Q_THREADS), 0, s,
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

int64_t sk_groups(int64_t K) { return (K + 4 * F8_BLOCK - 1) / (4 * F8_BLOCK); }
// A wave a group up to 8, then two each: the same in both kernels, so that their sums are.
unsigned sk_threads(int64_t K) {
    const int64_t groups = sk_groups(K), waves = groups <= 8 ? groups : (groups + 1) / 2;
    return 64 * (unsigned) (waves < SK_WAVES ? waves : SK_WAVES);
}
size_t few_bytes(int64_t K, int64_t N) {
    return (size_t) (N * (sk_groups(K) * 516 + 16));
}
template <int XTYPE>
int few(const F8Args& a, const trc_hip_tensor& x, hipStream_t s) {
    static_assert(F8_FUSED == 2, "a kernel for each");
    const bool deep = sk_groups(a.K) > 8;
    auto* const k = a.N == 1 ? (deep ? k_f8_few<1, XTYPE, true> : k_f8_few<1, XTYPE, false>)
                             : (deep ? k_f8_few<2, XTYPE, true> : k_f8_few<2, XTYPE, false>);
    hipLaunchKernelGGL(k, dim3((unsigned) ((a.M + 15) / 16)), dim3(sk_threads(a.K)), few_bytes(a.K, a.N), s, a,
                       (const uint8_t*) x.data, x.nb[1]);
    return check_launch("fp8 (few tokens)");
}

}  // namespace

int launch_f8_quantize(const trc_hip_tensor& x, const trc_hip_fp8& q, hipStream_t s) {
    const bool rows = q.scale.ne[1] == x.ne[1];
    if (x.type == TRC_HIP_TYPE_F32) return rows ? rows_of<TRC_HIP_TYPE_F32>(x, q, s) : blocks_of<TRC_HIP_TYPE_F32>(x, q, s);
    if (x.type == TRC_HIP_TYPE_F16) return rows ? rows_of<TRC_HIP_TYPE_F16>(x, q, s) : blocks_of<TRC_HIP_TYPE_F16>(x, q, s);
    return rows ? rows_of<TRC_HIP_TYPE_BF16>(x, q, s) : blocks_of<TRC_HIP_TYPE_BF16>(x, q, s);
}

int launch_f8_skinny(const F8Args& a, hipStream_t s) {
    auto* const k = a.N <= 16 ? k_f8_skinny<1> : a.N <= 32 ? k_f8_skinny<2> : a.N <= 48 ? k_f8_skinny<3> : k_f8_skinny<4>;
    hipLaunchKernelGGL(k, dim3((unsigned) ((a.M + 15) / 16)), dim3(sk_threads(a.K)), 0, s, a);
    return check_launch("fp8 (few tokens)");
}

int launch_f8_matvec(const F8Args& a, const trc_hip_tensor& x, hipStream_t s) {
    if (a.N <= F8_FUSED && few_bytes(a.K, a.N) <= SK_LDS) {
        if (x.type == TRC_HIP_TYPE_F32) return few<TRC_HIP_TYPE_F32>(a, x, s);
        return x.type == TRC_HIP_TYPE_F16 ? few<TRC_HIP_TYPE_F16>(a, x, s) : few<TRC_HIP_TYPE_BF16>(a, x, s);
    }
    // codes and exponents in the stream's workspace
    const int64_t kb = (a.K + F8_BLOCK - 1) / F8_BLOCK, pitch = kb * F8_BLOCK, words = (kb + 3) / 4 * 4;
    if (f8_held(a.K, a.N) > qm_workspace_bytes()) {
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
    rc = launch_f8_quantize(x, q, s);
    if (rc != TRC_HIP_OK) return rc;
    F8Args b = a;
    b.x = wsp;
    b.x_nb1 = pitch;
    b.xs = wsp + a.N * pitch;
    b.xs_nb1 = words;
    return launch_f8_product(b, false, s);
}

}  // namespace trc_hip
