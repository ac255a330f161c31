// The products with an 8-bit weight for many tokens: tiles on the matrix cores (see fp8_mm.hip).
#pragma once

#include "fp8.h"

namespace trc_hip {

struct F8Tiles {
    F8Args a;
    int64_t rows;       // of the result: M, or K on the way back
    int steps;          // blocks of 128 summed over
    int part_steps;     // of one part of the sum, a multiple of 4 where there are several
    int tm, tn;         // tiles along rows and tokens
    float* sums;        // several parts: their sums, [part][token][rows]; else null
    int64_t sums_nb1;   // floats from token to token
};

// FAST: the 8-bit matrix instruction, or binary16 with sums in 32 bits (fp8_mm.hip says when). POW2: the weight's
// scales are bytes.
template <int BM, int BN, int WM, int WN, bool TRANS, bool FAST, bool POW2>
void f8_tiles_launch(const F8Tiles& t, unsigned parts, hipStream_t s);

namespace {

constexpr uint32_t F8_RSRC = 0x00027000;

typedef __attribute__((address_space(3))) uint8_t lds_byte;
typedef int i2v __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i2v lds_i2v;

// 16-byte chunks of a tile's row in LDS lie at slots chunk ^ f8_turn(row), so that eight rows' reads fall on
// different banks. CH: chunks of a row.
template <int CH>
__device__ __forceinline__ int f8_turn(int row) {
    return CH == 4 ? (row >> 1) & 3 : row & 7;
}

// One operand's tile of a step, ROWS rows of 16 CH bytes, from memory to LDS without a way through registers: piece
// p of a thread lands 16 THREADS bytes after piece p - 1, and the slots' turn is in the address it is read from.
template <int ROWS, int CH, int THREADS>
struct F8Slab {
    static constexpr int PIECES = ROWS * CH / THREADS, PER = THREADS / CH;  // rows of a piece
    static constexpr int BYTES = ROWS * CH * 16;
    static_assert(PIECES * THREADS == ROWS * CH && PER % 8 == 0, "whole pieces, the same turn in each");
    uint32_t off;
    __device__ __forceinline__ F8Slab(int tid, int64_t nb1) {
        const int row = tid / CH, slot = tid % CH;
        off = (uint32_t) (row * nb1) + (uint32_t) (slot ^ f8_turn<CH>(row)) * 16;
    }
    __device__ __forceinline__ void load(const uint8_t* base, int64_t bytes, int64_t nb1, lds_byte* lds, int wave) const {
        const __amdgpu_buffer_rsrc_t r =
            __builtin_amdgcn_make_buffer_rsrc((void*) base, (short) 0, (int) (uint32_t) bytes, F8_RSRC);
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*) (lds + (p * THREADS + wave * 64) * 16), 16, off,
                                                     (uint32_t) (p * PER * nb1), 0, 0);
    }
};

template <int BM, int BN, int WM, int WN, bool TRANS, bool FAST, bool POW2>
__global__ __launch_bounds__(WM * WN * 64, 2) void k_f8_tiles(F8Tiles t) {
    constexpr int THREADS = WM * WN * 64, TM = BM / WM, TN = BN / WN, IT = TM / 16, JT = TN / 16;
    constexpr int ACH = TRANS ? BM / 16 : 8;
    static_assert(TM <= F8_BLOCK && F8_BLOCK % TM == 0, "a wave's rows share their scales");
    typedef F8Slab<TRANS ? F8_BLOCK : BM, ACH, THREADS> ASlab;
    typedef F8Slab<BN, 8, THREADS> BSlab;
    __shared__ __attribute__((aligned(128))) uint8_t lds_all[2 * (ASlab::BYTES + BSlab::BYTES)];
    lds_byte* const lds = (lds_byte*) lds_all;

    const int per_xcd = (t.tm * t.tn + 7) / 8;
    const int tile = (int) (blockIdx.x & 7) * per_xcd + (int) (blockIdx.x >> 3);
    if (tile >= t.tm * t.tn) return;
    // four tiles of rows by all of the tokens', then the next four: neighbours on an XCD share operands in its L2
    const int in = tile % (4 * t.tn), first = tile / (4 * t.tn) * 4, high = min(4, t.tm - first);
    const int64_t row0 = (int64_t) (first + in % high) * BM, n0 = (int64_t) (in / high) * BN;

    const int tid = (int) threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WM, wn = wave / WM, r16 = lane & 15, chunk = lane >> 4;
    const F8Args& a = t.a;
    const int s0 = (int) blockIdx.y * t.part_steps, s1 = min(s0 + t.part_steps, t.steps);

    const ASlab slab_a(tid, a.w_nb1);
    const BSlab slab_b(tid, a.x_nb1);
    const int64_t pitch = (a.K + F8_BLOCK - 1) / F8_BLOCK * F8_BLOCK;
    const int64_t a_rows = min((int64_t) BM, a.M - row0), b_rows = min((int64_t) BN, a.N - n0);
    const uint8_t* const x0 = a.x + n0 * a.x_nb1;
    // rows past an operand are read as zeros (on the way back: the weight's last rows of a step)
    auto load = [&](int s, int buf) {
        lds_byte* const at = lds + buf * (ASlab::BYTES + BSlab::BYTES);
        if constexpr (TRANS) {
            const int64_t left = min((int64_t) F8_BLOCK, a.M - (int64_t) s * F8_BLOCK);
            slab_a.load(a.w + (int64_t) s * F8_BLOCK * a.w_nb1 + row0, (left - 1) * a.w_nb1 + pitch - row0, a.w_nb1, at, wave);
        } else {
            slab_a.load(a.w + row0 * a.w_nb1 + (int64_t) s * F8_BLOCK, (a_rows - 1) * a.w_nb1 + F8_BLOCK, a.w_nb1, at, wave);
        }
        slab_b.load(x0 + (int64_t) s * F8_BLOCK, (b_rows - 1) * a.x_nb1 + F8_BLOCK, a.x_nb1, at + ASlab::BYTES, wave);
    };
    // the tokens' exponents, four steps in a word
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        (void*) (a.xs + n0 * a.xs_nb1), (short) 0, (int) ((b_rows - 1) * a.xs_nb1 + (t.steps + 3) / 4 * 4), F8_RSRC);
    uint32_t exps[JT], more[JT];
    auto load_exps = [&](int s) {
#pragma unroll
        for (int j = 0; j < JT; ++j)
            more[j] = __builtin_amdgcn_raw_buffer_load_b32(rs, (uint32_t) ((wn * TN + j * 16 + r16) * a.xs_nb1) + s, 0, 0);
    };
    // the weight's scale of a step
    const int64_t rb = min((row0 + wm * TM) / F8_BLOCK, (t.rows - 1) / F8_BLOCK);
    const uint8_t* ws = a.ws + (TRANS ? rb * (POW2 ? 1 : 4) : rb * a.ws_nb1);
    const int64_t ws_step = TRANS ? a.ws_nb1 : (POW2 ? 1 : 4);

    f4 acc[IT][JT];
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int j = 0; j < JT; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

    // (loaded a step ahead and taken after the wait below, so that the loads to LDS are waited for there only)
    uint32_t wbits, wnext = 0;
    auto load_ws = [&](int s) {
        if constexpr (POW2) wnext = ws[s * ws_step];
        else wnext = *(const uint32_t*) (ws + s * ws_step);
    };
    if (s0 < s1) {
        load_exps(s0);
        load_ws(s0);
        load(s0, 0);
    }
    for (int s = s0; s < s1; ++s) {
        // this step's tiles have landed, and every wave has read the last one's
        __builtin_amdgcn_s_waitcnt(0);
        __builtin_amdgcn_s_barrier();
        const int buf = (s - s0) & 1;
        if ((s & 3) == 0 || s == s0) {
#pragma unroll
            for (int j = 0; j < JT; ++j) exps[j] = more[j] >> (8 * (s & 3));
            if ((s | 3) + 1 < s1) load_exps((s | 3) + 1);
        } else {
#pragma unroll
            for (int j = 0; j < JT; ++j) exps[j] >>= 8;
        }
        wbits = wnext;
        if (s + 1 < s1) {
            load_ws(s + 1);
            load(s + 1, buf ^ 1);
        }

        const lds_byte* const la = lds + buf * (ASlab::BYTES + BSlab::BYTES);
        const lds_byte* const lb = la + ASlab::BYTES;
        auto read = [&](const lds_byte* base, int row) {
            F8Frag f;
            const lds_byte* const p = base + row * 128;
            f.half[0] = *(const __attribute__((address_space(3))) u4v*) (p + ((chunk ^ f8_turn<8>(row)) * 16));
            f.half[1] = *(const __attribute__((address_space(3))) u4v*) (p + (((chunk + 4) ^ f8_turn<8>(row)) * 16));
            return f;
        };
        // The weight turned: eight of its rows by 16 of its columns at a time. Lane l of 16 gives the address of half
        // a row and gets a column.
        auto read_turned = [&](int col) {
            F8Frag f;
            const int half = r16 >> 1;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int m = 16 * chunk + 8 * (q & 1) + 64 * (q >> 1) + half;
                const lds_byte* const p = la + m * BM + (((col >> 4) ^ f8_turn<ACH>(m)) * 16) + (r16 & 1) * 8;
                f.quarter[q] = __builtin_bit_cast(u2v, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i2v*) p));
            }
            return f;
        };
        if constexpr (FAST) {
            F8Frag b[JT];
#pragma unroll
            for (int j = 0; j < JT; ++j) b[j] = read(lb, wn * TN + j * 16 + r16);
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                F8Frag f;
                if constexpr (TRANS) f = read_turned(wm * TM + i * 16);
                else f = read(la, wm * TM + i * 16 + r16);
#pragma unroll
                for (int j = 0; j < JT; ++j) {
                    if constexpr (POW2) {
                        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(f.all, b[j].all, acc[i][j], 0, 0, 0, (int) wbits, 0,
                                                                                    (int) exps[j]);
                    } else {
                        const f4 zero = {0.f, 0.f, 0.f, 0.f};
                        const f4 part =
                            __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(f.all, b[j].all, zero, 0, 0, 0, 127, 0, (int) exps[j]);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            acc[i][j][k] = fmaf(part[k], __builtin_bit_cast(float, wbits), acc[i][j][k]);
                    }
                }
            }
        } else {
            const float wscale = POW2 ? f8_scale(wbits) : __builtin_bit_cast(float, wbits);
#pragma unroll
            for (int j = 0; j < JT; ++j) {
                const F8Half b(read(lb, wn * TN + j * 16 + r16));
                const float scale = f8_scale(exps[j] & 255u);
#pragma unroll
                for (int i = 0; i < IT; ++i) {
                    F8Frag f;
                    if constexpr (TRANS) f = read_turned(wm * TM + i * 16);
                    else f = read(la, wm * TM + i * 16 + r16);
                    const f4 part = f8_dot(F8Half(f), b);
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[i][j][k] = fmaf(part[k] * scale, wscale, acc[i][j][k]);
                }
            }
        }
    }

    // a lane holds four neighbouring rows of one token
#pragma unroll
    for (int j = 0; j < JT; ++j) {
        const int64_t n = n0 + wn * TN + j * 16 + r16;
        if (n >= a.N) continue;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int64_t r = row0 + wm * TM + i * 16 + chunk * 4;
            if (r >= t.rows) continue;
            const int left = (int) min((int64_t) 4, t.rows - r);
            if (t.sums != nullptr || a.y_type == TRC_HIP_TYPE_F32) {
                float* const p = t.sums != nullptr ? t.sums + ((int64_t) blockIdx.y * a.N + n) * t.sums_nb1 + r
                                                   : (float*) (a.y + n * a.y_nb1) + r;
                if (left == 4) *(f4a4*) p = acc[i][j];
                else
                    for (int k = 0; k < left; ++k) p[k] = acc[i][j][k];
            } else {
                uint16_t* const p = (uint16_t*) (a.y + n * a.y_nb1) + r;
                uint16_t v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = f8_bits(a.y_type, acc[i][j][k]);
                if (left == 4) {
                    typedef uint32_t u2a2 __attribute__((ext_vector_type(2), aligned(2)));
                    *(u2a2*) p = (u2a2){(uint32_t) v[0] | (uint32_t) v[1] << 16, (uint32_t) v[2] | (uint32_t) v[3] << 16};
                } else {
                    for (int k = 0; k < left; ++k) p[k] = v[k];
                }
            }
        }
    }
}

}  // namespace

#define F8_INSTANCE(BM, BN, WM, WN, TRANS, FAST, POW2)                                                                \
    template <>                                                                                                       \
    void f8_tiles_launch<BM, BN, WM, WN, TRANS, FAST, POW2>(const F8Tiles& t, unsigned parts, hipStream_t s) {        \
        hipLaunchKernelGGL((k_f8_tiles<BM, BN, WM, WN, TRANS, FAST, POW2>), dim3((unsigned) ((t.tm * t.tn + 7) / 8 * 8), parts), \
                           dim3(WM * WN * 64), 0, s, t);                                                              \
    }
#define F8_INSTANCES(BM, BN, WM, WN, FAST)          \
    F8_INSTANCE(BM, BN, WM, WN, false, FAST, false) \
    F8_INSTANCE(BM, BN, WM, WN, false, FAST, true)  \
    F8_INSTANCE(BM, BN, WM, WN, true, FAST, false)  \
    F8_INSTANCE(BM, BN, WM, WN, true, FAST, true)

}  // namespace trc_hip
