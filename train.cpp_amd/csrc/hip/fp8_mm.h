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

// POW2: the weight's scales are bytes.
template <int BM, int BN, int WM, int WN, int KG, int STAGES, bool TRANS, bool POW2>
void f8_tiles_launch(const F8Tiles& t, unsigned parts, hipStream_t s);

namespace {

constexpr uint32_t F8_RSRC = 0x00027000;

typedef __attribute__((address_space(3))) uint8_t lds_byte;
typedef int i2v __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i2v lds_i2v;

// 16-byte chunks of a tile's row in LDS lie at slots chunk ^ f8_turn(row), so that what is read together falls on
// different banks (64 of 4 bytes). Rows of 128 bytes read 16 bytes a lane: eight rows, one chunk. A weight that is read
// turned, 32 lanes at once: rows m to m + 7 and m + 16 to m + 23, 16 bytes of each (by rows of CH chunks; with row & 7
// there every such read took two passes).
template <bool TURNED, int CH>
__device__ __forceinline__ int f8_turn(int row) {
    if (!TURNED) return row & 7;
    if (CH == 8) return ((row >> 1) & 3) | ((row >> 4) & 1) << 2;
    return ((row >> 2) & 1) | ((row >> 4) & 1) << 1;
}

// One operand's tile of a step, ROWS rows of 16 CH bytes, from memory to LDS without a way through registers, in pieces of
// 16 bytes a thread: piece p lands 16 THREADS bytes after piece p - 1, and the slots' turn is in the address it is read
// from.
template <int ROWS, int CH, int THREADS, bool TURNED>
struct F8Slab {
    static constexpr int PIECES = ROWS * CH / THREADS, PER = THREADS / CH;  // rows of a piece
    static constexpr int BYTES = ROWS * CH * 16;
    static_assert(PIECES * THREADS == ROWS * CH && PER % 32 == 0, "whole pieces, the same turn in each");
    uint32_t off;
    __device__ __forceinline__ F8Slab(int tid, int64_t nb1) {
        const int row = tid / CH, slot = tid % CH;
        off = (uint32_t) (row * nb1) + (uint32_t) (slot ^ f8_turn<TURNED, CH>(row)) * 16;
    }
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, int p, int64_t nb1, lds_byte* lds, int wave) const {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*) (lds + (p * THREADS + wave * 64) * 16), 16, off,
                                                 (uint32_t) (p * PER * nb1), 0, 0);
    }
};

// Waves of a SIMD: a workgroup's, twice where its stages leave room in LDS for another workgroup.
constexpr int f8_waves(int bm, int bn, int waves, int groups, int stages) {
    return (waves * groups + 3) / 4 * (groups * stages * ((bm + bn) * F8_BLOCK + 4 * bn) <= 80 * 1024 ? 2 : 1);
}

// A wave waits until `n` of its loads from memory at most are under way, and for its accesses to LDS.
template <int N>
__device__ __forceinline__ void f8_wait() {
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4);
}

// A bare barrier: __syncthreads' fence would wait for the loads that are to stay under way.
__device__ __forceinline__ void f8_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A tile: where it lies, its operands' way to LDS and from there, and its results' to memory. KG groups of WM WN waves take
// every KG-th step each, with stages of their own.
template <int BM, int BN, int WM, int WN, int KG, int STAGES, bool TRANS, bool POW2>
struct F8Tile {
    static constexpr int THREADS = WM * WN * 64, TM = BM / WM, TN = BN / WN, IT = TM / 16, JT = TN / 16;
    static constexpr int ACH = TRANS ? BM / 16 : 8;
    static_assert(TM <= F8_BLOCK && F8_BLOCK % TM == 0, "a wave's rows share their scales");
    typedef F8Slab<TRANS ? F8_BLOCK : BM, ACH, THREADS, TRANS> ASlab;
    typedef F8Slab<BN, 8, THREADS, false> BSlab;
    static constexpr int STAGE = ASlab::BYTES + BSlab::BYTES + BN * 4, LOADS = ASlab::PIECES + BSlab::PIECES + 1;
    static constexpr int GROUP = STAGES * STAGE;  // bytes of LDS

    const F8Tiles& t;
    const int tid, kg, lane, wave;  // (tid and wave: within the group)
    lds_byte* const lds;
    const int wm, wn, r16, chunk;
    int64_t row0, n0, a_rows, b_rows, pitch;
    const ASlab slab_a;
    const BSlab slab_b;
    const uint8_t* x0;
    __amdgpu_buffer_rsrc_t rs;  // the tokens' exponents, a word of four steps of each
    uint32_t e_off;
    int a_bytes, a_last, b_bytes;  // of a step's tiles from their first byte on; of the weight's last step, on the way back
    uint64_t ws;
    int64_t ws_step;

    __device__ __forceinline__ F8Tile(const F8Tiles& tiles, uint8_t* shared, int tile)
        : t(tiles), tid((int) threadIdx.x % THREADS), kg(KG == 1 ? 0 : __builtin_amdgcn_readfirstlane((int) threadIdx.x / THREADS)),
          lane(tid & 63), wave(__builtin_amdgcn_readfirstlane(tid >> 6)), lds((lds_byte*) shared + kg * GROUP), wm(wave % WM),
          wn(wave / WM), r16(lane & 15), chunk(lane >> 4), slab_a(tid, tiles.a.w_nb1), slab_b(tid, tiles.a.x_nb1) {
        const F8Args& a = t.a;
        // four tiles of rows by all of the tokens', then the next four: neighbours on an XCD share operands in its L2
        const int in = tile % (4 * t.tn), first = tile / (4 * t.tn) * 4, high = min(4, t.tm - first);
        row0 = (int64_t) (first + in % high) * BM;
        n0 = (int64_t) (in / high) * BN;
        pitch = (a.K + F8_BLOCK - 1) / F8_BLOCK * F8_BLOCK;
        a_rows = min((int64_t) BM, a.M - row0);
        b_rows = min((int64_t) BN, a.N - n0);
        x0 = a.x + n0 * a.x_nb1;
        const int64_t width = TRANS ? pitch - row0 : F8_BLOCK;
        a_bytes = (int) (uint32_t) (((TRANS ? min((int64_t) F8_BLOCK, a.M) : a_rows) - 1) * a.w_nb1 + width);
        a_last = TRANS ? (int) (uint32_t) ((a.M - 1) % F8_BLOCK * a.w_nb1 + width) : a_bytes;
        b_bytes = (int) (uint32_t) ((b_rows - 1) * a.x_nb1 + F8_BLOCK);
        rs = __builtin_amdgcn_make_buffer_rsrc((void*) (a.xs + n0 * a.xs_nb1), (short) 0,
                                               (int) ((b_rows - 1) * a.xs_nb1 + (t.steps + 3) / 4 * 4), F8_RSRC);
        e_off = (uint32_t) ((tid % BN) * a.xs_nb1);
        const int64_t rb = min((row0 + wm * TM) / F8_BLOCK, (t.rows - 1) / F8_BLOCK);
        ws = (uint64_t) (a.ws + (TRANS ? rb * (POW2 ? 1 : 4) : rb * a.ws_nb1));
        ws_step = TRANS ? a.ws_nb1 : (POW2 ? 1 : 4);
    }
    // Where a step's tiles lie. Rows past an operand are read as zeros (on the way back: the weight's last rows of a step),
    // and so is all of a step from `end` on: what is loaded ahead needs no branch.
    struct Source {
        __amdgpu_buffer_rsrc_t a, b;
        int word;
    };
    __device__ __forceinline__ Source source(int s, int end) const {
        const F8Args& g = t.a;
        const bool some = s < end;
        s = min(s, end - 1);
        const uint8_t* const w = TRANS ? g.w + (int64_t) s * F8_BLOCK * g.w_nb1 + row0 : g.w + row0 * g.w_nb1 + (int64_t) s * F8_BLOCK;
        // (selections, without a branch: it would keep the products before it apart from those behind it)
        const int bytes = TRANS && s == t.steps - 1 ? a_last : a_bytes;
        return {__builtin_amdgcn_make_buffer_rsrc((void*) w, (short) 0, some ? bytes : 0, F8_RSRC),
                __builtin_amdgcn_make_buffer_rsrc((void*) (x0 + (int64_t) s * F8_BLOCK), (short) 0, some ? b_bytes : 0, F8_RSRC),
                s & ~3};
    }
    // piece p of LOADS on its way to a stage
    __device__ __forceinline__ void load(const Source& from, int stage, int p) const {
        lds_byte* const at = lds + stage * STAGE;
        if (p < ASlab::PIECES) slab_a.load(from.a, p, t.a.w_nb1, at, wave);
        else if (p < LOADS - 1) slab_b.load(from.b, p - ASlab::PIECES, t.a.x_nb1, at + ASlab::BYTES, wave);
        else
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                rs, (__attribute__((address_space(3))) void*) (at + ASlab::BYTES + BSlab::BYTES + (wave * 64 % BN) * 4), 4, e_off, from.word, 0, 0);
    }
    // the weight's scale of a step, by the scalar unit
    __device__ __forceinline__ uint32_t scale(int s, int end) const {
        s = min(s, end - 1);
        typedef const __attribute__((address_space(4))) uint32_t scalar_word;
        const uint64_t at = ws + (uint64_t) (s * ws_step);
        const uint32_t word = *(scalar_word*) (at & ~(uint64_t) 3);
        return POW2 ? word >> (8 * (at & 3)) & 255u : word;
    }
    __device__ __forceinline__ F8Frag rows_of(const lds_byte* base, int row) const {
        F8Frag f;
        const lds_byte* const p = base + row * 128;
        const int turn = f8_turn<false, 8>(row);
        f.half[0] = *(const __attribute__((address_space(3))) u4v*) (p + ((chunk ^ turn) * 16));
        f.half[1] = *(const __attribute__((address_space(3))) u4v*) (p + (((chunk + 4) ^ turn) * 16));
        return f;
    }
    // Fragment i of the weight. Turned: eight of its rows by 16 of its columns at a time; lane l of 16 gives the address of
    // half a row and gets a column.
    __device__ __forceinline__ F8Frag weight(int stage, int i) const {
        const lds_byte* const base = lds + stage * STAGE;
        if constexpr (!TRANS) return rows_of(base, wm * TM + i * 16 + r16);
        F8Frag f;
        const int col = (wm * TM + i * 16) >> 4;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int m = 16 * chunk + 8 * (q & 1) + 64 * (q >> 1) + (r16 >> 1);
            const lds_byte* const p = base + m * BM + ((col ^ f8_turn<true, ACH>(m)) * 16) + (r16 & 1) * 8;
            f.quarter[q] = __builtin_bit_cast(u2v, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i2v*) p));
        }
        return f;
    }
    __device__ __forceinline__ F8Frag token(int stage, int j) const {
        return rows_of(lds + stage * STAGE + ASlab::BYTES, wn * TN + j * 16 + r16);
    }
    // (of a step of zeros from `end` on the last step's: what lies behind a row's exponents may be anything, and 0 times the
    // infinity or NaN that it stands for would be NaN)
    __device__ __forceinline__ uint32_t exponent(int s, int end, int stage, int j) const {
        s = min(s, end - 1);
        const lds_byte* const p = lds + stage * STAGE + ASlab::BYTES + BSlab::BYTES;
        return ((const __attribute__((address_space(3))) uint32_t*) p)[wn * TN + j * 16 + r16] >> (8 * (s & 3)) & 255u;
    }
    // The groups' sums added in their order, and stored: a lane holds four neighbouring rows of one token.
    __device__ __forceinline__ void store(f4 (&acc)[IT][JT]) const {
        const F8Args& a = t.a;
        f8_wait<0>();  // (what was loaded ahead: zeros, to LDS that this or another workgroup has another use for)
        if constexpr (KG > 1) {
            static_assert(KG == 2 && IT * JT * THREADS * 16 <= GROUP, "the other group's sums fit its stages");
            typedef __attribute__((address_space(3))) f4 lds_f4;
            lds_f4* const sums = (lds_f4*) (lds - kg * GROUP + GROUP);
            if (kg == 1) {
                // (its waves have read their stages' last, but not all at once)
                f8_barrier();
#pragma unroll
                for (int i = 0; i < IT; ++i)
#pragma unroll
                    for (int j = 0; j < JT; ++j) sums[(i * JT + j) * THREADS + tid] = acc[i][j];
                f8_wait<0>();
                f8_barrier();
                return;
            }
            f8_barrier();
            f8_barrier();
#pragma unroll
            for (int i = 0; i < IT; ++i)
#pragma unroll
                for (int j = 0; j < JT; ++j) acc[i][j] += sums[(i * JT + j) * THREADS + tid];
        }
        const int64_t first = row0 + wm * TM;
#pragma unroll
        for (int j = 0; j < JT; ++j) {
            const int64_t n = n0 + wn * TN + j * 16 + r16;
            if (t.sums != nullptr || a.y_type == TRC_HIP_TYPE_F32) {
                if (n >= a.N) continue;
                float* const p = t.sums != nullptr ? t.sums + ((int64_t) blockIdx.y * a.N + n) * t.sums_nb1 : (float*) (a.y + n * a.y_nb1);
#pragma unroll
                for (int i = 0; i < IT; ++i) {
                    const int64_t r = first + i * 16 + chunk * 4;
                    if (r + 4 <= t.rows) *(f4a4*) (p + r) = acc[i][j];
                    else
                        for (int k = 0; r + k < t.rows; ++k) p[r + k] = acc[i][j][k];
                }
            } else {
                // Of two fragments' rows a lane has four each; it changes one four with its neighbour 16 lanes on, and has
                // eight of one: 64 bytes of a token are stored at once (from larger tiles 33 MB took 17 us in pieces of 32 bytes, 9 so).
                uint16_t* const p = (uint16_t*) (a.y + n * a.y_nb1);
#pragma unroll
                for (int i = 0; i < IT; i += 2) {
                    uint32_t v[4];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        auto two = [&](const f4& x) {
                            return (uint32_t) f8_bits(a.y_type, x[2 * k]) | (uint32_t) f8_bits(a.y_type, x[2 * k + 1]) << 16;
                        };
                        const auto s = __builtin_amdgcn_permlane16_swap(two(acc[i][j]), two(acc[i + 1][j]), false, false);
                        v[k] = s[0];
                        v[k + 2] = s[1];
                    }
                    const int64_t r = first + (i + (chunk & 1)) * 16 + (chunk >> 1) * 8;
                    if (n >= a.N) continue;
                    typedef uint32_t u4a2 __attribute__((ext_vector_type(4), aligned(2)));
                    if (r + 8 <= t.rows) *(u4a2*) (p + r) = (u4a2){v[0], v[1], v[2], v[3]};
                    else
                        for (int k = 0; r + k < t.rows && k < 8; ++k) p[r + k] = (uint16_t) (v[k / 2] >> (16 * (k & 1)));
                }
            }
        }
    }
};

// Products in binary16.
template <int BM, int BN, int WM, int WN, int KG, int STAGES, bool TRANS, bool POW2>
__device__ __forceinline__ void f8_multiply(const F8Tiles& t, uint8_t* shared, int tile) {
    typedef F8Tile<BM, BN, WM, WN, KG, STAGES, TRANS, POW2> Tile;
    // (pieces from memory at once: all of them in the first two rounds of products)
    constexpr int IT = Tile::IT, JT = Tile::JT, EACH = (Tile::LOADS + 1) / 2;
    const Tile w(t, shared, tile);
    const int first = (int) blockIdx.y * t.part_steps, s1 = min(first + t.part_steps, t.steps), s0 = first + w.kg;
    const int rounds = (s1 - first + KG - 1) / KG;  // (a step from s1 on is one of zeros)
    f4 acc[IT][JT];
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int j = 0; j < JT; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < STAGES - 1; ++k) {
        const typename Tile::Source from = w.source(s0 + k * KG, s1);
#pragma unroll
        for (int p = 0; p < Tile::LOADS; ++p) w.load(from, k, p);
    }
    uint32_t wnext = w.scale(s0, s1);
    int stage = 0, s = s0;
    for (int round = 0; round < rounds; ++round, s += KG) {
        // this step's tiles have landed (the next STAGES - 2 may not have), and every wave has read the last step's
        f8_wait<Tile::LOADS * (STAGES - 2)>();
        f8_barrier();
        const float wscale = POW2 ? f8_scale(wnext) : __builtin_bit_cast(float, wnext);
        wnext = w.scale(s + KG, s1);
        const typename Tile::Source from = w.source(s + (STAGES - 1) * KG, s1);
        const int into = stage == 0 ? STAGES - 1 : stage - 1;
        h8v wh[IT][4], x[4];
        auto half = [](const F8Frag& f, h8v (&h)[4]) {
#pragma unroll
            for (int q = 0; q < 4; ++q) h[q] = f8_half8(f.quarter[q]);
        };
        half(w.token(stage, 0), x);
#pragma unroll
        for (int i = 0; i < IT; ++i) half(w.weight(stage, i), wh[i]);
        f4 part[2][IT];
        float scale[2];
        auto add = [&](int j) {
#pragma unroll
            for (int i = 0; i < IT; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[i][j][k] = fmaf(part[j & 1][i][k], scale[j & 1], acc[i][j][k]);
        };
#pragma unroll
        for (int j = 0; j < JT; ++j) {
            h8v next[4];
            scale[j & 1] = f8_scale(w.exponent(s, s1, stage, j)) * wscale;
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int i = 0; i < IT; ++i) {
                    const f4 zero = {0.f, 0.f, 0.f, 0.f};
                    part[j & 1][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh[i][q], x[q], q == 0 ? zero : part[j & 1][i], 0, 0, 0);
                }
            if (j + 1 < JT) half(w.token(stage, j + 1), next);
            if (j > 0) add(j - 1);
#pragma unroll
            for (int p = j * EACH; p < (j + 1) * EACH && p < Tile::LOADS; ++p) w.load(from, into, p);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int q = 0; q < 4; ++q) x[q] = next[q];
        }
        add(JT - 1);
        stage = stage == STAGES - 1 ? 0 : stage + 1;
    }
    w.store(acc);
}

// An XCD (workgroup b is on XCD b % 8) takes neighbouring tiles.
template <int BM, int BN, int WM, int WN, int KG, int STAGES, bool TRANS, bool POW2>
__global__ __launch_bounds__(WM * WN * KG * 64, f8_waves(BM, BN, WM * WN, KG, STAGES)) void k_f8_tiles(F8Tiles t) {
    __shared__ __attribute__((aligned(128))) uint8_t shared[KG * F8Tile<BM, BN, WM, WN, KG, STAGES, TRANS, POW2>::GROUP];
    const int tile = (int) (blockIdx.x & 7) * ((t.tm * t.tn + 7) / 8) + (int) (blockIdx.x >> 3);
    if (tile < t.tm * t.tn) f8_multiply<BM, BN, WM, WN, KG, STAGES, TRANS, POW2>(t, shared, tile);
}

}  // namespace

#define F8_INSTANCE(BM, BN, WM, WN, KG, STAGES, TRANS, POW2)                                                                \
    template <>                                                                                                        \
    void f8_tiles_launch<BM, BN, WM, WN, KG, STAGES, TRANS, POW2>(const F8Tiles& t, unsigned parts, hipStream_t s) {       \
        hipLaunchKernelGGL((k_f8_tiles<BM, BN, WM, WN, KG, STAGES, TRANS, POW2>),                                          \
                           dim3((unsigned) (8 * ((t.tm * t.tn + 7) / 8)), parts), dim3(WM * WN * KG * 64), 0, s, t);       \
    }
#define F8_INSTANCES(BM, BN, WM, WN, KG, STAGES)          \
    F8_INSTANCE(BM, BN, WM, WN, KG, STAGES, false, false) \
    F8_INSTANCE(BM, BN, WM, WN, KG, STAGES, false, true)  \
    F8_INSTANCE(BM, BN, WM, WN, KG, STAGES, true, false)  \
    F8_INSTANCE(BM, BN, WM, WN, KG, STAGES, true, true)

}  // namespace trc_hip
