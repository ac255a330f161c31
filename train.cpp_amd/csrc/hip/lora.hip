// Low-rank adapters of the requests of a batch beside the projection they share
// (Hu et al., "LoRA: Low-Rank Adaptation of Large Language Models", 2021), and their
// gradients. Request q holds tokens start[q] .. start[q+1]-1 and uses adapter a = ids[q]:
//
//   h_t  = A_a x_t              y_t  = base_t + s_a B_a h_t
//   g_t  = s_a B_a^T dy_t       dx_t = base_t + A_a^T g_t
//   dA_a = sum_t g_t x_t^T      dB_a = s_a sum_t dy_t h_t^T
//
// Three steps make all six, on v_mfma_f32_16x16x4_f32 (products as exact as float
// FMAs; adapters in 16 bits are widened). h and y of bfloat16 adapters are made on the
// bfloat16 instructions instead, the other factor in three parts, which is exact as well (but an
// infinite weight's products may be NaN: it meets a part that is 0) and takes a fifth of the
// matrix cores' time: 1001 tokens of 13 requests, K 4096, M 14336, R 64 in 42 us, 51 with the FP32
// instructions. (y of ranks that are not whole fours, and of the last columns, stays on
// those: see Expand::singly.)
//   contract  h and g: a wide activation times a matrix of R rows or columns
//   expand    y and dx: base plus a matrix times h or g
//   outer     dA and dB: sums over tokens of outer products
// The first two take 16 tokens of one request at a time, so a request of one token costs one
// reading of its adapter, and a long one reads it once per 16 tokens, from the L2.
//
// In that instruction lane l holds A[i][k] and B[k][j] at i = j = l % 16, k = l / 16, and
// the sums at i = 4 (l / 16) + v, j = l % 16. The order of a sum's terms is free, so a lane takes
// four neighbours of the long axis with one load and feeds them to four instructions.
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace trc_hip {

namespace {

constexpr int LT = 16;             // tokens of a tile
constexpr int L_WAVES = 12;        // waves of a workgroup that makes h and y
constexpr int LO_WAVES = 16;       // waves of a workgroup of the backward pass
constexpr int LE_THREADS = 256;    // k_expand
constexpr int LE_COLS = 64;        // outputs a wave makes of each token at a time
constexpr int LO_COLS = 32;        // outer: columns of a workgroup
constexpr int L_G_PARTS = 4;       // parts of g where it has few tiles, at most
constexpr int LR = 64;             // rank that is summed at a time, at most
constexpr int L_MAX_RANK = TRC_HIP_LORA_MAX_RANK;

// Registers for four waves a SIMD: with fewer, the loads in flight do not fill memory's latency.
#define L_FOUR_WAVES __attribute__((amdgpu_waves_per_eu(4)))

typedef float f4v __attribute__((ext_vector_type(4), may_alias));
typedef uint16_t h4 __attribute__((ext_vector_type(4)));
// elements whose address is only as aligned as one
typedef float f2u __attribute__((ext_vector_type(2), aligned(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t h2u __attribute__((ext_vector_type(2), aligned(2)));
typedef uint16_t h4u __attribute__((ext_vector_type(4), aligned(2)));

// Weights as they are loaded, four or fewer at a time; they are widened where they are
// multiplied, so that nothing waits for a load before.
template <int TYPE>
struct Wt {
    typedef uint16_t Elem;
    template <int N>
    using Raw = std::conditional_t<N == 1, uint16_t, std::conditional_t<N == 2, h2u, h4u>>;
    static __device__ __forceinline__ float get(Elem x) {
        return TYPE == TRC_HIP_TYPE_F16 ? half_bits_to_float(x) : __builtin_bit_cast(float, (uint32_t) x << 16);
    }
};
template <>
struct Wt<TRC_HIP_TYPE_F32> {
    typedef float Elem;
    template <int N>
    using Raw = std::conditional_t<N == 1, float, std::conditional_t<N == 2, f2u, f4u>>;
    static __device__ __forceinline__ float get(Elem x) { return x; }
};
template <class R>
__device__ __forceinline__ auto element(const R& r, int i) {
    if constexpr (std::is_arithmetic_v<R>) {
        return r;
    } else {
        return r[i];
    }
}

// A value of another lane by data-parallel primitives, which need no LDS: 0 where there is no such lane.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ int from_lane(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, true); }
template <int CTRL>
__device__ __forceinline__ float from_lane(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_XOR8 = 0x128;  // (quads permuted; a row of 16 rotated by 8)
constexpr int DPP_SHR = 0x110, DPP_BCAST15 = 0x142, DPP_BCAST31 = 0x143;
// Lane ^ MASK among each 32 lanes, MASK under 32.
template <int MASK>
__device__ __forceinline__ float swizzle_xor(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, x), MASK << 10 | 0x1f));
}

// 16 bytes at any address that is whole elements.
struct __attribute__((packed, aligned(2))) v16u {
    f4v v;
};

// Keeps the loads before it where they are: without it the compiler moves the loads of a loop's next
// round behind the products of this one, and every round waits for memory.
__device__ __forceinline__ void loads_stay() { asm volatile("" ::: "memory"); }
// A wave's LDS operations run in order; this keeps the compiler from changing it.
__device__ __forceinline__ void lds_in_order() { asm volatile("" ::: "memory"); }

// A load at a base all lanes share, kept in scalar registers, and a lane's 32-bit offset.
template <class V>
__device__ __forceinline__ V load_at(const void* base, uint32_t offset) {
    return *(const V*) ((const uint8_t*) base + offset);
}

struct Batch {
    const int32_t* start;
    const int32_t* ids;
    const float* scale;
    int64_t T;
    int32_t requests, adapters;
};

struct Tile {
    int lo;       // first token
    int tokens;   // 0: none
    int adapter;  // -1: none
};

// Requests q0 .. q0+63: a lane's tokens and, in every lane, the tiles of the requests up to its own. What start holds
// is only compared and clamped, so no value of it leads out of the T tokens (wrong ones may overflow the sums).
struct Requests {
    int lo, hi;
    uint32_t mine, upto;
    __device__ __forceinline__ Requests(const Batch& b, int q0) : lo(0), hi(0) {
        const int q = q0 + ((int) threadIdx.x & 63), T = (int) b.T;
        if (q < b.requests) {
            lo = min(max(b.start[q], 0), T);
            hi = min(max(b.start[q + 1], lo), T);
        }
        mine = ((uint32_t) (hi - lo) + LT - 1) / LT;
        upto = mine;
        upto += (uint32_t) from_lane<DPP_SHR + 1>((int) upto);
        upto += (uint32_t) from_lane<DPP_SHR + 2>((int) upto);
        upto += (uint32_t) from_lane<DPP_SHR + 4>((int) upto);
        upto += (uint32_t) from_lane<DPP_SHR + 8>((int) upto);
        upto += (uint32_t) from_lane<DPP_BCAST15, 0xa>((int) upto);
        upto += (uint32_t) from_lane<DPP_BCAST31, 0xc>((int) upto);
    }
    __device__ __forceinline__ uint32_t all() const { return (uint32_t) __builtin_amdgcn_readlane((int) upto, 63); }
};

// Tile `index` of the batch, requests in order and each in tiles of LT tokens. The whole workgroup has to be here;
// the result is the same in all of it and held in scalar registers. Every wave goes through the requests, 64 at a time; of
// more than 256 each wave counts the tiles of 64 first (1024 requests of a token, K = M = 256: 20 us, 23 otherwise;
// 4096 113 and 188; but 256 6.5 and 6.0).
template <int WAVES>
__device__ __forceinline__ Tile find_tile(const Batch& b, uint32_t index) {
    const int wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    int q0 = 0;
    if (b.requests > 256) {
        __shared__ uint32_t counts[WAVES];
        bool found = false;
        for (int at = 0; at < b.requests && !found; at += 64 * WAVES) {
            const uint32_t mine = Requests(b, at + 64 * wave).all();  // (by all lanes, so before the branch)
            if ((threadIdx.x & 63) == 0) counts[wave] = mine;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const uint32_t count = (uint32_t) __builtin_amdgcn_readfirstlane((int) counts[w]);
                if (found) continue;
                found = index < count;
                if (found) q0 = at + 64 * w;
                else index -= count;
            }
            __syncthreads();
        }
        if (!found) return {0, 0, -1};
    }
    for (; q0 < b.requests; q0 += 64) {
        const int id = b.ids[min(q0 + ((int) threadIdx.x & 63), b.requests - 1)];
        const Requests r(b, q0);
        const uint32_t all = r.all();
        const uint64_t in = __ballot(index < r.upto && r.mine > 0);
        if (in != 0) {
            const int src = __ffsll((unsigned long long) in) - 1;
            const int lo = __builtin_amdgcn_readlane(r.lo, src), hi = __builtin_amdgcn_readlane(r.hi, src);
            const int a = __builtin_amdgcn_readlane(id, src);
            const uint32_t before = (uint32_t) __builtin_amdgcn_readlane((int) (r.upto - r.mine), src);
            const int64_t first = lo + (int64_t) (index - before) * LT;
            if (first < lo || first >= hi) return {0, 0, -1};
            return {(int) first, min(hi - (int) first, LT), a >= 0 && a < b.adapters ? a : -1};
        }
        index -= all;
    }
    return {0, 0, -1};
}

__device__ __forceinline__ f4 mfma(float a, float b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

struct Matrix {
    const void* p;
    int64_t row, adapter;  // strides in elements
};

struct Rows {
    const uint8_t* p;
    size_t nb1;
    int64_t n;  // elements of a row
};

template <int WAVES, int RT>
using Partial = f4[WAVES][RT][64];

// Element e = (j * 64 + lane) * 4 + v of the waves' sums, added in order.
template <int WAVES, int RT>
__device__ __forceinline__ float joined(const Partial<WAVES, RT>& part, int e) {
    const float* const p = (const float*) part + e;
    float x[WAVES];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) x[w] = p[w * RT * 256];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) x[0] += x[w];
    return x[0];
}

// Both operands of the instruction want neighbouring lanes in different rows, and a load whose
// neighbouring lanes are not neighbours in memory is split up lane by lane (64 tag lookups
// instead of 16 for 1 KB; that, not HBM, bounded these kernels at first). So 16 rows are loaded
// along the rows and turned through LDS, each wave in a piece of its own: its LDS
// operations run in order, so no barrier is needed.
//
// Rows16: 16 rows of CN elements, as loaded: lane l of load i has 16 bytes (or four elements) of
// row i * RPI + l / LPR. Rows in LDS are 16 bytes longer than CN elements, which spreads 16 rows at one
// column over all banks.
template <class Elem, int CN>
struct Rows16 {
    static constexpr int ES = sizeof(Elem), LPR = CN * ES / 16, RPI = 64 / LPR, LOADS = 16 / RPI;
    static constexpr int PITCH = CN * ES + 16, BYTES = 16 * PITCH;
    static_assert(LOADS >= 1, "a load has 16 rows at most");
    f4v raw[LOADS];
    // row(i): the byte offset of row i, for its lane
    template <class RowOffset>
    static __device__ __forceinline__ void offsets(uint32_t (&o)[LOADS], RowOffset&& row) {
        const int lane = (int) threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) o[i] = row(i * RPI + lane / LPR) + 16 * (lane % LPR);
    }
    __device__ __forceinline__ void load(const uint8_t* base, const uint32_t (&o)[LOADS]) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) raw[i] = load_at<v16u>(base, o[i]).v;
    }
    __device__ __forceinline__ void stage(uint8_t* lds) const {
        const int lane = (int) threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) *(f4v*) (lds + (i * RPI + lane / LPR) * PITCH + 16 * (lane % LPR)) = raw[i];
    }
    // Elements 16 u + 4 (lane / 16) .. + 3 of row lane % 16.
    typedef std::conditional_t<ES == 4, f4, h4> Four;
    static __device__ __forceinline__ Four four(const uint8_t* lds, int u) {
        const int lane = (int) threadIdx.x & 63;
        return *(const Four*) (lds + (lane & 15) * PITCH + (16 * u + 4 * (lane >> 4)) * ES);
    }
};

// N floats, each the sum of three in bfloat16 that hold 8 bits of it each (down to 2^-126; an infinity or NaN
// is in the first alone), so that products with numbers in bfloat16 are exact. A NaN is made quiet first: a signalling
// one may have its payload in the lower half alone, and its upper half is an infinity's.
template <int N>
struct Thirds {
    typedef uint32_t Bits __attribute__((ext_vector_type(N / 2)));
    Bits hi, mid, lo;
    __device__ __forceinline__ explicit Thirds(const float (&x)[N]) {
        uint32_t a[N], b[N], c[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const float quiet = __builtin_canonicalizef(x[k]);
            a[k] = __builtin_bit_cast(uint32_t, quiet);
            const bool finite = __builtin_fabsf(quiet) < __builtin_inff();
            const float rest = finite ? quiet - __builtin_bit_cast(float, a[k] & 0xffff0000u) : 0.f;
            b[k] = __builtin_bit_cast(uint32_t, rest);
            c[k] = __builtin_bit_cast(uint32_t, rest - __builtin_bit_cast(float, b[k] & 0xffff0000u));
        }
#pragma unroll
        for (int k = 0; k < N / 2; ++k) {  // (the upper halves of two)
            hi[k] = __builtin_amdgcn_perm(a[2 * k + 1], a[2 * k], 0x07060302u);
            mid[k] = __builtin_amdgcn_perm(b[2 * k + 1], b[2 * k], 0x07060302u);
            lo[k] = __builtin_amdgcn_perm(c[2 * k + 1], c[2 * k], 0x07060302u);
        }
    }
};
// Products of bfloat16, 4 or 8 to a lane: sums over 16 or 32
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f4 mfma_bf16(u2 a, u2 b, f4 c) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s4, a), __builtin_bit_cast(s4, b), c, 0, 0, 0);
}
__device__ __forceinline__ f4 mfma_bf16(u4 a, u4 b, f4 c) {
    typedef __bf16 b8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

constexpr int L_CHUNK = 32;  // elements of the long axis that a wave takes at a time
// a wave's piece of LDS for contract_tile: x, then 16 columns of A
template <class Elem, bool OUTER>
constexpr int contract_lds = Rows16<float, L_CHUNK>::BYTES + (OUTER ? 0 : Rows16<Elem, L_CHUNK>::BYTES);

// sum_n x[t][n] W(n, r) for the tile's tokens, n in lo .. hi-1 and r in r0 .. r0 + 16 RT - 1,
// where W(n, r) is w[r][n] (A) or, with OUTER, w[n][r] (B); each sum goes to
// sink(token, r, sum). Columns of the weights past R read others again and do not reach
// the sink, as tokens past the tile's. The waves take chunks of the long axis in turn, each with
// the loads of the next chunk under way. part may be the memory that is staged through.
template <int TYPE, bool OUTER, int WAVES, int RT, class Sink>
__device__ __forceinline__ void contract_tile(const Tile& t, const Rows& x, const Matrix& wm, int R, int r0, int64_t lo,
                                              int64_t hi, uint8_t* lds, Partial<WAVES, RT>& part, Sink&& sink) {
    typedef Wt<TYPE> W;
    typedef typename W::Elem Elem;
    constexpr int CN = L_CHUNK, U = CN / 16;
    constexpr int ES = sizeof(Elem);
    typedef Rows16<float, CN> X;
    typedef Rows16<Elem, CN> A;
    const int lane = (int) threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    uint8_t* const xs = lds + wave * contract_lds<Elem, OUTER>;
    uint8_t* const ws = xs + X::BYTES;
    const uint8_t* const xb = x.p + (int64_t) t.lo * x.nb1;
    const uint32_t wrow = (uint32_t) wm.row * ES;
    const uint8_t* const wb = (const uint8_t*) wm.p + (t.adapter * wm.adapter + (OUTER ? 0 : r0 * wm.row)) * ES;
    uint32_t xo[X::LOADS], ao[OUTER ? 1 : RT][A::LOADS], bo = 0;
    X::offsets(xo, [&](int row) { return (uint32_t) min(row, t.tokens - 1) * (uint32_t) x.nb1; });
    // A: tile j's column is r0 + 16 j + col. B: columns side by side, r0 + RT col + j, so that one
    // load has a lane's columns of all tiles; the last ones are moved back into the row (R >= RT).
    if constexpr (OUTER) {
        bo = 4 * quad * wrow + (uint32_t) min(r0 + RT * col, R - RT) * ES;
    } else {
#pragma unroll
        for (int j = 0; j < RT; ++j) A::offsets(ao[j], [&](int row) { return (uint32_t) min(16 * j + row, R - 1 - r0) * wrow; });
    }
    f4 acc[RT];
#pragma unroll
    for (int j = 0; j < RT; ++j) acc[j] = f4{0.f, 0.f, 0.f, 0.f};
    // Whether a chunk's weights are loaded with its x, a chunk ahead; else 16 columns ahead, which takes
    // fewer registers.
    constexpr bool AHEAD = RT * ES <= 4;
    struct Chunk {
        X x;
        A a[OUTER || !AHEAD ? 1 : RT];
        typename W::template Raw<RT> b[OUTER ? U : 1][4];
    };
    auto load = [&](Chunk& c, int64_t i) {  // the wave's chunk i
        const int64_t n = lo + (wave + i * WAVES) * CN;
        c.x.load(xb + n * 4, xo);
        if constexpr (OUTER) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    c.b[u][k] = load_at<typename W::template Raw<RT>>(wb + (n + 16 * u + k) * (int64_t) wrow, bo);
        } else if constexpr (AHEAD) {
#pragma unroll
            for (int j = 0; j < RT; ++j) c.a[j].load(wb + n * ES, ao[j]);
        }
    };
    auto multiply = [&](const Chunk& c, int64_t i) {
        const int64_t n = lo + (wave + i * WAVES) * CN;
        A ring[2];
        if constexpr (!OUTER && !AHEAD) ring[0].load(wb + n * ES, ao[0]);
        c.x.stage(xs);
        lds_in_order();
        f4 xv[U];
#pragma unroll
        for (int u = 0; u < U; ++u) xv[u] = X::four(xs, u);
        if constexpr (OUTER) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int j = 0; j < RT; ++j) acc[j] = mfma(xv[u][k], W::get(element(c.b[u][k], j)), acc[j]);
        } else {
            static_assert(U == 2, "a chunk is 32 elements here, 8 to a lane");
            const float x8[8] = {xv[0][0], xv[0][1], xv[0][2], xv[0][3], xv[1][0], xv[1][1], xv[1][2], xv[1][3]};
            const Thirds<8> x3(x8);
#pragma unroll
            for (int j = 0; j < RT; ++j) {
                if constexpr (AHEAD) {
                    c.a[j].stage(ws);
                } else {
                    if (j + 1 < RT) ring[(j + 1) & 1].load(wb + n * ES, ao[j + 1 < RT ? j + 1 : 0]);
                    loads_stay();
                    ring[j & 1].stage(ws);
                }
                lds_in_order();
                typename A::Four wv[U];
#pragma unroll
                for (int u = 0; u < U; ++u) wv[u] = A::four(ws, u);
                lds_in_order();
                if constexpr (TYPE == TRC_HIP_TYPE_BF16) {
                    const u4 w8 = __builtin_bit_cast(u4, __builtin_shufflevector(wv[0], wv[1], 0, 1, 2, 3, 4, 5, 6, 7));
                    acc[j] = mfma_bf16(x3.lo, w8, acc[j]);
                    acc[j] = mfma_bf16(x3.mid, w8, acc[j]);
                    acc[j] = mfma_bf16(x3.hi, w8, acc[j]);
                    continue;
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[j] = mfma(xv[u][k], W::get(wv[u][k]), acc[j]);
            }
        }
        lds_in_order();
    };
    const int64_t chunks = (hi - lo) / CN;
    // Two chunks in turn and no branch around the loads, so that what is waited for is counted in order
    // and nothing is copied.
    const int64_t mine = wave < chunks ? (chunks - wave + WAVES - 1) / WAVES : 0;
    if (mine > 0) {
        Chunk c0, c1;
        load(c0, 0);
        int64_t i = 0;
        for (; i + 2 < mine; i += 2) {
            load(c1, i + 1);
            loads_stay();
            multiply(c0, i);
            load(c0, i + 2);
            loads_stay();
            multiply(c1, i + 1);
        }
        if (i + 1 < mine) {
            load(c1, i + 1);
            loads_stay();
            multiply(c0, i);
            multiply(c1, i + 1);
        } else {
            multiply(c0, i);
        }
    }
    // the rest, in groups of 16 and element by element: both operands are 0 past the end
    for (int64_t n = lo + chunks * CN + wave * 16; n < hi; n += WAVES * 16) {
        const uint32_t xt = (uint32_t) min(col, t.tokens - 1) * (uint32_t) x.nb1;
        float xk[4], wk[4][RT];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t at = (uint32_t) min((int64_t) (4 * quad + k), hi - 1 - n);
            xk[k] = load_at<float>(xb + n * 4, xt + 4 * at);
#pragma unroll
            for (int j = 0; j < RT; ++j) {
                const uint32_t o = OUTER ? at * wrow + (uint32_t) (min(r0 + RT * col, R - RT) + j) * ES
                                         : (uint32_t) min(16 * j + col, R - 1 - r0) * wrow + at * ES;
                wk[k][j] = W::get(load_at<Elem>(OUTER ? wb + n * (int64_t) wrow : wb + n * ES, o));
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const bool in = n + 4 * quad + k < hi;
#pragma unroll
            for (int j = 0; j < RT; ++j) acc[j] = mfma(in ? xk[k] : 0.f, in ? wk[k][j] : 0.f, acc[j]);
        }
    }
    __syncthreads();  // (part may lie over what is staged)
#pragma unroll
    for (int j = 0; j < RT; ++j) part[wave][j][lane] = acc[j];
    __syncthreads();
    for (int e = (int) threadIdx.x; e < RT * 256; e += WAVES * 64) {
        const float sum = joined<WAVES, RT>(part, e);
        const int j = e >> 8, l = (e >> 2) & 63, tok = 4 * (l >> 4) + (e & 3), own = r0 + RT * (l & 15);
        // (a moved column's sums belong to the lane whose own column it is)
        const int r = OUTER ? min(own, R - RT) + j : r0 + 16 * j + (l & 15);
        if (r < R && (!OUTER || r >= own) && tok < t.tokens) sink(tok, r, sum);
    }
}

// The same of one token and A, without the matrix instructions, which would do 16 tokens' work (64 tokens of as
// many adapters, F16, K = M = 4096, R 16: 7.9 us, 12.0 by tiles): each
// lane multiplies eight neighbours of n, a wave takes eight columns r at a time, and as many
// waves as there are share a column's 512-element chunks. red: [wave][8].
template <int TYPE, int WAVES, class Sink>
__device__ __forceinline__ void contract_one(const Tile& t, const Rows& x, const Matrix& wm, int R, int64_t lo, int64_t hi,
                                             float* red, Sink&& sink) {
    typedef Wt<TYPE> W;
    typedef typename W::Elem Elem;
    constexpr int ES = sizeof(Elem);
    const int lane = (int) threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    const uint8_t* const xb = x.p + (int64_t) t.lo * x.nb1;
    const uint8_t* const wb = (const uint8_t*) wm.p + t.adapter * wm.adapter * ES;
    const int groups = (R + 7) / 8;
    for (int g0 = 0; g0 < groups; g0 += WAVES) {
        const int here = min(groups - g0, WAVES), per = WAVES / here;  // waves that share a group
        const int g = g0 + wave % here, sub = wave / here;
        float acc[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) acc[r] = 0.f;
        if (sub < per) {
            for (int64_t n = lo + sub * 512; n < hi; n += per * 512) {
                const int left = (int) min((int64_t) 8, max((int64_t) 0, hi - n - 8 * lane));
                if (left == 8) {
                    const f4u x0 = load_at<f4u>(xb + n * 4, 32 * lane), x1 = load_at<f4u>(xb + n * 4, 32 * lane + 16);
                    f4v raw[8][ES / 2];
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        const uint8_t* const row = wb + (min(8 * g + r, R - 1) * wm.row + n) * ES;
#pragma unroll
                        for (int k = 0; k < ES / 2; ++k) raw[r][k] = load_at<v16u>(row, 8 * ES * lane + 16 * k).v;
                    }
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        Elem w[8];
                        __builtin_memcpy(w, raw[r], sizeof(w));
#pragma unroll
                        for (int k = 0; k < 4; ++k) acc[r] = fmaf(x1[k], W::get(w[4 + k]), fmaf(x0[k], W::get(w[k]), acc[r]));
                    }
                } else {
                    for (int k = 0; k < left; ++k) {
                        const float xk = load_at<float>(xb + n * 4, 32 * lane + 4 * k);
#pragma unroll
                        for (int r = 0; r < 8; ++r) {
                            const uint8_t* const row = wb + (min(8 * g + r, R - 1) * wm.row + n) * ES;
                            acc[r] = fmaf(xk, W::get(load_at<Elem>(row, (8 * lane + k) * ES)), acc[r]);
                        }
                    }
                }
            }
        }
        // Eight sums over 64 lanes: three rounds that halve the sums a lane keeps, three that add up.
        // What lane bits 0, 1 and 3 keep apart, and so a lane's column: bits 2, 1 and 0 of it.
        const bool b0 = (lane & 1) != 0, b1 = (lane & 2) != 0, b3 = (lane & 8) != 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r] = (b0 ? acc[r + 4] : acc[r]) + from_lane<DPP_XOR1>(b0 ? acc[r] : acc[r + 4]);
#pragma unroll
        for (int r = 0; r < 2; ++r) acc[r] = (b1 ? acc[r + 2] : acc[r]) + from_lane<DPP_XOR2>(b1 ? acc[r] : acc[r + 2]);
        float s = (b3 ? acc[1] : acc[0]) + from_lane<DPP_XOR8>(b3 ? acc[0] : acc[1]);
        s += swizzle_xor<4>(s);
        s += swizzle_xor<16>(s);
        s += __shfl_xor(s, 32, 64);
        __syncthreads();
        if ((lane & 52) == 0) red[wave * 8 + (b0 ? 4 : 0) + (b1 ? 2 : 0) + (b3 ? 1 : 0)] = s;
        __syncthreads();
        for (int i = (int) threadIdx.x; i < here * 8; i += WAVES * 64) {
            const int r = 8 * (g0 + i / 8) + i % 8;
            float part[WAVES], sum = 0.f;
#pragma unroll
            for (int k = 0; k < WAVES; ++k) part[k] = red[min(k * here + i / 8, WAVES - 1) * 8 + i % 8];
#pragma unroll
            for (int k = 0; k < WAVES; ++k) sum += k < per ? part[k] : 0.f;
            if (r < R) sink(0, r, sum);
        }
    }
}

// A row's first byte up to 2^31 on; what lies further is neither read (0 comes back) nor stored
// to. Nothing is, with no memory.
constexpr uint32_t L_RSRC_WORD3 = 0x00020000u;  // gfx9 buffer resource: raw 32-bit dwords
constexpr uint32_t L_SPAN = 0x80000000u, L_OUTSIDE = 0xffffff00u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t span(const uint8_t* p, bool memory) {
    return __builtin_amdgcn_make_buffer_rsrc((void*) p, (short) 0, memory ? (int) L_SPAN : 0, L_RSRC_WORD3);
}

// out[t][n] = base[t][n] + sum_r hs[t][r] W(n, r) for n in n_lo .. n_hi-1: W(n, r) is w[n][r] (B)
// or, with OUTER, w[r][n] (A). hs has rows of Rp + 4 floats with zeros from R to Rp, R
// rounded up to 16 RT. A wave makes 64 columns of the 16 tokens at a time; column
// 4 (l % 16) + c of the 64 is tile c's, so a lane has four neighbours of each of its four
// tokens, and base and out are read and written in runs of 256 bytes. Tokens past the tile's are left out
// by their offsets, so no tile has a branch around its loads and stores: with one, a wait for
// loads waits for all that is under way.
template <int TYPE, bool OUTER, int WAVES, int RT, bool WIDE = false, bool EARLY = false>
struct Expand {
    typedef Wt<TYPE> W;
    typedef typename W::Elem Elem;
    static constexpr int ES = sizeof(Elem);
    // A block is KB of the rank, as loaded. A: [k] is row r0 + 4 quad + k, columns 4 col .. + 3. B: [i] is row
    // 16 i + lane / 4 of the 64, r0 + F (lane % 4) .. + F-1; it is turned through LDS. A lane's F elements are
    // 16 bytes for F32 and WIDE, else 8: a row's 64 bytes side by side are read at twice the rate of 32 (1001 tokens of 13
    // requests, K 4096, M 14336, R 64: bfloat16 43 us, 49 without WIDE, F16 55 and 62).
    static constexpr int F = WIDE ? 8 : 4, KB = 4 * F;
    typedef Elem Four __attribute__((ext_vector_type(F)));
    typedef Elem FourU __attribute__((ext_vector_type(F), aligned(ES)));
    struct Weights {
        Four w[4];
    };
    // such blocks that are under way ahead of the one that is multiplied (in 32 registers at most)
    static constexpr int NB = 16 * RT / KB, D = NB < 32 / (F * ES) ? NB : 32 / (F * ES);
    // B in LDS: row n of the 64 is (n % 4, n / 4), since a lane reads rows 4 col + c; the
    // paddings spread both the rows of a store and those of a read over the banks.
    static constexpr int PITCH = 5 * F * ES, BLOCK = 16 * PITCH + 4 * F * ES;
    static constexpr int LDS = OUTER ? 0 : 4 * BLOCK;  // bytes of a wave
    struct Base {
        f4 b[4];
    };
    const Tile& t;
    const uint8_t *w, *bp, *op;
    uint32_t wrow;
    uint8_t* lds;
    int R, lane, col, quad, wave;
    bool based, in_place;  // in_place: base is out
    int64_t N, n_lo, steps;  // steps: whole ones
    uint32_t bo[4], oo[4];
    Weights window[D];
    Base b;

    __device__ __forceinline__ Expand(const Tile& t, const Matrix& wm, int R, const uint8_t* base, size_t base_nb1, int64_t N,
                                      uint8_t* out, size_t out_nb1, int64_t n_lo, int64_t n_hi, uint8_t* all_lds)
        : t(t), R(R), based(base != nullptr), in_place(base == out && base_nb1 == out_nb1), N(min(n_hi, N)), n_lo(n_lo) {
        lane = (int) threadIdx.x & 63;
        col = lane & 15;
        quad = lane >> 4;
        wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
        lds = all_lds + wave * LDS;
        w = (const uint8_t*) wm.p + max(t.adapter, 0) * wm.adapter * ES;
        wrow = (uint32_t) wm.row * ES;
        bp = base + (int64_t) t.lo * base_nb1;
        op = out + (int64_t) t.lo * out_nb1;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const uint32_t tok = (uint32_t) (4 * quad + v);
            bo[v] = (int) tok < t.tokens ? tok * (uint32_t) base_nb1 + 16 * col : L_OUTSIDE;
            oo[v] = (int) tok < t.tokens ? tok * (uint32_t) out_nb1 + 16 * col : L_OUTSIDE;
        }
        steps = (this->N - n_lo) / LE_COLS;
    }
    // Whether weights are loaded in blocks; of the lanes' elements past R the last ones are read again.
    __device__ __forceinline__ bool fours() const { return t.adapter >= 0 && R % F == 0; }

    __device__ __forceinline__ void load(Weights& s, int64_t n0, int r0) const {
        const uint32_t r = (uint32_t) min(r0 + F * (OUTER ? quad : lane & 3), R - F);
        const uint32_t o = OUTER ? r * wrow + 4 * col * ES : (lane >> 2) * wrow + r * ES;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            s.w[k] = load_at<FourU>(OUTER ? w + n0 * ES + k * (int64_t) wrow : w + (n0 + 16 * k) * wrow, o);
    }
    // base is read and the outputs are written once, past the caches (auxiliary bit 1): 4096 tokens, K = M = 4096,
    // R 16 in 37 us, with plain accesses 44
    __device__ __forceinline__ void load(Base& s, int64_t n0, bool wanted = true) const {
        const __amdgpu_buffer_rsrc_t m = span(bp + n0 * 4, based && wanted);
#pragma unroll
        for (int v = 0; v < 4; ++v) s.b[v] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(m, bo[v], 0, 2));
    }
    __device__ __forceinline__ void store(const f4 (&sum)[4], int64_t n0, bool wanted = true) const {
        const __amdgpu_buffer_rsrc_t m = span(op + n0 * 4, wanted);
#pragma unroll
        for (int v = 0; v < 4; ++v) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, sum[v]), m, oo[v], 0, 2);
    }
    // zeros past R, whatever was read there; `loaded` once s may be loaded again
    template <class Then>
    __device__ __forceinline__ void multiply(const Weights& s, const float* hrow, int r0, f4 (&acc)[4], Then&& loaded) const {
        float hv[F];
#pragma unroll
        for (int k = 0; k < F; k += 4) {
            const f4 x = *(const f4*) (hrow + r0 + k);
#pragma unroll
            for (int i = 0; i < 4; ++i) hv[k + i] = x[i];
        }
        const bool in = r0 + KB <= R || r0 + F * quad < R;
        Four v[4];
        if constexpr (!OUTER) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int n = 16 * i + (lane >> 2);
                *(Four*) (lds + (n & 3) * BLOCK + (n >> 2) * PITCH + (lane & 3) * F * ES) = s.w[i];
            }
            lds_in_order();
            loaded();
            auto turned = [&](int c) { return *(const Four*) (lds + c * BLOCK + col * PITCH + quad * F * ES); };
            if constexpr (TYPE == TRC_HIP_TYPE_BF16) {
                typedef typename Thirds<F>::Bits Bits;
                const Thirds<F> h3(hv);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const Bits x = in ? __builtin_bit_cast(Bits, turned(c)) : Bits(0);
                    acc[c] = mfma_bf16(h3.lo, x, acc[c]);
                    acc[c] = mfma_bf16(h3.mid, x, acc[c]);
                    acc[c] = mfma_bf16(h3.hi, x, acc[c]);
                }
                lds_in_order();
                return;
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) v[c] = turned(c);
            lds_in_order();
        }
#pragma unroll
        for (int k = 0; k < F; ++k) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float x = W::get(OUTER ? s.w[k][c] : v[c][k]);
                acc[c] = mfma(hv[k], in ? x : 0.f, acc[c]);
            }
        }
        if (OUTER) loaded();
    }
    static __device__ __forceinline__ void clear(f4 (&acc)[4]) {
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[c] = f4{0.f, 0.f, 0.f, 0.f};
    }
    static __device__ __forceinline__ void add(Base& b, const f4 (&acc)[4]) {
#pragma unroll
        for (int v = 0; v < 4; ++v) b.b[v] += f4{acc[0][v], acc[1][v], acc[2][v], acc[3][v]};
    }

    // The wave's first columns: weights, then base, since loads arrive in the order they are waited for.
    __device__ __forceinline__ void begin() {
        const int64_t n0 = n_lo + wave * LE_COLS;
#pragma unroll
        for (int j = 0; j < D; ++j) load(window[j], n0, KB * j);
        load(b, n0);
    }
    __device__ __forceinline__ bool begins() const { return fours() && wave < steps; }
    // With EARLY, they are loaded long before run().
    __device__ __forceinline__ void start() {
        if (EARLY && begins()) begin();
    }
    // 64 columns. A block's registers are loaded with the block D further on, of the next columns in the end; then
    // base of those.
    template <bool NEXT>
    __device__ __forceinline__ void step(const float* hrow, int64_t n0, int64_t n_next) {
        f4 acc[4];
        clear(acc);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            Weights& s = window[j % D];
            multiply(s, hrow, KB * j, acc, [&] {
                if (j + D < NB) load(s, n0, KB * (j + D));
                else if (NEXT) load(s, n_next, KB * (j + D - NB));
                loads_stay();
            });
        }
        for (int r0 = KB * NB; r0 < R; r0 += KB) {
            Weights s;
            load(s, n0, r0);
            multiply(s, hrow, r0, acc, [] {});
        }
        add(b, acc);
        f4 sum[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) sum[v] = b.b[v];
        if (NEXT) {
            load(b, n_next);
            loads_stay();
        }
        store(sum, n0);
    }
    __device__ __forceinline__ void whole_steps(const float* hrow) {
        constexpr int64_t S = WAVES * LE_COLS;
        int64_t n0 = n_lo + wave * LE_COLS;
        if (!EARLY) begin();
        for (int64_t left = (steps - 1 - wave) / WAVES; left > 0; --left, n0 += S) step<true>(hrow, n0, n0 + S);
        step<false>(hrow, n0, 0);
    }
    // Weights one by one, for ranks that are not whole fours and for the last columns.
    __device__ __forceinline__ void singly(const float* hrow, int64_t n0, f4 (&acc)[4]) const {
        const uint8_t* const wn = w + n0 * (OUTER ? (int64_t) ES : (int64_t) wrow);
        uint32_t nc[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) nc[c] = (uint32_t) min((int64_t) (4 * col + c), N - 1 - n0) * (OUTER ? ES : wrow);
        for (int r0 = 0; r0 < R; r0 += 4) {  // four of r, one for each quad
            const int r = r0 + quad;
            const uint32_t rc = (uint32_t) min(r, R - 1) * (OUTER ? wrow : ES);
            const float hv = hrow[r0 + quad - F * quad];
            Elem x[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) x[c] = load_at<Elem>(wn, nc[c] + rc);
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] = mfma(hv, r < R ? W::get(x[c]) : 0.f, acc[c]);
        }
    }
    // One step of any rank and any columns, with or without an adapter.
    __device__ __forceinline__ void any_step(const float* hrow, int64_t n0) {
        f4 acc[4];
        clear(acc);
        if (t.adapter >= 0) singly(hrow, n0, acc);
        if (n0 + LE_COLS <= N) {
            load(b, n0);
            add(b, acc);
            store(b.b, n0);
            return;
        }
        const __amdgpu_buffer_rsrc_t from = span(bp + n0 * 4, based), to = span(op + n0 * 4, true);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const bool in = n0 + 4 * col + k < N;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const uint32_t at = in ? bo[v] + 4 * k : L_OUTSIDE;
                b.b[v][k] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(from, at, 0, 0));
            }
        }
        add(b, acc);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const bool in = n0 + 4 * col + k < N;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const uint32_t at = in ? oo[v] + 4 * k : L_OUTSIDE;
                __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, (float) b.b[v][k]), to, at, 0, 0);
            }
        }
    }
    // A tile without an adapter: base as it is, four steps under way. 4096 tokens, some of them without an adapter,
    // K = M = 4096, R 8, F32: 44 us, step by step 45.
    __device__ __forceinline__ void copy() const {
        constexpr int64_t S = WAVES * LE_COLS;
        for (int64_t i = wave; i < steps; i += 4 * WAVES) {
            Base c[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) load(c[u], n_lo + i * LE_COLS + u * S, i + u * WAVES < steps);
            loads_stay();
#pragma unroll
            for (int u = 0; u < 4; ++u) store(c[u].b, n_lo + i * LE_COLS + u * S, i + u * WAVES < steps);
        }
    }
    __device__ __forceinline__ void run(const float* hs) {
        if (t.adapter < 0 && in_place) return;
        const float* const hrow = hs + col * ((R + 16 * RT - 1) / (16 * RT) * (16 * RT) + 4) + F * quad;
        int64_t i = wave;
        if (begins()) {
            whole_steps(hrow);
            i += ((steps - 1 - wave) / WAVES + 1) * WAVES;
        }
        if (t.adapter < 0 && i < steps) {
            copy();
            i += ((steps - 1 - wave) / WAVES + 1) * WAVES;
        }
        for (; n_lo + i * LE_COLS < N; i += WAVES) any_step(hrow, n_lo + i * LE_COLS);
    }
};

// The same of one token and B, without the matrix instructions. 16 bytes of a row of B are a lane's,
// G lanes (a power of two) make one output together, so a wave reads 1 KB of rows side by side at a time.
template <int TYPE, int WAVES>
struct ExpandOne {
    typedef Wt<TYPE> W;
    typedef typename W::Elem Elem;
    static constexpr int ES = sizeof(Elem), E = 16 / ES, U = 4;
    const uint8_t* w;
    uint32_t wrow;
    const float* bt;
    float* ot;
    int R, lane, G, logG, r0, per;  // per: outputs of a wave at a time
    int64_t n_lo, n_hi;
    f4v raw[U];
    float b[U];

    __device__ __forceinline__ ExpandOne(const Tile& t, const Matrix& wm, int R, const uint8_t* base, size_t base_nb1, int64_t N,
                                         uint8_t* out, size_t out_nb1, int64_t lo, int64_t hi)
        : R(R), lane((int) threadIdx.x & 63), G(1), logG(0) {
        while (G * E < R) G <<= 1, ++logG;
        r0 = (lane & (G - 1)) * E;
        per = 64 >> logG;
        w = (const uint8_t*) wm.p + t.adapter * wm.adapter * ES;
        wrow = (uint32_t) wm.row * ES;
        bt = base != nullptr ? (const float*) (base + (int64_t) t.lo * base_nb1) : nullptr;
        ot = (float*) (out + (int64_t) t.lo * out_nb1);
        n_lo = lo + __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6) * (per * U);
        n_hi = min(hi, N);
    }
    __device__ __forceinline__ uint32_t output(int u, int64_t n0) const {
        return (uint32_t) min((int64_t) (u * per + (lane >> logG)), n_hi - 1 - n0);
    }
    __device__ __forceinline__ void load(int64_t n0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t i = output(u, n0);
            if (R % E == 0) raw[u] = load_at<v16u>(w + n0 * (int64_t) wrow, i * wrow + (uint32_t) min(r0, R - E) * ES).v;
            b[u] = bt != nullptr ? load_at<float>(bt + n0, 4 * i) : 0.f;
        }
    }
    // The first outputs' loads, which may be long before run().
    __device__ __forceinline__ void start() {
        if (n_lo < n_hi) load(n_lo);
    }
    __device__ __forceinline__ void run(const float* hs) {
        float hv[E];
#pragma unroll
        for (int e = 0; e < E; ++e) hv[e] = r0 + e < R ? hs[r0 + e] : 0.f;
        for (int64_t n0 = n_lo; n0 < n_hi; n0 += WAVES * per * U) {
            if (n0 != n_lo) load(n0);
            float sum[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                typedef Elem Piece __attribute__((ext_vector_type(E)));
                Piece x;
                if (R % E == 0) {
                    x = __builtin_bit_cast(Piece, raw[u]);
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        x[e] = load_at<Elem>(w + n0 * (int64_t) wrow, output(u, n0) * wrow + (uint32_t) min(r0 + e, R - 1) * ES);
                }
                sum[u] = 0.f;
#pragma unroll
                for (int e = 0; e < E; ++e) sum[u] = fmaf(hv[e], r0 + e < R ? W::get(x[e]) : 0.f, sum[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (G > 1) sum[u] += from_lane<DPP_XOR1>(sum[u]);
                if (G > 2) sum[u] += from_lane<DPP_XOR2>(sum[u]);
                if (G > 4) sum[u] += swizzle_xor<4>(sum[u]);
                if (G > 8) sum[u] += from_lane<DPP_XOR8>(sum[u]);
                if (G > 16) sum[u] += swizzle_xor<16>(sum[u]);
                if (G > 32) sum[u] += __shfl_xor(sum[u], 32, 64);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t n = n0 + u * per + (lane >> logG);
                if ((lane & (G - 1)) == 0 && n < n_hi) ot[n] = b[u] + sum[u];
            }
        }
    }
};

// The tile's h as Expand wants it: the sum of its parts times s.
template <int RT>
__device__ __forceinline__ void stage_h(const Tile& t, const float* __restrict__ h, int parts, int64_t T, int R, float s,
                                        float* __restrict__ h_sum, float* hs, int threads) {
    const int Rp = (R + 16 * RT - 1) / (16 * RT) * (16 * RT);
    for (int i = (int) threadIdx.x; i < LT * Rp; i += threads) {
        const int tok = i / Rp, r = i % Rp;
        float v = 0.f;
        if (tok < t.tokens && r < R && t.adapter >= 0) {
            const float* const p = h + (int64_t) (t.lo + tok) * R + r;
            for (int k = 0; k < parts; k += 4) {  // (four loads under way)
                float x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = p[min(k + j, parts - 1) * T * R];
#pragma unroll
                for (int j = 0; j < 4; ++j) v += k + j < parts ? x[j] : 0.f;
            }
        }
        if (h_sum != nullptr && tok < t.tokens && r < R) h_sum[(int64_t) (t.lo + tok) * R + r] = v;
        hs[tok * (Rp + 4) + r] = v * s;
    }
    __syncthreads();
}

__device__ __forceinline__ void zero_h(const Tile& t, int R, int r0, int rn, float* out, int threads) {
    for (int i = (int) threadIdx.x; i < t.tokens * rn; i += threads) {
        const int r = r0 + i % rn;
        if (r < R) out[(int64_t) (t.lo + i / rn) * R + r] = 0.f;
    }
}

template <int TYPE, bool OUTER, int WAVES, int RT>
union ContractLds {
    __attribute__((aligned(16))) uint8_t stage[WAVES * contract_lds<typename Wt<TYPE>::Elem, OUTER>];
    Partial<WAVES, RT> part;
};
// floats of a tile's h in LDS
template <int RT>
constexpr int h_floats = LT * ((RT == 4 ? L_MAX_RANK : 16 * RT) + 4);

// h alone. Blocks: (tile, 16 RT of the rank, part of the long axis); part p goes to out + p T R.
template <int TYPE, int RT>
__global__ __launch_bounds__(512) L_FOUR_WAVES void k_contract(Rows x, Matrix wm, int R, Batch b, int64_t part_len,
                                                                float* __restrict__ out) {
    const Tile t = find_tile<8>(b, blockIdx.x);
    if (t.tokens == 0) return;
    __shared__ ContractLds<TYPE, false, 8, RT> lds;
    out += (int64_t) blockIdx.z * b.T * R;
    const int r0 = (int) blockIdx.y * (16 * RT);
    const int64_t lo = (int64_t) blockIdx.z * part_len, hi = min(lo + part_len, x.n);
    auto sink = [&](int tok, int r, float v) { out[(int64_t) (t.lo + tok) * R + r] = v; };
    if (t.adapter < 0) {
        zero_h(t, R, r0, 16 * RT, out, 512);
    } else if (t.tokens == 1) {
        wm.p = (const uint8_t*) wm.p + r0 * wm.row * (int64_t) sizeof(typename Wt<TYPE>::Elem);
        contract_one<TYPE, 8>(t, x, wm, min(R - r0, 16 * RT), lo, hi, (float*) lds.stage,
                              [&](int, int r, float v) { sink(0, r0 + r, v); });
    } else {
        contract_tile<TYPE, false, 8, RT>(t, x, wm, R, r0, lo, hi, lds.stage, lds.part, sink);
    }
}

// Whether 16-bit adapters are expanded 16 bytes of a row at a time
template <int TYPE, int RT>
constexpr bool may_be_wide = TYPE != TRC_HIP_TYPE_F32 && RT > 1;
template <int TYPE, int RT, class Body>
__device__ __forceinline__ void either_width(int R, Body&& body) {
    if constexpr (may_be_wide<TYPE, RT>) {
        if (R % 8 == 0) {
            body(std::true_type{});
            return;
        }
    }
    body(std::false_type{});
}
template <int TYPE, int RT>  // bytes of a wave
constexpr int expand_lds = Expand<TYPE, false, 1, RT, may_be_wide<TYPE, RT>>::LDS;

// y of a tile's columns blockIdx.y * cols .. from h in parts; the first columns' workgroups
// store the sum of more than one part.
template <int TYPE, int RT>
__global__ __launch_bounds__(LE_THREADS) L_FOUR_WAVES void k_expand(const float* __restrict__ h, int parts, Matrix wm, int R, Batch b,
                                                        const uint8_t* base, size_t base_nb1, int64_t N, uint8_t* out,
                                                        size_t out_nb1, float* __restrict__ h_sum, int cols) {
    // Workgroups are dealt out to the 8 XCDs in turn: an XCD has every eighth slice of the columns, so that its
    // L2 holds that part of the adapters alone.
    const int tiles = (int) gridDim.x, slices = (int) gridDim.y, id = (int) (blockIdx.y * gridDim.x + blockIdx.x);
    int tile = (int) blockIdx.x, slice = (int) blockIdx.y;
    if (id < slices / 8 * 8 * tiles) {
        tile = id / 8 % tiles;
        slice = id / 8 / tiles * 8 + id % 8;
    }
    const Tile t = find_tile<LE_THREADS / 64>(b, tile);
    if (t.tokens == 0) return;
    __shared__ __attribute__((aligned(16))) float hs[h_floats<RT>];
    __shared__ __attribute__((aligned(16))) uint8_t stage[LE_THREADS / 64 * expand_lds<TYPE, RT>];
    const int64_t n_lo = (int64_t) slice * cols;
    const float s = t.adapter >= 0 ? b.scale[t.adapter] : 1.f;
    float* const sums = n_lo == 0 ? h_sum : nullptr;
    if (t.tokens == 1 && t.adapter >= 0) {
        ExpandOne<TYPE, LE_THREADS / 64> e(t, wm, R, base, base_nb1, N, out, out_nb1, n_lo, n_lo + cols);
        e.start();
        stage_h<RT>(t, h, parts, b.T, R, s, sums, hs, LE_THREADS);
        e.run(hs);
    } else {
        either_width<TYPE, RT>(R, [&](auto wide) {
            Expand<TYPE, false, LE_THREADS / 64, RT, decltype(wide)::value, true> e(t, wm, R, base, base_nb1, N, out, out_nb1, n_lo,
                                                                                    n_lo + cols, stage);
            e.start();
            stage_h<RT>(t, h, parts, b.T, R, s, sums, hs, LE_THREADS);
            e.run(hs);
        });
    }
}

// Both in one launch: a workgroup makes h of its tile for itself, then y of `cols` columns. 12 waves, one workgroup a
// CU: 4096 tokens, K = M = 4096, R 16, F32 36 us, with 16 waves 38; with 8, two workgroups a CU, 42 (but 42 instead of
// 44 where the tiles are just more than the CUs).
template <int TYPE, int RT>
__global__ __launch_bounds__(L_WAVES * 64) void k_lora(Rows x, Matrix am, Matrix bm, int R, Batch b, const uint8_t* base,
                                                      size_t base_nb1, int64_t N, uint8_t* out, size_t out_nb1,
                                                      float* __restrict__ h, int cols) {
    const Tile t = find_tile<L_WAVES>(b, blockIdx.x);
    if (t.tokens == 0) return;
    __shared__ union {
        ContractLds<TYPE, false, L_WAVES, RT> contract;
        __attribute__((aligned(16))) uint8_t expand[L_WAVES * expand_lds<TYPE, RT>];
    } lds;
    __shared__ __attribute__((aligned(16))) float hs[h_floats<RT>];
    const int hrow = (R + 16 * RT - 1) / (16 * RT) * (16 * RT) + 4;
    const int64_t n_lo = (int64_t) blockIdx.y * cols;
    const float s = t.adapter >= 0 ? b.scale[t.adapter] : 1.f;
    auto sink = [&](int tok, int r, float v) {
        hs[tok * hrow + r] = v * s;
        if (blockIdx.y == 0) h[(int64_t) (t.lo + tok) * R + r] = v;
    };
    if (t.tokens == 1 && t.adapter >= 0) {
        ExpandOne<TYPE, L_WAVES> e(t, bm, R, base, base_nb1, N, out, out_nb1, n_lo, n_lo + cols);
        e.start();
        contract_one<TYPE, L_WAVES>(t, x, am, R, 0, x.n, (float*) lds.contract.stage, sink);
        __syncthreads();
        e.run(hs);
        return;
    }
    either_width<TYPE, RT>(R, [&](auto wide) {
        Expand<TYPE, false, L_WAVES, RT, decltype(wide)::value> e(t, bm, R, base, base_nb1, N, out, out_nb1, n_lo, n_lo + cols,
                                                                         lds.expand);
        if (t.adapter < 0) {
            if (blockIdx.y == 0) zero_h(t, R, 0, R, h, L_WAVES * 64);
        } else {
            for (int i = (int) threadIdx.x; i < LT * hrow; i += L_WAVES * 64) hs[i] = 0.f;
            __syncthreads();
            for (int r0 = 0; r0 < R; r0 += 16 * RT) {
                contract_tile<TYPE, false, L_WAVES, RT>(t, x, am, R, r0, 0, x.n, lds.contract.stage, lds.contract.part, sink);
                __syncthreads();
            }
        }
        e.run(hs);
    });
}

// d(n, r) (+)= scale sum_t x[t][n] h[t][r] over the tokens of one adapter's requests:
// d(n, r) is d[n][r] (dB), or d[r][n] with ROWS (dA).
struct Outer {
    Rows x;
    const float* h;
    int h_parts;  // h is the sum of so many, T R floats apart (dA only, and RT <= 2: L_G_PARTS at most)
    float* d;
    int64_t d_row, d_adapter;
    bool scaled, accumulate;
    int col_blocks, rank_blocks, splits;  // blocks: columns fastest, then ranks, adapters, splits
    int64_t split_len;                    // tokens
    float* parts;                         // [split][adapter], then as in d, where there is more than one split
    int64_t blocks(int adapters) const { return (int64_t) col_blocks * rank_blocks * adapters * splits; }
};

// Each wave takes four tokens at a time; a lane holds two neighbouring columns of one
// token, which feed two accumulators. The waves' sums are joined in order.
template <bool ROWS, int RT>
__device__ __forceinline__ void outer_block(int64_t block, const Outer& o, int R, const Batch& b, Partial<LO_WAVES, RT>& part) {
    const int lane = (int) threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    const int64_t n0 = block % o.col_blocks * LO_COLS;
    block /= o.col_blocks;
    const int r0 = (int) (block % o.rank_blocks) * 16 * RT;
    block /= o.rank_blocks;
    const int adapter = (int) (block % b.adapters), split = (int) (block / b.adapters);
    const int64_t t_lo = split * o.split_len, t_hi = min(t_lo + o.split_len, b.T);
    const int64_t N = o.x.n;
    const bool whole = n0 + LO_COLS <= N;
    f4 acc[2][RT];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int j = 0; j < RT; ++j) acc[c][j] = f4{0.f, 0.f, 0.f, 0.f};
    constexpr int U = 4;  // tokens of a lane that are loaded together
    int turn = wave;      // chunks of 4 U tokens until the wave's next
    for (int q0 = 0; q0 < b.requests; q0 += 64) {
        // each lane looks at a request; those of this adapter are taken in order
        const int q = min(q0 + lane, b.requests - 1);
        const int lo_q = (int) max(min(max((int64_t) b.start[q], (int64_t) 0), b.T), t_lo);
        const int hi_q = (int) min(max((int64_t) b.start[q + 1], (int64_t) lo_q), t_hi);
        uint64_t mine = __ballot(q0 + lane < b.requests && b.ids[q] == adapter && lo_q < hi_q);
        for (; mine != 0; mine &= mine - 1) {
            const int from = __builtin_ctzll(mine);
            const int64_t lo = __builtin_amdgcn_readlane(lo_q, from), hi = __builtin_amdgcn_readlane(hi_q, from);
            int64_t t0 = lo + 4 * U * turn;
            for (; t0 < hi; t0 += 4 * U * LO_WAVES) {
                // tokens past the last read it again, as zeros; columns past N read the last one
                float xv[U][2], hv[U][RT];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const uint32_t t = (uint32_t) min((int64_t) (4 * u + quad), hi - 1 - t0);
                    const uint8_t* const xb = o.x.p + t0 * o.x.nb1 + n0 * 4;
                    if (whole) {
                        const f2u v = load_at<f2u>(xb, t * (uint32_t) o.x.nb1 + 8 * col);
                        xv[u][0] = v[0], xv[u][1] = v[1];
                    } else {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const uint32_t at = (uint32_t) min((int64_t) (2 * col + c), N - 1 - n0);
                            xv[u][c] = load_at<float>(xb, t * (uint32_t) o.x.nb1 + 4 * at);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < RT; ++j)
                        hv[u][j] = load_at<float>(o.h + t0 * R, 4 * (t * R + (uint32_t) min(r0 + 16 * j + col, R - 1)));
                }
                if constexpr (ROWS && RT <= 2) {
                    if (o.h_parts > 1) {
                        float more[L_G_PARTS - 1][U][RT];
#pragma unroll
                        for (int k = 1; k < L_G_PARTS; ++k) {
                            const float* const hk = o.h + (min(k, o.h_parts - 1) * b.T + t0) * R;
#pragma unroll
                            for (int u = 0; u < U; ++u) {
                                const uint32_t t = (uint32_t) min((int64_t) (4 * u + quad), hi - 1 - t0);
#pragma unroll
                                for (int j = 0; j < RT; ++j)
                                    more[k - 1][u][j] = load_at<float>(hk, 4 * (t * R + (uint32_t) min(r0 + 16 * j + col, R - 1)));
                            }
                        }
#pragma unroll
                        for (int k = 1; k < L_G_PARTS; ++k)
#pragma unroll
                            for (int u = 0; u < U; ++u)
#pragma unroll
                                for (int j = 0; j < RT; ++j) hv[u][j] += k < o.h_parts ? more[k - 1][u][j] : 0.f;
                    }
                }
                if (t0 + 4 * U > hi) {
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const bool in = t0 + 4 * u + quad < hi;
                        xv[u][0] = in ? xv[u][0] : 0.f, xv[u][1] = in ? xv[u][1] : 0.f;
#pragma unroll
                        for (int j = 0; j < RT; ++j) hv[u][j] = in ? hv[u][j] : 0.f;
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int j = 0; j < RT; ++j) acc[c][j] = mfma(xv[u][c], hv[u][j], acc[c][j]);
            }
            turn = (int) ((t0 - hi) / (4 * U));
        }
    }
    const float s = o.scaled ? b.scale[adapter] : 1.f;
    float* const d = o.d + adapter * o.d_adapter;
    float* const p = o.parts + ((int64_t) split * b.adapters + adapter) * N * R;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < RT; ++j) part[wave][j][lane] = acc[c][j];
        __syncthreads();
        for (int e = (int) threadIdx.x; e < RT * 256; e += LO_WAVES * 64) {
            const float sum = joined<LO_WAVES, RT>(part, e);
            const int l = (e >> 2) & 63, r = r0 + 16 * (e >> 8) + (l & 15);
            const int64_t at = n0 + 2 * (4 * (l >> 4) + (e & 3)) + c;
            if (r >= R || at >= N) continue;
            if (o.splits > 1) {
                p[ROWS ? r * N + at : at * R + r] = sum;
            } else {
                float* const q = d + (ROWS ? r * o.d_row + at : at * o.d_row + r);
                *q = o.accumulate ? *q + sum * s : sum * s;
            }
        }
    }
}

// The first launch of the backward pass: dB, then g = s B^T dy in parts of the long axis.
template <int TYPE, int RT>
__global__ __launch_bounds__(LO_WAVES * 64) void k_back_b(Outer o, int outers, Rows dy, Matrix bm, int R, Batch b, int parts,
                                                           int64_t part_len, float* __restrict__ g) {
    __shared__ ContractLds<TYPE, true, LO_WAVES, RT> lds;
    if ((int) blockIdx.x < outers) {
        outer_block<false, RT>(blockIdx.x, o, R, b, lds.part);
        return;
    }
    const int i = (int) blockIdx.x - outers, rank_blocks = (R + 16 * RT - 1) / (16 * RT);
    const Tile t = find_tile<LO_WAVES>(b, i / rank_blocks / parts);
    if (t.tokens == 0) return;
    const int r0 = i % rank_blocks * (16 * RT), part = i / rank_blocks % parts;
    const int64_t lo = part * part_len;
    g += part * b.T * R;
    if (t.adapter < 0) {
        zero_h(t, R, r0, 16 * RT, g, LO_WAVES * 64);
        return;
    }
    const float s = b.scale[t.adapter];
    contract_tile<TYPE, true, LO_WAVES, RT>(t, dy, bm, R, r0, lo, min(lo + part_len, dy.n), lds.stage, lds.part,
                                            [&](int tok, int r, float v) { g[(int64_t) (t.lo + tok) * R + r] = v * s; });
}

// The second: dA, then dx, `cols` columns of it a workgroup; those of the first ones store g if it came in parts.
template <int TYPE, int RT>
__global__ __launch_bounds__(LO_WAVES * 64) void k_back_a(Outer o, int outers, const float* __restrict__ g, int parts, Matrix am,
                                                           int R, Batch b, const uint8_t* base, size_t base_nb1, int64_t N,
                                                           uint8_t* dx, size_t dx_nb1, int cols, float* __restrict__ g_sum) {
    __shared__ union {
        Partial<LO_WAVES, RT> part;
        __attribute__((aligned(16))) float hs[h_floats<RT>];
    } lds;
    if ((int) blockIdx.x < outers) {
        outer_block<true, RT>(blockIdx.x, o, R, b, lds.part);
        return;
    }
    const int i = (int) blockIdx.x - outers, slices = (int) ((N + cols - 1) / cols);
    const Tile t = find_tile<LO_WAVES>(b, i / slices);
    if (t.tokens == 0) return;
    const int64_t n_lo = (int64_t) (i % slices) * cols;
    // (512 tokens, K = M = 4096, R 16, F32: 17 us, 18 without the early loads; with more tiles of the rank they cost registers:
    // R 32 20.0 us, 21.6 with them)
    typedef Expand<TYPE, true, LO_WAVES, RT, false, RT == 1> E;
    E e(t, am, R, base, base_nb1, N, dx, dx_nb1, n_lo, n_lo + cols, nullptr);
    e.start();
    stage_h<RT>(t, g, parts, b.T, R, 1.f, n_lo == 0 ? g_sum : nullptr, lds.hs, LO_WAVES * 64);
    e.run(lds.hs);
}

// Gradients whose tokens were split: the parts in order. dB's are in `first` blocks, dA's in the others.
__global__ __launch_bounds__(256) void k_back_join(Outer db, int first, Outer da, int R, Batch b) {
    const bool rows = (int) blockIdx.x >= first;
    const Outer o = rows ? da : db;
    const int64_t N = o.x.n, per = N * R, all = per * b.adapters;
    const int64_t i = (int64_t) (blockIdx.x - (rows ? first : 0)) * 256 + threadIdx.x;
    if (i >= all) return;
    float sum = 0.f;
    for (int k0 = 0; k0 < o.splits; k0 += 8) {  // eight loads under way
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = o.parts[min(k0 + k, o.splits - 1) * all + i];
#pragma unroll
        for (int k = 0; k < 8; ++k) sum += k0 + k < o.splits ? x[k] : 0.f;
    }
    const int64_t a = i / per, row = i % per / (rows ? N : R), at = i % per % (rows ? N : R);
    if (o.scaled) sum *= b.scale[a];
    float* const e = o.d + a * o.d_adapter + row * o.d_row + at;
    *e = o.accumulate ? *e + sum : sum;
}

struct Call {
    Matrix a, b;
    Batch batch;
    int type;
    int R;
    hipStream_t s;
    int64_t tiles() const { return std::min(batch.T, (batch.T + (int64_t) batch.requests * (LT - 1)) / LT); }
};

Call call_of(const trc_hip_lora_set& q, int64_t T, hipStream_t s) {
    const size_t es = q.a.type == TRC_HIP_TYPE_F32 ? 4 : 2;
    return {{q.a.data, (int64_t) (q.a.nb[1] / es), (int64_t) (q.a.nb[2] / es)},
            {q.b.data, (int64_t) (q.b.nb[1] / es), (int64_t) (q.b.nb[2] / es)},
            {(const int32_t*) q.start.data, (const int32_t*) q.adapter.data, (const float*) q.scale.data, T,
             (int32_t) q.adapter.ne[0], (int32_t) q.a.ne[2]},
            q.a.type, (int) q.a.ne[1], s};
}

Rows rows_of(const trc_hip_tensor& t) { return {(const uint8_t*) t.data, t.nb[1], t.ne[0]}; }

template <class F>
void with_type(int type, F&& f) {
    if (type == TRC_HIP_TYPE_F32) f(std::integral_constant<int, TRC_HIP_TYPE_F32>());
    if (type == TRC_HIP_TYPE_F16) f(std::integral_constant<int, TRC_HIP_TYPE_F16>());
    if (type == TRC_HIP_TYPE_BF16) f(std::integral_constant<int, TRC_HIP_TYPE_BF16>());
}
// f with the tiles of 16 that a rank is summed in at a time
template <class F>
void with_rank(int R, F&& f) {
    if (R <= 16) return f(std::integral_constant<int, 1>());
    if (R <= 32) return f(std::integral_constant<int, 2>());
    f(std::integral_constant<int, 4>());
}
int rank_blocks(int R) { return R <= 16 ? 1 : R <= 32 ? 1 : (R + LR - 1) / LR; }

int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// The long axis in parts where the tiles leave CUs idle, of 1024 or more each (512 or more takes as long); the
// parts' sums are kept in the stream's workspace. 256 tokens, K 4096, M 14336, R 64: 20 us, in one part 28.
int64_t contract_parts(const Call& c, int64_t N) {
    const int64_t blocks = c.tiles() * rank_blocks(c.R);
    int64_t parts = std::min(device_cus() / std::max(blocks, (int64_t) 1), N / 1024);
    const int64_t room = (int64_t) (qm_workspace_bytes() / sizeof(float)) / (c.batch.T * c.R);
    parts = std::min(parts, std::min(room, (int64_t) 16));
    return std::max(parts, (int64_t) 1);
}

int forward_apart(const Call& c, const trc_hip_tensor& x, const trc_hip_tensor* base, const trc_hip_tensor& h,
                  const trc_hip_tensor& dst) {
    const int64_t K = x.ne[0], M = dst.ne[0], parts = contract_parts(c, K);
    const int64_t len = parts > 1 ? round_up((K + parts - 1) / parts, 64) : K;
    float* sums = (float*) h.data;
    if (parts > 1) {
        uint8_t* ws = nullptr;
        const int rc = qm_stream_workspace(c.s, &ws);
        if (rc != TRC_HIP_OK) return rc;
        sums = (float*) ws;
    }
    with_type(c.type, [&](auto type) {
        with_rank(c.R, [&](auto rt) {
            hipLaunchKernelGGL((k_contract<decltype(type)::value, decltype(rt)::value>),
                               dim3((unsigned) c.tiles(), (unsigned) rank_blocks(c.R), (unsigned) parts), dim3(512), 0, c.s,
                               rows_of(x), c.a, c.R, c.batch, len, sums);
        });
    });
    int rc = check_launch("lora (contract)");
    if (rc != TRC_HIP_OK) return rc;
    // four workgroups a CU at a time, of at least 256 columns (a step of each wave): 1001 tokens, K 4096, M 14336, R 64
    // 43 us; two a CU 50, eight 43
    const int64_t slices = std::max(std::min(4 * device_cus() / c.tiles(), (M + 255) / 256), (int64_t) 1);
    const int cols = (int) round_up((M + slices - 1) / slices, 256);
    with_type(c.type, [&](auto type) {
        with_rank(c.R, [&](auto rt) {
            hipLaunchKernelGGL((k_expand<decltype(type)::value, decltype(rt)::value>),
                               dim3((unsigned) c.tiles(), (unsigned) ((M + cols - 1) / cols)), dim3(LE_THREADS), 0, c.s, sums,
                               (int) parts, c.b, c.R, c.batch, base != nullptr ? (const uint8_t*) base->data : nullptr,
                               base != nullptr ? base->nb[1] : (size_t) 0, M, (uint8_t*) dst.data, dst.nb[1],
                               parts > 1 ? (float*) h.data : nullptr, cols);
        });
    });
    return check_launch("lora (expand)");
}

// How a gradient's blocks are laid out: tokens split in three or more, 512 of an adapter's or more each, where that
// leaves half of the CUs to the other blocks of the launch, and while the parts fit into `room` floats at `ws`. One
// adapter, bfloat16, R 16, us with and without: K = M = 512, 16384 tokens 44 and 119, 4096 19.3 and 35, 2048 15.8 and 18.9;
// K = M = 2048, 4096 tokens in two parts 37 and 35.
Outer outer_of(const Call& c, const trc_hip_tensor& x, const float* h, const trc_hip_tensor& d, bool scaled, bool accumulate,
               float* ws, int64_t room) {
    Outer o{rows_of(x), h, 1, (float*) d.data, (int64_t) (d.nb[1] / 4), (int64_t) (d.nb[2] / 4), scaled, accumulate,
            0, 0, 1, c.batch.T, ws};
    o.col_blocks = (int) ((x.ne[0] + LO_COLS - 1) / LO_COLS);
    o.rank_blocks = rank_blocks(c.R);
    const int64_t blocks = o.blocks(c.batch.adapters), T = c.batch.T;
    int64_t n = std::min((int64_t) device_cus() / (2 * blocks), T / (512 * c.batch.adapters));
    n = std::min(n, room / (x.ne[0] * c.R * c.batch.adapters));
    if (n >= 3) {
        o.split_len = round_up((T + n - 1) / n, 64);
        o.splits = (int) ((T + o.split_len - 1) / o.split_len);
    }
    return o;
}

}  // namespace

int launch_lora(const trc_hip_lora_set& q, const trc_hip_tensor& x, const trc_hip_tensor* base, const trc_hip_tensor& h,
                const trc_hip_tensor& dst, hipStream_t s) {
    const Call c = call_of(q, x.ne[1], s);
    const int64_t K = x.ne[0], M = dst.ne[0], tiles = c.tiles();
    if (tiles * rank_blocks(c.R) > max_groups(L_WAVES * 64)) {
        return fail(TRC_HIP_E_SHAPE, "trc_hip_lora: %lld tiles of tokens", (long long) tiles);
    }
    // One launch, every workgroup of a tile making h for itself, unless two let a workgroup read so much less that a
    // second launch pays: of A and x, which two take in parts, over 300 KB where tiles are single tokens and over 120 KB
    // else (x counts as the 16 rows that a tile loads); of base and y, where CUs were idle, over 200 KB. Measured, in
    // us, one and two launches, K = M = 4096 but where said:
    //   64 single tokens, F16, R 24 (156 KB) 10.5 and 11.6, R 32 (204) 11.5 and 12.4, R 48 (300) 16.0 and 15.7
    //   128 tokens of 8 requests, F16, K 2048, R 16 (96 KB) 8.0 and 8.7, R 32 (128) 11.1 and 10.9; K 4096, R 8 (240) 11.5
    //   and 8.7; 64 of 32, R 8 (240) 11.1 and 9.5; but 512 of 2, M 2048, K 2048, R 16 (96) 10.4 and 9.3
    //   one adapter, F32, R 16, idle CUs: 3300 tokens (96 KB) 36.3 and 39.7, 2700 (172) 31.9 and 32.1, 2300 (222) 31.2
    //   and 29.4; but bfloat16, M 11008, 3300 tokens (258) 78 and 85
    const int64_t cus = device_cus(), slices = std::max(std::min(cus / tiles, (M + 255) / 256), (int64_t) 1);
    const bool single = c.batch.T <= c.batch.requests;
    const int64_t reads = K * (c.R * (c.type == TRC_HIP_TYPE_F32 ? 4 : 2) + (single ? 1 : LT) * 4);
    const int64_t saved = reads - reads / contract_parts(c, K);
    const int64_t idle = LT * 8 * M / slices * std::max(cus - tiles * slices, (int64_t) 0) / cus;
    if ((single ? 2 : 5) * saved + 3 * idle > 600 << 10) return forward_apart(c, x, base, h, dst);
    const int cols = (int) round_up((M + slices - 1) / slices, LE_COLS);
    with_type(c.type, [&](auto type) {
        with_rank(c.R, [&](auto rt) {
            constexpr int TYPE = decltype(type)::value, RT = decltype(rt)::value;
            hipLaunchKernelGGL((k_lora<TYPE, RT>), dim3((unsigned) tiles, (unsigned) ((M + cols - 1) / cols)),
                               dim3(L_WAVES * 64), 0, s, rows_of(x), c.a, c.b, c.R, c.batch,
                               base != nullptr ? (const uint8_t*) base->data : nullptr,
                               base != nullptr ? base->nb[1] : (size_t) 0, M, (uint8_t*) dst.data, dst.nb[1],
                               (float*) h.data, cols);
        });
    });
    return check_launch("lora");
}

int launch_lora_back(const trc_hip_lora_set& q, const trc_hip_tensor& x, const trc_hip_tensor& h, const trc_hip_tensor& dy,
                     const trc_hip_tensor& g, const trc_hip_tensor* base, const trc_hip_tensor* dx, const trc_hip_tensor& da,
                     const trc_hip_tensor& db, bool accumulate, hipStream_t s) {
    const Call c = call_of(q, x.ne[1], s);
    const int64_t K = x.ne[0], tiles = c.tiles();
    const int64_t half = (int64_t) (qm_workspace_bytes() / sizeof(float)) / 2;
    Outer ob = outer_of(c, dy, (const float*) h.data, db, true, accumulate, nullptr, half);
    Outer oa = outer_of(c, x, (const float*) g.data, da, false, accumulate, nullptr, half);
    if (ob.splits > 1 || oa.splits > 1) {
        uint8_t* ws = nullptr;
        const int rc = qm_stream_workspace(s, &ws);
        if (rc != TRC_HIP_OK) return rc;
        ob.parts = (float*) ws;
        oa.parts = (float*) ws + half;
    }
    const int64_t nb = ob.blocks(c.batch.adapters), na = oa.blocks(c.batch.adapters);
    // g in parts of 512 of the long axis or more, where CUs would be idle; they are summed where they are used. 512
    // tokens, F32, K = M = 4096, R 16: 17 us in three parts, 22 in one.
    int64_t ng = tiles * rank_blocks(c.R), parts = 1;
    float* sums = (float*) g.data;
    if (dx != nullptr && c.R <= 32 && ob.splits == 1 && oa.splits == 1 && nb < device_cus()) {
        parts = std::min((device_cus() - nb) / ng, dy.ne[0] / 512);
        parts = std::min(parts, std::min((int64_t) L_G_PARTS, half / (c.batch.T * c.R)));
        parts = std::max(parts, (int64_t) 1);
    }
    if (parts > 1) {
        uint8_t* ws = nullptr;
        const int rc = qm_stream_workspace(s, &ws);
        if (rc != TRC_HIP_OK) return rc;
        ng *= parts;
        sums = (float*) ws;
        oa.h = sums;
        oa.h_parts = (int) parts;
    }
    const int64_t part_len = round_up((dy.ne[0] + parts - 1) / parts, 64);
    // two workgroups a CU, of 1024 columns or more: 2048 tokens of three requests (one without an adapter), bfloat16,
    // K = M = 4096, R 64 51 us; one a CU 54, four of 512 56
    const int64_t slices = std::max(std::min(2 * device_cus() / tiles, (K + 1023) / 1024), (int64_t) 1);
    const int cols = (int) round_up((K + slices - 1) / slices, LE_COLS);
    const int64_t nx = dx != nullptr ? tiles * ((K + cols - 1) / cols) : 0;
    if (nb + ng > max_groups(LO_WAVES * 64) || na + nx > max_groups(LO_WAVES * 64)) {
        return fail(TRC_HIP_E_SHAPE, "trc_hip_lora_back: %lld workgroups", (long long) std::max(nb + ng, na + nx));
    }
    with_type(c.type, [&](auto type) {
        with_rank(c.R, [&](auto rt) {
            hipLaunchKernelGGL((k_back_b<decltype(type)::value, decltype(rt)::value>), dim3((unsigned) (nb + ng)),
                               dim3(LO_WAVES * 64), 0, s, ob, (int) nb, rows_of(dy), c.b, c.R, c.batch, (int) parts, part_len,
                               sums);
        });
    });
    int rc = check_launch("lora_back (dB, g)");
    if (rc != TRC_HIP_OK) return rc;
    with_type(c.type, [&](auto type) {
        with_rank(c.R, [&](auto rt) {
            hipLaunchKernelGGL((k_back_a<decltype(type)::value, decltype(rt)::value>), dim3((unsigned) (na + nx)),
                               dim3(LO_WAVES * 64), 0, s, oa, (int) na, sums, (int) parts, c.a, c.R, c.batch,
                               base != nullptr ? (const uint8_t*) base->data : nullptr,
                               base != nullptr ? base->nb[1] : (size_t) 0, K, dx != nullptr ? (uint8_t*) dx->data : nullptr,
                               dx != nullptr ? dx->nb[1] : (size_t) 0, cols, parts > 1 ? (float*) g.data : nullptr);
        });
    });
    rc = check_launch("lora_back (dA, dx)");
    if (rc != TRC_HIP_OK) return rc;
    auto joins = [&](const Outer& o) { return o.splits > 1 ? (o.x.n * c.R * c.batch.adapters + 255) / 256 : 0; };
    if (joins(ob) + joins(oa) == 0) return TRC_HIP_OK;
    hipLaunchKernelGGL(k_back_join, dim3((unsigned) (joins(ob) + joins(oa))), dim3(256), 0, s, ob, (int) joins(ob), oa, c.R,
                       c.batch);
    return check_launch("lora_back (join)");
}

}  // namespace trc_hip
