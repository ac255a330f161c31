// y = W x and dx = W^T dy for a weight in 8-bit floating point with a scale for each 128 x 128 block and activations (or
// gradients) quantized the same way, each token's in blocks of 128:
//
//   y[m,n]  = sum_b ws[m/128,b] 2^e[n,b] sum_{k in block b} w[m,k] x[n,k]
//   dx[k,n] = sum_b ws[b,k/128] 2^e[n,b] sum_{m in block b} w[m,k] g[n,m]
//
// Codes are multiplied in binary16, which holds all of them and whose products are exact, with sums in 32 bits: 1e-7 off. (The
// 8-bit matrix instructions are twice as fast, or as fast, but add eight products with some 12 bits below the largest:
// 6e-4 of a sum's magnitudes in a search, which a result of 16 bits shows.) A block's sum is scaled in 32 bits.
//
// A weight's scales lie on its rows' blocks both ways, so the way back reads the same bytes, turned on their way from LDS
// (ds_read_tr8). Bound by the matrix units, power and what does not overlap: 4096 tokens 4096 -> 14336 with bfloat16 results 417 us
// (1.15 PFLOP/s; 437 at least and 470 in the median under the profiler, where the clock falls; the vendor library's bfloat16
// product of that size 390 to 405, 1.38 PFLOP/s at 8192 x 8192 x 8192), back 2048 tokens 14336 <- 4096 218 (1.10); F32 results, 2048
// tokens 4096 -> 4096, 65 (1.06; 70 under the profiler; the products and the reads from LDS alone took 51).
#include "fp8_mm.h"

namespace trc_hip {

#define F8_DECLARE(BM, BN, WM, WN, KG, STAGES, TRANS, POW2) \
    template <>                                         \
    void f8_tiles_launch<BM, BN, WM, WN, KG, STAGES, TRANS, POW2>(const F8Tiles& t, unsigned parts, hipStream_t s);
#define F8_DECLARE_ALL(BM, BN, WM, WN, KG, STAGES)       \
    F8_DECLARE(BM, BN, WM, WN, KG, STAGES, false, false) \
    F8_DECLARE(BM, BN, WM, WN, KG, STAGES, false, true)  \
    F8_DECLARE(BM, BN, WM, WN, KG, STAGES, true, false)  \
    F8_DECLARE(BM, BN, WM, WN, KG, STAGES, true, true)

F8_DECLARE_ALL(128, 128, 2, 2, 1, 2)
F8_DECLARE_ALL(128, 64, 2, 2, 2, 3)
F8_DECLARE_ALL(64, 64, 2, 2, 2, 2)
F8_DECLARE_ALL(64, 64, 2, 2, 2, 3)

namespace {

constexpr int JOIN_THREADS = 256;

// The parts' sums added in their order, four rows of a token per thread.
__global__ __launch_bounds__(JOIN_THREADS) void k_f8_join(const float* __restrict__ sums, int64_t nb1, int64_t N, int64_t rows, int parts,
                                                           uint32_t quads, uint8_t* __restrict__ y, int64_t y_nb1, int y_type) {
    const uint32_t at = blockIdx.x * JOIN_THREADS + threadIdx.x, n = at / quads, r = (at - n * quads) * 4;
    if (n >= N) return;
    f4 v = {0.f, 0.f, 0.f, 0.f};
    for (int p = 0; p < parts; ++p) v += *(const f4*) (sums + ((int64_t) p * N + n) * nb1 + r);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (r + k >= rows) break;
        if (y_type == TRC_HIP_TYPE_F32) ((float*) (y + n * y_nb1))[r + k] = v[k];
        else ((uint16_t*) (y + n * y_nb1))[r + k] = f8_bits(y_type, v[k]);
    }
}

template <int BM, int BN, int WM, int WN, int KG, int STAGES>
void launch(const F8Tiles& t, bool trans, unsigned parts, hipStream_t s) {
    const bool pow2 = !t.a.ws_float;
    auto* const f = trans ? (pow2 ? f8_tiles_launch<BM, BN, WM, WN, KG, STAGES, true, true> : f8_tiles_launch<BM, BN, WM, WN, KG, STAGES, true, false>)
                          : (pow2 ? f8_tiles_launch<BM, BN, WM, WN, KG, STAGES, false, true>
                                  : f8_tiles_launch<BM, BN, WM, WN, KG, STAGES, false, false>);
    f(t, parts, s);
}

}  // namespace

int launch_f8_product(const F8Args& a, bool trans, hipStream_t s) {
    // Up to 64 tokens a workgroup with 16 of the weight's rows has all of K, and reads all tokens: its time grows with
    // K, with tokens and with the rounds of workgroups. Tiles of 64 rows read the tokens less often; where few of them leave a
    // long sum in parts, joining those costs some 14 steps. F8_FUSED tokens are added up as by the kernel that quantizes them
    // itself (K, M, tokens, us so and in tiles; joined: 4096, 4096, 48 10.8 and 10.9, 64 13.7 and 11.4, 14336, 4096, 16 15.8 and
    // 16.6, 32 22.0 and 16.9, 8192, 8192, 8 15.9 and 17.5, 16 18.2 and 17.7, 32 25.7 and 18.2; not joined: 2048, 2048, 64 8.0 and
    // 8.7, 1024, 8192, 32 5.8 and 6.1, 48 7.2 and 6.2, 2048, 6000, 32 8.3 and 8.7, 48 10.4 and 8.8, 4096, 14336, 4 16.1 and 14.2,
    // 16 18.9 and 14.3, 1000, 777, 64 6.1 and 6.2).
    const int64_t cus = device_cus(), n16 = (a.N + 15) / 16 * 16, rounds = ((a.M + 15) / 16 + cus - 1) / cus;
    const bool joined = (a.M + 63) / 64 * 2 <= cus && a.K > 21 * F8_BLOCK;
    const bool many = a.N > F8_FUSED && (joined ? n16 > 16 && rounds * a.K * n16 > 240000 : rounds * n16 > 64 || rounds > 3);
    if (!trans && a.N <= TRC_HIP_FP8_MATVEC_MAX_N && !many) return launch_f8_skinny(a, s);
    F8Tiles t{};
    t.a = a;
    t.rows = trans ? a.K : a.M;
    t.steps = (int) (((trans ? a.M : a.K) + F8_BLOCK - 1) / F8_BLOCK);
    auto tiles = [&](int64_t edge) { return ((t.rows + edge - 1) / edge) * ((a.N + edge - 1) / edge); };
    // Which tiles: 64 x 64 up to one a CU, else 128 x 64 up to one a CU, else 128 x 128, but 64 x 64 again while three CUs
    // in four would not have one of those (K, M, tokens, us in tiles of 64, 128 x 64 and 128: 4096, 4096, 512 26.2, 24.2, 37.9,
    // 777 45.0, 41.1, 38.1, 1000, 6000, 400 13.6, 17.2, 14.3).
    const int64_t high = (t.rows + 127) / 128 * ((a.N + 63) / 64);
    const bool by_128 = tiles(64) > cus && high <= cus;
    const int edge = tiles(64) <= cus || by_128 || tiles(128) * 4 < cus * 3 ? 64 : 128;
    if (tiles(edge) > max_groups(512) - 8) return fail(TRC_HIP_E_SHAPE, "trc_hip_fp8_mul_mat: %lld tiles", (long long) tiles(edge));
    t.tm = by_128 ? (int) ((t.rows + 127) / 128) : (int) ((t.rows + edge - 1) / edge);
    t.tn = (int) ((a.N + edge - 1) / edge);
    // Few tiles: the sum in parts of 8 steps or more, where each is 14 steps or more short of the whole, which is what joining
    // them takes (tiles, steps, us whole and in parts: 26, 8 6.0 and 7.5, 16 8.6 and 8.3, 24 11.2 and 9.2, 112 39.7 and 13.8;
    // 128, 24 11.5 and 11.6, 32 14.3 and 13.1).
    int64_t parts = 1;
    size_t used = 0;
    if (edge == 64 && tiles(64) * 2 <= cus) {
        t.sums_nb1 = (t.rows + 3) / 4 * 4;
        // (activations that trc_hip_fp8_matvec holds there, room for them in every call: as many parts, the same bits)
        used = trans || a.N > TRC_HIP_FP8_MATVEC_MAX_N ? 0 : (f8_held(a.K, a.N) + 255) / 256 * 256;
        const size_t room = qm_workspace_bytes();
        const int64_t fit = (int64_t) ((used < room ? room - used : 0) / 4) / (a.N * t.sums_nb1);
        parts = cus / tiles(64);
        if (parts > (t.steps + 7) / 8) parts = (t.steps + 7) / 8;
        if (parts > fit) parts = fit;
        if (parts < 1) parts = 1;
    }
    t.part_steps = (int) (((t.steps + parts - 1) / parts + 3) / 4 * 4);
    if (t.steps - t.part_steps < 14) t.part_steps = t.steps;
    parts = (t.steps + t.part_steps - 1) / t.part_steps;
    if (parts > 1) {
        uint8_t* ws = nullptr;
        const int rc = qm_stream_workspace(s, &ws);
        if (rc != TRC_HIP_OK) return rc;
        t.sums = (float*) (ws + used);
    }
    const unsigned p = (unsigned) parts;
    if (edge == 128) launch<128, 128, 2, 2, 1, 2>(t, trans, p, s);
    else if (by_128) launch<128, 64, 2, 2, 2, 3>(t, trans, p, s);
    else if (t.tm * t.tn > cus) launch<64, 64, 2, 2, 2, 2>(t, trans, p, s);
    // (three stages where a CU has one workgroup: four took 2 to 5 % longer at 1 to 64 tokens of K and M from 777 to 14336)
    else launch<64, 64, 2, 2, 2, 3>(t, trans, p, s);
    const int rc = check_launch("fp8_mul_mat");
    if (rc != TRC_HIP_OK || parts == 1) return rc;
    const int64_t quads = t.sums_nb1 / 4;
    hipLaunchKernelGGL(k_f8_join, dim3((unsigned) ((a.N * quads + JOIN_THREADS - 1) / JOIN_THREADS)), dim3(JOIN_THREADS), 0, s, t.sums,
                       t.sums_nb1, a.N, t.rows, (int) parts, (uint32_t) quads, a.y, a.y_nb1, a.y_type);
    return check_launch("fp8_mul_mat (join)");
}

}  // namespace trc_hip
