// Low-rank adapters of the requests of a batch beside the projection they share
// (Hu et al., "LoRA: Low-Rank Adaptation of Large Language Models", 2021), and their
// gradients. Request q holds tokens start[q] .. start[q+1]-1 and uses adapter a = ids[q]:
//
//   h_t  = A_a x_t              y_t  = base_t + s_a B_a h_t
//   g_t  = s_a B_a^T dy_t       dx_t = base_t + A_a^T g_t
//   dA_a = sum_t g_t x_t^T      dB_a = s_a sum_t dy_t h_t^T
//
// Three kernels serve all six, on v_mfma_f32_16x16x4_f32 (F32 products as exact as
// float FMAs; adapters in 16 bits are widened):
//   k_contract  h and g: a wide activation times a matrix of R rows or columns
//   k_expand    y and dx: base plus a matrix times h or g
//   k_outer     dA and dB: sums over tokens of outer products
// A workgroup of the first two takes 16 tokens of one request, so a request of one token
// costs one reading of its adapter and a long one reads it once per 16 tokens, from the L2.
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace trc_hip {

namespace {

constexpr int LT = 16;           // tokens of a tile
constexpr int LC_THREADS = 512;  // k_contract: 8 waves split the long axis
constexpr int LE_THREADS = 256;  // k_expand
constexpr int LE_COLS = 512;     // outputs of a workgroup's tokens
constexpr int LO_THREADS = 512;  // k_outer: 8 waves split the tokens
constexpr int LR = 64;           // rank of one pass, at most
constexpr int L_MAX_RANK = TRC_HIP_LORA_MAX_RANK;

// four elements whose address is only as aligned as one
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t h4u __attribute__((ext_vector_type(4), aligned(2)));

template <int TYPE>
struct Wt {
    typedef uint16_t Elem;
    static __device__ __forceinline__ float get(Elem x) {
        return TYPE == TRC_HIP_TYPE_F16 ? half_bits_to_float(x) : __builtin_bit_cast(float, (uint32_t) x << 16);
    }
    static __device__ __forceinline__ f4 get4(const Elem* p) {
        const h4u h = *(const h4u*) p;
        return f4{get(h[0]), get(h[1]), get(h[2]), get(h[3])};
    }
};
template <>
struct Wt<TRC_HIP_TYPE_F32> {
    typedef float Elem;
    static __device__ __forceinline__ float get(Elem x) { return x; }
    static __device__ __forceinline__ f4 get4(const Elem* p) { return *(const f4u*) p; }
};

struct Batch {
    const int32_t* start;
    const int32_t* ids;
    const float* scale;
    int64_t T;
    int32_t requests, adapters;
};

struct Tile {
    int64_t lo;   // first token
    int tokens;   // 0: none
    int adapter;  // -1: none
};

// Tile `index` of the batch, requests in order and each in tiles of LT tokens. Every lane
// of a wave has to be here. What start holds is only compared and clamped, so
// no value of it leads out of the T tokens.
__device__ __forceinline__ Tile find_tile(const Batch& b, int64_t index) {
    const int lane = (int) threadIdx.x & 63;
    for (int q0 = 0; q0 < b.requests; q0 += 64) {
        const int q = q0 + lane;
        int64_t lo = 0, hi = 0;
        if (q < b.requests) {
            lo = min(max((int64_t) b.start[q], (int64_t) 0), b.T);
            hi = min(max((int64_t) b.start[q + 1], lo), b.T);
        }
        const int64_t mine = (hi - lo + LT - 1) / LT;
        int64_t upto = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t v = __shfl_up(upto, d, 64);
            if (lane >= d) upto += v;
        }
        const uint64_t in = __ballot(index < upto);
        if (in != 0) {
            const int src = __ffsll((unsigned long long) in) - 1;
            const int64_t first = __shfl(lo, src, 64) + (index - __shfl(upto - mine, src, 64)) * LT;
            const int64_t end = __shfl(hi, src, 64);
            const int id = b.ids[q0 + src];
            return {first, (int) min(end - first, (int64_t) LT), id >= 0 && id < b.adapters ? id : -1};
        }
        index -= __shfl(upto, 63, 64);
    }
    return {0, 0, -1};
}

__device__ __forceinline__ f4 mfma(float a, float b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

struct Matrix {
    const void* p;
    int64_t row, adapter;  // strides in elements
};

// out[t][r] = scale sum_n x[t][n] W(n, r), where W(n, r) is w[r][n] (A) or, with OUTER,
// w[n][r] (B). Blocks: (tile, 64 of the rank, part of n); part p goes to out + p * T * R.
// A lane of the x operand holds token lane % 16 and of each 16 of n the four from
// 4 * (lane / 16) on, one per instruction; the weights' lanes hold column r = lane % 16 the
// same way, so the four products of a lane's vector need no shuffle. Lanes past the
// tile's tokens or past R read the last one and are not stored.
template <int TYPE, bool OUTER, int RT>
__global__ __launch_bounds__(LC_THREADS) void k_contract(const uint8_t* __restrict__ x, size_t x_nb1, int64_t N, Matrix wm,
                                                          int R, Batch b, bool scaled, int64_t part_len,
                                                          float* __restrict__ out) {
    typedef Wt<TYPE> W;
    constexpr int WAVES = LC_THREADS / 64;
    const Tile t = find_tile(b, blockIdx.x);
    if (t.tokens == 0) return;
    out += (int64_t) blockIdx.z * b.T * R;
    const int r0 = (int) blockIdx.y * LR;
    if (t.adapter < 0) {
        for (int i = (int) threadIdx.x; i < t.tokens * LR; i += LC_THREADS) {
            const int r = r0 + i % LR;
            if (r < R) out[(t.lo + i / LR) * R + r] = 0.f;
        }
        return;
    }
    const int lane = (int) threadIdx.x & 63, wave = (int) threadIdx.x >> 6, col = lane & 15, quad = lane >> 4;
    const float* const xt = (const float*) (x + (t.lo + min(col, t.tokens - 1)) * x_nb1);
    const typename W::Elem* const w = (const typename W::Elem*) wm.p + t.adapter * wm.adapter;
    const typename W::Elem* wr[RT];
#pragma unroll
    for (int j = 0; j < RT; ++j) wr[j] = w + (int64_t) min(r0 + 16 * j + col, R - 1) * (OUTER ? 1 : wm.row);
    f4 acc[RT];
#pragma unroll
    for (int j = 0; j < RT; ++j) acc[j] = f4{0.f, 0.f, 0.f, 0.f};
    const int64_t lo = (int64_t) blockIdx.z * part_len, hi = min(lo + part_len, N);
    auto weights = [&](int j, int64_t n) {
        if (!OUTER) return W::get4(wr[j] + n);
        f4 v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = W::get(wr[j][(n + k) * wm.row]);
        return v;
    };
    constexpr int U = 4;  // groups of 16 that are loaded together
    int64_t n = lo + wave * (16 * U) + 4 * quad;
    const int64_t whole = lo + (hi - lo) / (16 * U) * (16 * U);
    for (; n - 4 * quad < whole; n += WAVES * 16 * U) {
        f4 xv[U], wv[U][RT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            xv[u] = *(const f4u*) (xt + n + 16 * u);
#pragma unroll
            for (int j = 0; j < RT; ++j) wv[u][j] = weights(j, n + 16 * u);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int j = 0; j < RT; ++j) acc[j] = mfma(xv[u][k], wv[u][j][k], acc[j]);
    }
    // the rest, in groups of 16: both operands are 0 past the end, so nothing there counts
    for (n = whole + wave * 16; n < hi; n += WAVES * 16) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t at = n + 4 * quad + k;
            const float xk = at < hi ? xt[at] : 0.f;
#pragma unroll
            for (int j = 0; j < RT; ++j) acc[j] = mfma(xk, at < hi ? W::get(wr[j][OUTER ? at * wm.row : at]) : 0.f, acc[j]);
        }
    }
    __shared__ f4 part[WAVES][RT][64];
#pragma unroll
    for (int j = 0; j < RT; ++j) part[wave][j][lane] = acc[j];
    __syncthreads();
    const float s = scaled ? b.scale[t.adapter] : 1.f;
    for (int i = (int) threadIdx.x; i < RT * 64; i += LC_THREADS) {
        const int j = i >> 6, l = i & 63, r = r0 + 16 * j + (l & 15);
        f4 sum = part[0][j][l];
#pragma unroll
        for (int v = 1; v < WAVES; ++v) sum += part[v][j][l];
        if (r >= R) continue;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int tok = 4 * (l >> 4) + v;
            if (tok < t.tokens) out[(t.lo + tok) * R + r] = sum[v] * s;
        }
    }
}

// out[t][n] = base[t][n] + scale sum_r h[t][r] W(n, r): W(n, r) is w[n][r] (B) or, with
// OUTER, w[r][n] (A). Blocks: (tile, LE_COLS of n). h comes in `parts` parts that are
// summed here; where there is more than one, the workgroups of the first columns store the sum.
// The weights are the first operand, so a lane's four sums are neighbours in n of one token.
template <int TYPE, bool OUTER>
__global__ __launch_bounds__(LE_THREADS) void k_expand(const float* __restrict__ h, int parts, Matrix wm, int R, Batch b,
                                                        bool scaled, const uint8_t* base, size_t base_nb1, int64_t N,
                                                        uint8_t* out, size_t out_nb1, float* __restrict__ h_sum) {
    typedef Wt<TYPE> W;
    const Tile t = find_tile(b, blockIdx.x);
    if (t.tokens == 0) return;
    const int64_t n_lo = (int64_t) blockIdx.y * LE_COLS, n_hi = min(n_lo + LE_COLS, N);
    const int lane = (int) threadIdx.x & 63, wave = (int) threadIdx.x >> 6, col = lane & 15, quad = lane >> 4;
    const int Rp = (R + 15) / 16 * 16;
    // h of the tile, [token][r] with a row of 4 more floats than Rp: 16-byte rows that start on other banks
    __shared__ __attribute__((aligned(16))) float hs[LT * (L_MAX_RANK + 4)];
    const int hrow = Rp + 4;
    const float s = t.adapter >= 0 && scaled ? b.scale[t.adapter] : 1.f;
    for (int i = (int) threadIdx.x; i < LT * Rp; i += LE_THREADS) {
        const int tok = i / Rp, r = i % Rp;
        float v = 0.f;
        if (tok < t.tokens && r < R && t.adapter >= 0) {
            for (int p = 0; p < parts; ++p) v += h[((int64_t) p * b.T + t.lo + tok) * R + r];
        }
        if (h_sum != nullptr && blockIdx.y == 0 && tok < t.tokens && r < R) h_sum[(t.lo + tok) * R + r] = v;
        hs[tok * hrow + r] = v * s;
    }
    __syncthreads();
    const bool here = col < t.tokens;
    const int64_t tok = t.lo + (here ? col : 0);
    const float* const bt = base != nullptr ? (const float*) (base + tok * base_nb1) : nullptr;
    float* const ot = (float*) (out + tok * out_nb1);
    const typename W::Elem* const w = t.adapter >= 0 ? (const typename W::Elem*) wm.p + t.adapter * wm.adapter : nullptr;
    for (int64_t n0 = n_lo + wave * 16; n0 < n_hi; n0 += LE_THREADS / 64 * 16) {
        const int64_t n = n0 + 4 * quad;  // the first of this lane's four outputs
        f4 acc = {0.f, 0.f, 0.f, 0.f};
        f4 bv = acc;
        if (bt != nullptr && here) {
            if (n + 4 <= N) {
                bv = *(const f4u*) (bt + n);
            } else {
                for (int k = 0; n + k < N; ++k) bv[k] = bt[n + k];
            }
        }
        if (w != nullptr) {
            const int64_t nw = min(n0 + col, N - 1);  // this lane's row of weights
            for (int r = 4 * quad; r < Rp; r += 16) {
                const f4 hv = *(const f4*) (hs + col * hrow + r);
                f4 wv;
                if (!OUTER && r + 4 <= R) {
                    wv = W::get4(w + nw * wm.row + r);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        wv[k] = r + k < R ? W::get(OUTER ? w[(int64_t) (r + k) * wm.row + nw] : w[nw * wm.row + r + k]) : 0.f;
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) acc = mfma(wv[k], hv[k], acc);
            }
        }
        if (!here) continue;
        acc += bv;
        if (n + 4 <= N) {
            *(f4u*) (ot + n) = acc;
        } else {
            for (int k = 0; n + k < N; ++k) ot[n + k] = acc[k];
        }
    }
}

// d(n, r) (+)= scale sum_t x[t][n] h[t][r] over the tokens of one adapter's requests:
// d(n, r) is d[n][r] (dB), or d[r][n] with ROWS (dA). Blocks: (64 of n, 64 of the rank,
// adapter). Each wave takes four tokens at a time; a lane of x holds the four columns
// 4 * (lane % 16) .. + 3 of one token, which feed four accumulators.
template <bool ROWS, int RT>
__global__ __launch_bounds__(LO_THREADS) void k_outer(const uint8_t* __restrict__ x, size_t x_nb1, int64_t N,
                                                       const float* __restrict__ h, int R, Batch b, bool scaled, float* d,
                                                       int64_t d_row, int64_t d_adapter, bool accumulate) {
    constexpr int WAVES = LO_THREADS / 64;
    const int lane = (int) threadIdx.x & 63, wave = (int) threadIdx.x >> 6, col = lane & 15, quad = lane >> 4;
    const int64_t n0 = (int64_t) blockIdx.x * 64;
    const int r0 = (int) blockIdx.y * LR, adapter = (int) blockIdx.z;
    const int64_t n = n0 + 4 * col;  // this lane's columns of x
    f4 acc[4][RT];
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int j = 0; j < RT; ++j) acc[c][j] = f4{0.f, 0.f, 0.f, 0.f};
    for (int q = 0; q < b.requests; ++q) {
        if (b.ids[q] != adapter) continue;
        const int64_t lo = min(max((int64_t) b.start[q], (int64_t) 0), b.T);
        const int64_t hi = min(max((int64_t) b.start[q + 1], lo), b.T);
        for (int64_t t0 = lo + 4 * wave; t0 < hi; t0 += 4 * WAVES) {
            const int64_t t = t0 + quad;
            f4 xv = {0.f, 0.f, 0.f, 0.f};
            float hv[RT];
#pragma unroll
            for (int j = 0; j < RT; ++j) hv[j] = 0.f;
            if (t < hi) {
                const float* const xt = (const float*) (x + t * x_nb1);
                if (n + 4 <= N) {
                    xv = *(const f4u*) (xt + n);
                } else {
                    for (int k = 0; n + k < N; ++k) xv[k] = xt[n + k];
                }
#pragma unroll
                for (int j = 0; j < RT; ++j) hv[j] = h[t * R + min(r0 + 16 * j + col, R - 1)];
            }
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int j = 0; j < RT; ++j) acc[c][j] = mfma(xv[c], hv[j], acc[c][j]);
        }
    }
    // the waves' sums, joined in order, one accumulator of every wave at a time
    __shared__ f4 part[WAVES][RT][64];
    const float s = scaled ? b.scale[adapter] : 1.f;
    d += adapter * d_adapter;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < RT; ++j) part[wave][j][lane] = acc[c][j];
        __syncthreads();
        for (int i = (int) threadIdx.x; i < RT * 64; i += LO_THREADS) {
            const int j = i >> 6, l = i & 63, r = r0 + 16 * j + (l & 15);
            f4 sum = part[0][j][l];
#pragma unroll
            for (int v = 1; v < WAVES; ++v) sum += part[v][j][l];
            if (r >= R) continue;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int64_t at = n0 + 4 * (4 * (l >> 4) + v) + c;
                if (at >= N) continue;
                float* const p = d + (ROWS ? r * d_row + at : at * d_row + r);
                *p = accumulate ? *p + sum[v] * s : sum[v] * s;
            }
        }
    }
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

// The long axis in parts where the tiles leave CUs idle, of 1024 or more each; the
// parts' sums are kept in the stream's workspace.
int64_t contract_parts(const Call& c, int64_t N) {
    const int64_t blocks = c.tiles() * ((c.R + LR - 1) / LR);
    int64_t parts = std::min(device_cus() / std::max(blocks, (int64_t) 1), N / 1024);
    const int64_t room = (int64_t) (qm_workspace_bytes() / sizeof(float)) / (c.batch.T * c.R);
    parts = std::min(parts, std::min(room, (int64_t) 16));
    return std::max(parts, (int64_t) 1);
}

template <bool OUTER>
int contract(const Call& c, const trc_hip_tensor& x, const Matrix& w, bool scaled, int64_t parts, float* out) {
    const int64_t N = x.ne[0];
    const int64_t len = parts > 1 ? ((N + parts - 1) / parts + 63) / 64 * 64 : N;
    const dim3 grid((unsigned) c.tiles(), (unsigned) ((c.R + LR - 1) / LR), (unsigned) parts);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(LC_THREADS), 0, c.s, (const uint8_t*) x.data, x.nb[1], N, w, c.R, c.batch, scaled,
                           len, out);
    };
    auto ranks = [&](auto type) {
        constexpr int TYPE = decltype(type)::value;
        if (c.R <= 16) return go(k_contract<TYPE, OUTER, 1>);
        if (c.R <= 32) return go(k_contract<TYPE, OUTER, 2>);
        return go(k_contract<TYPE, OUTER, 4>);
    };
    if (c.type == TRC_HIP_TYPE_F32) ranks(std::integral_constant<int, TRC_HIP_TYPE_F32>());
    if (c.type == TRC_HIP_TYPE_F16) ranks(std::integral_constant<int, TRC_HIP_TYPE_F16>());
    if (c.type == TRC_HIP_TYPE_BF16) ranks(std::integral_constant<int, TRC_HIP_TYPE_BF16>());
    return check_launch("lora (contract)");
}

template <bool OUTER>
int expand(const Call& c, const float* h, int64_t parts, const Matrix& w, bool scaled, const trc_hip_tensor* base,
           const trc_hip_tensor& out, float* h_sum) {
    const int64_t N = out.ne[0];
    const dim3 grid((unsigned) c.tiles(), (unsigned) ((N + LE_COLS - 1) / LE_COLS));
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(LE_THREADS), 0, c.s, h, (int) parts, w, c.R, c.batch, scaled,
                           base != nullptr ? (const uint8_t*) base->data : nullptr, base != nullptr ? base->nb[1] : (size_t) 0, N,
                           (uint8_t*) out.data, out.nb[1], parts > 1 ? h_sum : nullptr);
    };
    if (c.type == TRC_HIP_TYPE_F32) go(k_expand<TRC_HIP_TYPE_F32, OUTER>);
    if (c.type == TRC_HIP_TYPE_F16) go(k_expand<TRC_HIP_TYPE_F16, OUTER>);
    if (c.type == TRC_HIP_TYPE_BF16) go(k_expand<TRC_HIP_TYPE_BF16, OUTER>);
    return check_launch("lora (expand)");
}

template <bool ROWS>
int outer(const Call& c, const trc_hip_tensor& x, const float* h, bool scaled, const trc_hip_tensor& d, bool accumulate) {
    const int64_t N = x.ne[0];
    const dim3 grid((unsigned) ((N + 63) / 64), (unsigned) ((c.R + LR - 1) / LR), (unsigned) c.batch.adapters);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(LO_THREADS), 0, c.s, (const uint8_t*) x.data, x.nb[1], N, h, c.R, c.batch, scaled,
                           (float*) d.data, (int64_t) (d.nb[1] / 4), (int64_t) (d.nb[2] / 4), accumulate);
    };
    if (c.R <= 16) {
        go(k_outer<ROWS, 1>);
    } else if (c.R <= 32) {
        go(k_outer<ROWS, 2>);
    } else {
        go(k_outer<ROWS, 4>);
    }
    return check_launch("lora (gradients)");
}

int parts_of(const Call& c, int64_t N, float* whole, int64_t* parts, float** out) {
    *parts = contract_parts(c, N);
    *out = whole;
    if (*parts == 1) return TRC_HIP_OK;
    uint8_t* ws = nullptr;
    const int rc = qm_stream_workspace(c.s, &ws);
    *out = (float*) ws;
    return rc;
}

}  // namespace

int launch_lora(const trc_hip_lora_set& q, const trc_hip_tensor& x, const trc_hip_tensor* base, const trc_hip_tensor& h,
                const trc_hip_tensor& dst, hipStream_t s) {
    const Call c = call_of(q, x.ne[1], s);
    int64_t parts = 1;
    float* sums = nullptr;
    int rc = parts_of(c, x.ne[0], (float*) h.data, &parts, &sums);
    if (rc != TRC_HIP_OK) return rc;
    rc = contract<false>(c, x, c.a, false, parts, sums);
    if (rc != TRC_HIP_OK) return rc;
    return expand<false>(c, sums, parts, c.b, true, base, dst, (float*) h.data);
}

int launch_lora_back(const trc_hip_lora_set& q, const trc_hip_tensor& x, const trc_hip_tensor& h, const trc_hip_tensor& dy,
                     const trc_hip_tensor& g, const trc_hip_tensor* base, const trc_hip_tensor* dx, const trc_hip_tensor& da,
                     const trc_hip_tensor& db, bool accumulate, hipStream_t s) {
    const Call c = call_of(q, x.ne[1], s);
    // (g has to be whole before dA reads it, so the long axis is never in parts here)
    int rc = contract<true>(c, dy, c.b, true, 1, (float*) g.data);
    if (rc != TRC_HIP_OK) return rc;
    if (dx != nullptr) {
        rc = expand<true>(c, (const float*) g.data, 1, c.a, false, base, *dx, nullptr);
        if (rc != TRC_HIP_OK) return rc;
    }
    rc = outer<false>(c, dy, (const float*) h.data, true, db, accumulate);
    if (rc != TRC_HIP_OK) return rc;
    return outer<true>(c, x, (const float*) g.data, false, da, accumulate);
}

}  // namespace trc_hip
