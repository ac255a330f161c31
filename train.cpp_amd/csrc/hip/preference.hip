// The loss that ranks a chosen answer above a rejected one (Rafailov et al., "Direct
// Preference Optimization", 2023), over logits, and the logits' gradient.
//
//   lse_t = log sum_v exp(l_tv)           L_s = sum over sequence s of (l_t,label - lse_t)
//   z_i = beta ((L_2i - ref_2i) - (L_2i+1 - ref_2i+1))
//   loss = mean_i  -(1 - e) log sigma(z_i) - e log sigma(-z_i)
//   slope_i = d/dz_i = e sigma(z_i) - (1 - e) sigma(-z_i)
//   dl_tv = dloss (+-) beta / P slope_i (1[v = label_t] - exp(l_tv - lse_t))
//
// Three launches: the rows' log-sums (each row read once, with a running maximum and
// sum), one workgroup over the pairs, and the gradient (each row read and written once).
// All three are bound by memory; the gradient cannot begin before the pair's last row is
// summed, so the logits are read twice.
#include "common.h"

namespace trc_hip {

namespace {

constexpr int PF_THREADS = 256;
constexpr int PF_JOIN_THREADS = 1024;
constexpr int PF_MAX_PARTS = 64;  // parts of a row, at most
constexpr float LOG2E = 1.44269504088896340736f;

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
        *(f4u*) p = v;
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
        *(h8u*) p = v;
    }
};
template <>
struct Row<TRC_HIP_TYPE_F16> : Row16<TRC_HIP_TYPE_F16> {};
template <>
struct Row<TRC_HIP_TYPE_BF16> : Row16<TRC_HIP_TYPE_BF16> {};

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }

// A maximum and the sum of exponentials taken from it. A maximum of -inf (nothing yet,
// or only -inf) is subtracted as 0, so that exp(-inf - m) is 0 and not NaN; infinities
// and NaNs reach the sum.
struct Soft {
    float m, s;
};
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ Soft join(Soft a, Soft b) {
    const float m = fmaxf(a.m, b.m), base = base_of(m);
    return {m, a.s * exp_of(a.m - base) + b.s * exp_of(b.m - base)};
}
__device__ __forceinline__ Soft wave_join(Soft a) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) a = join(a, {__shfl_xor(a.m, d, 64), __shfl_xor(a.s, d, 64)});
    return a;
}

// Rows whose label is negative are not counted: they are not read, and their lse is 0.
// gridDim.y parts of `len` elements each; one part writes lse, more write (m, s) to parts.
template <int TYPE>
__global__ __launch_bounds__(PF_THREADS) void k_pref_rows(const uint8_t* __restrict__ logits, size_t nb1, int64_t V,
                                                           const int32_t* __restrict__ labels, int64_t len,
                                                           float* __restrict__ lse, Soft* __restrict__ parts) {
    typedef Row<TYPE> R;
    constexpr int VEC = R::VEC, U = 4;
    const int64_t row = blockIdx.x;
    if (labels[row] < 0) {
        if (blockIdx.y == 0 && threadIdx.x == 0) lse[row] = 0.f;
        return;
    }
    const typename R::Elem* const p = (const typename R::Elem*) (logits + row * nb1);
    const int64_t lo = (int64_t) blockIdx.y * len, hi = lo + len < V ? lo + len : V;
    Soft a = {-INFINITY, 0.f};
    int64_t i = lo + (int) threadIdx.x * VEC;
    for (; i + (U - 1) * PF_THREADS * VEC + VEC <= hi; i += U * PF_THREADS * VEC) {
        float x[U][VEC];
#pragma unroll
        for (int u = 0; u < U; ++u) R::load(p + i + u * PF_THREADS * VEC, x[u]);
        float m = a.m;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < VEC; ++k) m = fmaxf(m, x[u][k]);
        const float base = base_of(m);
        float s = a.s * exp_of(a.m - base);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < VEC; ++k) s += exp_of(x[u][k] - base);
        a = {m, s};
    }
    for (; i < hi; i += PF_THREADS * VEC) {
        if (i + VEC <= hi) {
            float x[VEC], m = a.m;
            R::load(p + i, x);
#pragma unroll
            for (int k = 0; k < VEC; ++k) m = fmaxf(m, x[k]);
            const float base = base_of(m);
            float s = a.s * exp_of(a.m - base);
#pragma unroll
            for (int k = 0; k < VEC; ++k) s += exp_of(x[k] - base);
            a = {m, s};
        } else {
            for (int64_t j = i; j < hi; ++j) a = join(a, {R::get(p[j]), 1.f});
        }
    }
    __shared__ Soft w[PF_THREADS / 64];
    a = wave_join(a);
    if (((int) threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = a;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int k = 1; k < PF_THREADS / 64; ++k) a = join(a, w[k]);
    if (gridDim.y == 1) {
        lse[row] = a.m + logf(a.s);
    } else {
        parts[row * gridDim.y + blockIdx.y] = a;
    }
}

// One workgroup: the rows' parts joined where there are any, then a wave for each pair.
// The tokens' log-probabilities and the pair's terms are summed in 64 bits, each
// sum in one order: a sequence's sum is far larger than the ratios that come of it.
template <int TYPE>
__global__ __launch_bounds__(PF_JOIN_THREADS) void k_pref_pairs(
    const uint8_t* __restrict__ logits, size_t nb1, int64_t V, int64_t T, const int32_t* __restrict__ labels,
    const int32_t* __restrict__ start, int64_t pairs, const float* __restrict__ ref, float beta, float smooth, int n_parts,
    const Soft* __restrict__ parts, float* lse, float* __restrict__ logp, float* __restrict__ slope, float* __restrict__ loss) {
    typedef Row<TYPE> R;
    if (n_parts > 1) {
        for (int64_t t = threadIdx.x; t < T; t += PF_JOIN_THREADS) {
            if (labels[t] < 0) continue;
            Soft a = parts[t * n_parts];
            for (int k = 1; k < n_parts; ++k) a = join(a, parts[t * n_parts + k]);
            lse[t] = a.m + logf(a.s);
        }
        __syncthreads();
    }
    __shared__ double total[PF_JOIN_THREADS / 64];
    const int lane = (int) threadIdx.x & 63, wave = (int) threadIdx.x >> 6;
    double mine = 0.0;
    for (int64_t i = wave; i < pairs; i += PF_JOIN_THREADS / 64) {
        double L[2];
        for (int k = 0; k < 2; ++k) {
            const int64_t lo = min(max((int64_t) start[2 * i + k], (int64_t) 0), T);
            const int64_t hi = min(max((int64_t) start[2 * i + k + 1], lo), T);
            double sum = 0.0;
            for (int64_t t = lo + lane; t < hi; t += 64) {
                const int32_t y = labels[t];
                if (y < 0) continue;
                const float l = y < V ? R::get(((const typename R::Elem*) (logits + t * nb1))[y]) : NAN;
                sum += (double) l - (double) lse[t];
            }
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d, 64);
            L[k] = sum;
        }
        if (lane == 0) {
            logp[2 * i] = (float) L[0];
            logp[2 * i + 1] = (float) L[1];
            const double z = (double) beta * ((L[0] - (double) ref[2 * i]) - (L[1] - (double) ref[2 * i + 1]));
            const double e = (double) smooth, tail = log1p(exp(-fabs(z)));
            const double up = fmax(-z, 0.0) + tail, down = fmax(z, 0.0) + tail;  // -log sigma(z), -log sigma(-z)
            // (e = 0 takes no part of an infinite term)
            mine += z != z ? z : (1.0 - e) * up + (e == 0.0 ? 0.0 : e * down);
            slope[i] = (float) (e / (1.0 + exp(-z)) - (1.0 - e) / (1.0 + exp(z)));
        }
    }
    if (lane == 0) total[wave] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        double sum = 0.0;
        for (int k = 0; k < PF_JOIN_THREADS / 64; ++k) sum += total[k];
        loss[0] = (float) (sum / (double) pairs);
    }
}

// The sequence that holds row t: the last s with start[s] <= t, -1 if t is in none.
__device__ __forceinline__ int64_t sequence_of(const int32_t* start, int64_t n, int64_t t) {
    if (t < start[0] || t >= start[n]) return -1;
    int64_t lo = 0, hi = n;  // start[lo] <= t < start[hi]
    while (hi - lo > 1) {
        const int64_t mid = (lo + hi) >> 1;
        if (start[mid] <= t) {
            lo = mid;
        } else {
            hi = mid;
        }
    }
    return lo;
}

template <int TYPE>
__global__ __launch_bounds__(PF_THREADS) void k_pref_back(const uint8_t* logits, size_t nb1, int64_t V,
                                                           const int32_t* __restrict__ labels,
                                                           const int32_t* __restrict__ start, int64_t pairs,
                                                           const float* __restrict__ lse, const float* __restrict__ slope,
                                                           const float* __restrict__ dloss, float beta, int64_t len,
                                                           uint8_t* dlogits, size_t dnb1) {
    typedef Row<TYPE> R;
    constexpr int VEC = R::VEC, U = 4;
    const int64_t row = blockIdx.x;
    const int32_t y = labels[row];
    const int64_t seq = y < 0 ? -1 : sequence_of(start, 2 * pairs, row);
    const typename R::Elem* const p = (const typename R::Elem*) (logits + row * nb1);
    typename R::Elem* const d = (typename R::Elem*) (dlogits + row * dnb1);
    const int64_t lo = (int64_t) blockIdx.y * len, hi = lo + len < V ? lo + len : V;
    int64_t i = lo + (int) threadIdx.x * VEC;
    if (seq < 0) {  // not counted: zeros, whatever the logits hold
        float z[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) z[k] = 0.f;
        for (; i < hi; i += PF_THREADS * VEC) {
            if (i + VEC <= hi) {
                R::store(d + i, z);
            } else {
                for (int64_t j = i; j < hi; ++j) d[j] = R::put(0.f);
            }
        }
        return;
    }
    const float w = (float) ((double) slope[seq >> 1] * (double) beta / (double) pairs) * dloss[0] * ((seq & 1) ? -1.f : 1.f);
    const float base = lse[row];
    auto grad = [&](float l, int64_t v) { return w * ((v == y ? 1.f : 0.f) - exp_of(l - base)); };
    for (; i + (U - 1) * PF_THREADS * VEC + VEC <= hi; i += U * PF_THREADS * VEC) {
        float x[U][VEC];
#pragma unroll
        for (int u = 0; u < U; ++u) R::load(p + i + u * PF_THREADS * VEC, x[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t at = i + u * PF_THREADS * VEC;
#pragma unroll
            for (int k = 0; k < VEC; ++k) x[u][k] = grad(x[u][k], at + k);
            R::store(d + at, x[u]);
        }
    }
    for (; i < hi; i += PF_THREADS * VEC) {
        if (i + VEC <= hi) {
            float x[VEC];
            R::load(p + i, x);
#pragma unroll
            for (int k = 0; k < VEC; ++k) x[k] = grad(x[k], i + k);
            R::store(d + i, x);
        } else {
            for (int64_t j = i; j < hi; ++j) d[j] = R::put(grad(R::get(p[j]), j));
        }
    }
}

// Parts of a row, and their length: whole rows while there are rows for every CU
// several times over, else parts of 4096 elements or more.
int64_t part_length(int64_t V, int64_t T) {
    const int64_t wanted = ((int64_t) device_cus() * 8 + T - 1) / T;
    const int64_t most = V / 4096;
    int64_t parts = wanted < most ? wanted : most;
    if (parts > PF_MAX_PARTS) parts = PF_MAX_PARTS;
    if (parts < 2) return V;
    return ((V + parts - 1) / parts + 7) / 8 * 8;
}

template <int TYPE>
int forward(const trc_hip_tensor& l, const int32_t* labels, const int32_t* start, int64_t pairs, const float* ref, float beta,
            float smooth, float* lse, float* logp, float* slope, float* loss, hipStream_t s) {
    const int64_t V = l.ne[0], T = l.ne[1];
    int64_t len = part_length(V, T);
    int64_t n = (V + len - 1) / len;
    uint8_t* ws = nullptr;
    if (n > 1) {
        const int rc = qm_stream_workspace(s, &ws);
        if (rc != TRC_HIP_OK) return rc;
        if ((size_t) (n * T) * sizeof(Soft) > qm_workspace_bytes()) {  // rows enough without parts
            len = V;
            n = 1;
        }
    }
    hipLaunchKernelGGL(k_pref_rows<TYPE>, dim3((unsigned) T, (unsigned) n), dim3(PF_THREADS), 0, s, (const uint8_t*) l.data,
                       l.nb[1], V, labels, len, lse, (Soft*) ws);
    const int rc = check_launch("preference_loss (rows)");
    if (rc != TRC_HIP_OK) return rc;
    hipLaunchKernelGGL(k_pref_pairs<TYPE>, dim3(1), dim3(PF_JOIN_THREADS), 0, s, (const uint8_t*) l.data, l.nb[1], V, T, labels,
                       start, pairs, ref, beta, smooth, (int) n, (const Soft*) ws, lse, logp, slope, loss);
    return check_launch("preference_loss (pairs)");
}

template <int TYPE>
int backward(const trc_hip_tensor& l, const int32_t* labels, const int32_t* start, int64_t pairs, const float* lse,
             const float* slope, const float* dloss, float beta, const trc_hip_tensor& d, hipStream_t s) {
    const int64_t V = l.ne[0], T = l.ne[1];
    const int64_t len = part_length(V, T), n = (V + len - 1) / len;
    hipLaunchKernelGGL(k_pref_back<TYPE>, dim3((unsigned) T, (unsigned) n), dim3(PF_THREADS), 0, s, (const uint8_t*) l.data,
                       l.nb[1], V, labels, start, pairs, lse, slope, dloss, beta, len, (uint8_t*) d.data, d.nb[1]);
    return check_launch("preference_loss_back");
}

}  // namespace

int launch_preference_loss(const trc_hip_tensor& l, const int32_t* labels, const int32_t* start, int64_t pairs,
                           const float* ref, float beta, float smooth, float* lse, float* logp, float* slope, float* loss,
                           hipStream_t s) {
    if (l.ne[1] > max_groups(PF_THREADS)) {
        return fail(TRC_HIP_E_SHAPE, "trc_hip_preference_loss: %lld rows", (long long) l.ne[1]);
    }
    auto* const f = l.type == TRC_HIP_TYPE_F32   ? forward<TRC_HIP_TYPE_F32>
                    : l.type == TRC_HIP_TYPE_F16 ? forward<TRC_HIP_TYPE_F16>
                                                 : forward<TRC_HIP_TYPE_BF16>;
    return f(l, labels, start, pairs, ref, beta, smooth, lse, logp, slope, loss, s);
}

int launch_preference_loss_back(const trc_hip_tensor& l, const int32_t* labels, const int32_t* start, int64_t pairs,
                                const float* lse, const float* slope, const float* dloss, float beta,
                                const trc_hip_tensor& d, hipStream_t s) {
    if (l.ne[1] > max_groups(PF_THREADS)) {
        return fail(TRC_HIP_E_SHAPE, "trc_hip_preference_loss_back: %lld rows", (long long) l.ne[1]);
    }
    auto* const f = l.type == TRC_HIP_TYPE_F32   ? backward<TRC_HIP_TYPE_F32>
                    : l.type == TRC_HIP_TYPE_F16 ? backward<TRC_HIP_TYPE_F16>
                                                 : backward<TRC_HIP_TYPE_BF16>;
    return f(l, labels, start, pairs, lse, slope, dloss, beta, d, s);
}

}  // namespace trc_hip
