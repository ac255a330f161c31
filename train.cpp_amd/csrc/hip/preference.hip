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
constexpr int PF_WAVES = 16;       // of the join
constexpr int PF_MAX_PARTS = 64;   // parts of a row: a lane each where they are joined
constexpr int PF_LOADS = 4;        // 16-byte loads that a thread has under way
constexpr int64_t PF_MAX_ROWS = (int64_t) 1 << 20;  // their log-probabilities fit the stream's workspace
constexpr float PF_FAR = 1024.f;   // magnitude of a row's log-sum from which its float is not taken for the gradient
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

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }

// A maximum and the sum of exponentials taken from it (the difference first: its product with LOG2E cannot
// overflow where logits are the type's lowest value). A maximum of -inf (nothing yet, or only -inf)
// is subtracted as 0, so that exp(-inf - m) is 0 and not NaN; infinities and NaNs reach the sum.
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
// A row's log-sum, and the log-probability of its label's logit ly, in 64 bits: the sums over a sequence's rows, and
// differences of them, would show its rounding. The maximum goes first, or of rows far from 0 nothing would be left.
struct RowSums {
    float lse;
    double lp;
    __device__ __forceinline__ RowSums(Soft a, double ly) {
        const double log_s = log((double) a.s);
        lse = (float) ((double) a.m + log_s);
        lp = (ly - (double) a.m) - log_s;
    }
};

template <int N>
__device__ __forceinline__ void take(Soft& a, const float (&x)[N]) {
    float m = a.m;
#pragma unroll
    for (int k = 0; k < N; ++k) m = fmaxf(m, x[k]);
    const float base = base_of(m);
    float s = a.s * exp_of(a.m - base);
#pragma unroll
    for (int k = 0; k < N; ++k) s += exp_of(x[k] - base);
    a = {m, s};
}

// A thread's share of n elements at p, with the running maximum: 4 KB of a wave's loads under way together.
template <int TYPE>
__device__ __forceinline__ Soft careful_share(const typename Row<TYPE>::Elem* p, int n) {
    typedef Row<TYPE> R;
    constexpr int VEC = R::VEC, STEP = PF_THREADS * VEC;
    const int whole = n / VEC * VEC;
    Soft a = {-INFINITY, 0.f};
    for (int i = (int) threadIdx.x * VEC; i < whole; i += STEP) {
        float x[VEC];
        R::load(p + i, x);
        take(a, x);
    }
    if (whole + (int) threadIdx.x < n) a = join(a, {R::get(p[whole + threadIdx.x]), 1.f});
    return a;
}

// The same, with the exponentials taken from the largest of the thread's first elements rather than from a
// running maximum: their sum is as exact from any point near enough, and an element costs a
// multiply-add, an exponential and an add.
// The careful way go a sum over 2^64 (or not finite) and a largest of 2^23 / LOG2E or more in magnitude (or not finite):
// - Joins add up to 2^14 sums (256 threads, 64 parts) and drop one whose maximum lies 126 bits under another's: 2^78 is
//   finite, and 2^64 2^-126 nothing beside a sum that holds its maximum. A sum up to the largest float would be neither.
// - What rounding leaves out of m LOG2E is up to half a unit of its last place, past 2^30 so much that exp2 of it
//   is 0 or an infinity where all that a thread reads is one far mask. Under 2^23 it is 1/4 at most.
template <int TYPE>
__device__ __forceinline__ Soft share(const typename Row<TYPE>::Elem* p, int n) {
    typedef Row<TYPE> R;
    constexpr int VEC = R::VEC, U = PF_LOADS, STEP = PF_THREADS * VEC;
    const int whole = n / VEC * VEC;
    int i = (int) threadIdx.x * VEC;
    if (i + (U - 1) * STEP >= whole) return careful_share<TYPE>(p, n);
    float x[U * VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) R::load(p + i + u * STEP, x + u * VEC);
    float m = x[0];
#pragma unroll
    for (int k = 1; k < U * VEC; ++k) m = fmaxf(m, x[k]);
    const float unit = m * LOG2E;
    float s = 0.f;
    auto add = [&] {
#pragma unroll
        for (int k = 0; k < U * VEC; ++k) s += __builtin_amdgcn_exp2f(fmaf(x[k], LOG2E, -unit));
    };
    add();
    for (i += U * STEP; i + (U - 1) * STEP < whole; i += U * STEP) {
#pragma unroll
        for (int u = 0; u < U; ++u) R::load(p + i + u * STEP, x + u * VEC);
        add();
    }
#pragma unroll
    for (int k = 0; k < U * VEC; ++k) x[k] = -INFINITY;
#pragma unroll
    for (int u = 0; u < U - 1; ++u)
        if (i + u * STEP < whole) R::load(p + i + u * STEP, x + u * VEC);
    if (whole + (int) threadIdx.x < n) x[U * VEC - 1] = R::get(p[whole + threadIdx.x]);
    add();
    if (!(s <= 0x1p64f) || !(fabsf(unit) < 0x1p23f)) return careful_share<TYPE>(p, n);
    // what rounding m LOG2E left out, taken back
    return {m, s * exp_of(fmaf(m, LOG2E, -unit) * -(1.f / LOG2E))};
}

// Rows whose label is negative are not counted: they are not read, and their lse and log-probability are 0.
// gridDim.y parts of `len` elements each; one part writes lse and the label's log-probability lp, more
// write (m, s) to parts, and lp is the label's logit until they are joined.
template <int TYPE>
__global__ __launch_bounds__(PF_THREADS) void k_pref_rows(const uint8_t* __restrict__ logits, size_t nb1, int64_t V,
                                                           const int32_t* __restrict__ labels, int64_t len,
                                                           float* __restrict__ lse, double* __restrict__ lp,
                                                           Soft* __restrict__ parts) {
    typedef Row<TYPE> R;
    const int64_t row = blockIdx.x;
    const int32_t y = labels[row];
    if (y < 0) {
        if (blockIdx.y == 0 && threadIdx.x == 0) {
            lse[row] = 0.f;
            lp[row] = 0.0;
        }
        return;
    }
    const typename R::Elem* const all = (const typename R::Elem*) (logits + row * nb1);
    const int64_t lo = (int64_t) blockIdx.y * len;
    const float ly = y < V ? R::get(all[y]) : NAN;
    Soft a = share<TYPE>(all + lo, (int) (min(lo + len, V) - lo));
    __shared__ Soft w[PF_THREADS / 64];
    a = wave_join(a);
    if (((int) threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = a;
    __syncthreads();
    if (threadIdx.x != 0) return;
#pragma unroll
    for (int k = 1; k < PF_THREADS / 64; ++k) a = join(a, w[k]);
    if (gridDim.y == 1) {
        const RowSums r(a, ly);
        lse[row] = r.lse;
        lp[row] = r.lp;
    } else {
        parts[row * gridDim.y + blockIdx.y] = a;
        if (blockIdx.y == 0) lp[row] = ly;
    }
}

// One workgroup: the rows' parts joined where there are any, a wave a row, then a wave for each sequence.
// The tokens' log-probabilities and the pairs' terms are summed in 64 bits, each sum in one
// order: a sequence's sum is far larger than the ratios that come of it.
__global__ __launch_bounds__(PF_WAVES * 64) void k_pref_pairs(int64_t T, const int32_t* __restrict__ labels,
                                                               const int32_t* __restrict__ start, int64_t pairs,
                                                               const float* __restrict__ ref, float beta, float smooth,
                                                               int n_parts, const Soft* __restrict__ parts, float* lse,
                                                               double* lp, float* __restrict__ logp,
                                                               float* __restrict__ slope, float* __restrict__ loss) {
    const int lane = (int) threadIdx.x & 63, wave = (int) threadIdx.x >> 6;
    if (n_parts > 1) {
        for (int64_t t0 = wave; t0 < T; t0 += 4 * PF_WAVES) {
            Soft a[4], mine = {0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 4; ++k)  // (of rows not counted: whatever is there)
                a[k] = parts[min(t0 + k * PF_WAVES, T - 1) * n_parts + min(lane, n_parts - 1)];
            const int64_t t = t0 + lane * PF_WAVES;  // a row to each of four lanes
            const bool own = lane < 4 && t < T && labels[t] >= 0;
            const double l = own ? lp[t] : 0.0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const Soft all = wave_join(lane < n_parts ? a[k] : Soft{-INFINITY, 0.f});
                if (lane == k) mine = all;
            }
            if (own) {
                const RowSums r(mine, l);
                lse[t] = r.lse;
                lp[t] = r.lp;
            }
        }
        __syncthreads();
    }
    __shared__ double L[PF_WAVES], terms[PF_WAVES / 2];
    double mine = 0.0;
    for (int64_t s0 = 0; s0 < 2 * pairs; s0 += PF_WAVES) {
        if (s0 + wave < 2 * pairs) {
            const int64_t lo = min(max((int64_t) start[s0 + wave], (int64_t) 0), T);
            const int64_t hi = min(max((int64_t) start[s0 + wave + 1], lo), T);
            double sum = 0.0;
            for (int64_t t = lo + lane; t < hi; t += 8 * 64) {
                double x[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] = t + 64 * k < hi ? lp[t + 64 * k] : 0.0;
#pragma unroll
                for (int k = 0; k < 8; ++k) sum += x[k];
            }
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d, 64);
            if (lane == 0) {
                L[wave] = sum;
                logp[s0 + wave] = (float) sum;
            }
        }
        __syncthreads();
        const int64_t i = s0 / 2 + threadIdx.x;
        if (threadIdx.x < PF_WAVES / 2 && i < pairs) {
            const double chosen = L[2 * threadIdx.x] - (double) ref[2 * i];
            const double rejected = L[2 * threadIdx.x + 1] - (double) ref[2 * i + 1];
            const double z = (double) beta * (chosen - rejected);
            const double e = (double) smooth, small = exp(-fabs(z)), tail = log1p(small);
            const double up = fmax(-z, 0.0) + tail, down = fmax(z, 0.0) + tail;  // -log sigma(z), -log sigma(-z)
            // (a weight of 0 takes no part of an infinite term)
            mine += z != z ? z : (e == 1.0 ? 0.0 : (1.0 - e) * up) + (e == 0.0 ? 0.0 : e * down);
            const double near = 1.0 / (1.0 + small), far = small / (1.0 + small);  // sigma(|z|), sigma(-|z|)
            slope[i] = (float) (z != z ? z : z >= 0.0 ? e * near - (1.0 - e) * far : e * far - (1.0 - e) * near);
        }
        __syncthreads();
    }
    if (threadIdx.x < PF_WAVES / 2) terms[threadIdx.x] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        double sum = 0.0;
        for (int k = 0; k < PF_WAVES / 2; ++k) sum += terms[k];
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
    constexpr int VEC = R::VEC, U = PF_LOADS, STEP = PF_THREADS * VEC;
    // The last rows first: they are what the caches still hold of the forward pass. With stores that do not stay
    // there either, 8192 rows of 32000 in 16 bits take 227 us both ways, and 275 in order with plain stores.
    const int64_t row = gridDim.x - 1 - blockIdx.x;
    const int32_t y = labels[row];
    const int64_t seq = y < 0 ? -1 : sequence_of(start, 2 * pairs, row);
    float base = lse[row], part = 1.f;  // a probability is exp(l - base) part
    // A float is off by 2^-15 (3e-5 of every probability) at most under PF_FAR. Beyond, the row is summed again from its
    // maximum: of logits around -1e9 the float holds nothing of log s. The row's first workgroup does it, and
    // the whole row with it, since dlogits may be the logits and another would overwrite what it reads. 61 rows of 131071
    // in F32 take 78 us both ways if all are so, 26 otherwise; 8192 of 32000 in 16 bits 265, 224 otherwise.
    const bool far = seq >= 0 && fabsf(base) >= PF_FAR && fabsf(base) < INFINITY;
    if (far && blockIdx.y != 0) return;
    const int64_t lo = (int64_t) blockIdx.y * len;
    const typename R::Elem* const p = (const typename R::Elem*) (logits + row * nb1) + lo;
    typename R::Elem* const d = (typename R::Elem*) (dlogits + row * dnb1) + lo;
    const int n = (int) (far ? V : min(lo + len, V) - lo), whole = n / VEC * VEC;
    int i = (int) threadIdx.x * VEC;
    if (far) {
        __shared__ Soft sums[PF_THREADS / 64];
        Soft a = wave_join(careful_share<TYPE>(p, n));
        if (((int) threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = a;
        __syncthreads();
        a = sums[0];
#pragma unroll
        for (int k = 1; k < PF_THREADS / 64; ++k) a = join(a, sums[k]);
        base = a.m;
        part = 1.f / a.s;
    }
    if (seq < 0) {  // not counted: zeros, whatever the logits hold
        float z[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) z[k] = 0.f;
        for (; i < whole; i += STEP) R::store(d + i, z);
        if (whole + (int) threadIdx.x < n) d[whole + threadIdx.x] = R::put(0.f);
        return;
    }
    const float w = (float) ((double) slope[seq >> 1] * (double) beta / (double) pairs) * dloss[0] * ((seq & 1) ? -1.f : 1.f);
    const float wp = w * part;
    const int64_t label = y - lo;  // in this part
    // -w exp(l - lse), and w more at the label
    auto store = [&](int at, float* x) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) x[k] = exp_of(x[k] - base);
        if (label >= at && label < at + VEC) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) x[k] = (label == at + k ? 1.f : 0.f) - x[k] * part;
#pragma unroll
            for (int k = 0; k < VEC; ++k) x[k] *= w;
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k) x[k] *= -wp;
        }
        R::store(d + at, x);
    };
    for (; i + (U - 1) * STEP < whole; i += U * STEP) {
        float x[U][VEC];
#pragma unroll
        for (int u = 0; u < U; ++u) R::load(p + i + u * STEP, x[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) store(i + u * STEP, x[u]);
    }
    float x[U][VEC];
#pragma unroll
    for (int u = 0; u < U - 1; ++u)
        if (i + u * STEP < whole) R::load(p + i + u * STEP, x[u]);
    const int last = whole + (int) threadIdx.x;
    if (last < n) x[U - 1][0] = R::get(p[last]);
#pragma unroll
    for (int u = 0; u < U - 1; ++u)
        if (i + u * STEP < whole) store(i + u * STEP, x[u]);
    if (last < n) d[last] = R::put(w * ((label == last ? 1.f : 0.f) - exp_of(x[U - 1][0] - base) * part));
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
    const int64_t len = part_length(V, T), n = (V + len - 1) / len;  // (n T is about 8 CUs: little of the workspace)
    uint8_t* ws = nullptr;
    int rc = qm_stream_workspace(s, &ws);
    if (rc != TRC_HIP_OK) return rc;
    double* const lp = (double*) ws;
    Soft* const parts = (Soft*) (ws + (size_t) T * 8);
    if ((size_t) T * 8 + (n > 1 ? (size_t) (n * T) * sizeof(Soft) : 0) > qm_workspace_bytes()) {
        return fail(TRC_HIP_E_SHAPE, "trc_hip_preference_loss: %lld rows in %lld parts", (long long) T, (long long) n);
    }
    hipLaunchKernelGGL(k_pref_rows<TYPE>, dim3((unsigned) T, (unsigned) n), dim3(PF_THREADS), 0, s, (const uint8_t*) l.data,
                       l.nb[1], V, labels, len, lse, lp, parts);
    rc = check_launch("preference_loss (rows)");
    if (rc != TRC_HIP_OK) return rc;
    hipLaunchKernelGGL(k_pref_pairs, dim3(1), dim3(PF_WAVES * 64), 0, s, T, labels, start, pairs, ref, beta, smooth, (int) n,
                       parts, lse, lp, logp, slope, loss);
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
    if (l.ne[1] > PF_MAX_ROWS) {
        return fail(TRC_HIP_E_SHAPE, "trc_hip_preference_loss: %lld rows (at most %lld)", (long long) l.ne[1],
                    (long long) PF_MAX_ROWS);
    }
    auto* const f = l.type == TRC_HIP_TYPE_F32   ? forward<TRC_HIP_TYPE_F32>
                    : l.type == TRC_HIP_TYPE_F16 ? forward<TRC_HIP_TYPE_F16>
                                                 : forward<TRC_HIP_TYPE_BF16>;
    return f(l, labels, start, pairs, ref, beta, smooth, lse, logp, slope, loss, s);
}

int launch_preference_loss_back(const trc_hip_tensor& l, const int32_t* labels, const int32_t* start, int64_t pairs,
                                const float* lse, const float* slope, const float* dloss, float beta,
                                const trc_hip_tensor& d, hipStream_t s) {
    if (l.ne[1] > PF_MAX_ROWS) {
        return fail(TRC_HIP_E_SHAPE, "trc_hip_preference_loss_back: %lld rows (at most %lld)", (long long) l.ne[1],
                    (long long) PF_MAX_ROWS);
    }
    auto* const f = l.type == TRC_HIP_TYPE_F32   ? backward<TRC_HIP_TYPE_F32>
                    : l.type == TRC_HIP_TYPE_F16 ? backward<TRC_HIP_TYPE_F16>
                                                 : backward<TRC_HIP_TYPE_BF16>;
    return f(l, labels, start, pairs, lse, slope, dloss, beta, d, s);
}

}  // namespace trc_hip
