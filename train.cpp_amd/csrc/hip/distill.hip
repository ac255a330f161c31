// The loss of a student's logits against a teacher's top logits (Hinton, Vinyals and Dean, "Distilling the knowledge in
// a neural network", 2015), mixed with the labels' cross-entropy, and the logits' gradient.
//
//   p = softmax(z / tau) over the teacher's entries      q = softmax(l / tau)      r = softmax(l)
//   KL_t = sum_j p_j (log p_j - log q_id_j)              CE_t = -log r_label
//   loss = mean_t  alpha tau^2 KL_t + (1 - alpha) CE_t
//   dl_tv = dloss / n (alpha tau (q_v - sum_{id_j = v} p_j) + (1 - alpha) (r_v - 1[v = label]))
//
// Two launches for the loss, the rows and one workgroup for what comes of them, and one for the gradient, which reads and writes
// each row once more. Bound by memory, and by the exponentials where both temperatures are summed. 8192 rows of 32000
// bfloat16, three in four of them counted: rows 92 us (4.3 TB/s), mean 9 (one CU fetches every row's terms; eight rows of a thread
// at once were no faster), gradient 167 (5.5 TB/s). 61 rows of 131071 floats in 31 parts: 8, 7 and 12. (A single launch for the
// loss, whose last workgroups to arrive finish a row and the loss, was slower: each of its steps waits for a trip to memory that
// all XCDs see.)
#include "logit_rows.h"

namespace trc_hip {

namespace {

constexpr int DI_THREADS = 256;
constexpr int DI_MAX_PARTS = 64;  // parts of a row: a lane each where they are joined
constexpr int DI_LOADS = 4;       // 16-byte loads that a thread has under way
constexpr int DI_JOIN = 1024;     // threads of the mean's workgroup
constexpr int DI_STATS = 5;
constexpr int64_t DI_MAX_ROWS = (int64_t) 1 << 19;  // their terms fit the stream's workspace
constexpr float LOG2E = 1.44269504088896340736f;

// What is summed of a row: exponentials at one temperature (of factor c = log2 e / temperature), at 1 and at tau, or both where tau
// is 2 and the one is the other's square.
constexpr int DI_ONE = 0, DI_BOTH = 1, DI_SQUARE = 2;

// A point m near the largest of what is summed (its maximum, or the largest of some of it) and the sums of exponentials from
// there, at temperature 1 (or the only one) and at tau.
struct Sums {
    float m, a, b;
};
// c of `a` and of `b`
struct Factors {
    float a, b;
};
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
// a maximum of -inf (nothing yet, or only -inf) is subtracted as 0, so that exp(-inf - m) is 0 and not NaN
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

// Both exponentials of d, a difference from a maximum.
template <int MODE>
__device__ __forceinline__ void both(float d, Factors c, float& a, float& b) {
    if (MODE == DI_SQUARE) {
        b = exp2_of(d * c.b);
        a = b * b;
    } else {
        a = exp2_of(d * c.a);
        b = MODE == DI_BOTH ? exp2_of(d * c.b) : 0.f;
    }
}
template <int MODE>
__device__ __forceinline__ Sums join(Sums x, Sums y, Factors c) {
    const float m = fmaxf(x.m, y.m), base = base_of(m);
    float xa, xb, ya, yb;
    both<MODE>(x.m - base, c, xa, xb);
    both<MODE>(y.m - base, c, ya, yb);
    return {m, x.a * xa + y.a * ya, x.b * xb + y.b * yb};
}
template <int MODE>
__device__ __forceinline__ Sums wave_join(Sums x, Factors c) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1)
        x = join<MODE>(x, {__shfl_xor(x.m, d, 64), __shfl_xor(x.a, d, 64), __shfl_xor(x.b, d, 64)}, c);
    return x;
}

// A thread's share of n elements at p, with a running maximum.
template <int TYPE, int MODE>
__device__ __forceinline__ Sums careful_share(const typename Row<TYPE>::Elem* p, int n, Factors c) {
    typedef Row<TYPE> R;
    constexpr int VEC = R::VEC, STEP = DI_THREADS * VEC;
    const int whole = n / VEC * VEC;
    Sums s = {-INFINITY, 0.f, 0.f};
    for (int i = (int) threadIdx.x * VEC; i < whole; i += STEP) {
        float x[VEC], m = s.m;
        R::load(p + i, x);
#pragma unroll
        for (int k = 0; k < VEC; ++k) m = fmaxf(m, x[k]);
        const float base = base_of(m);
        float a, b;
        both<MODE>(s.m - base, c, a, b);
        s = {m, s.a * a, s.b * b};
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            both<MODE>(x[k] - base, c, a, b);
            s.a += a;
            s.b += b;
        }
    }
    if (whole + (int) threadIdx.x < n) s = join<MODE>(s, {R::get(p[whole + threadIdx.x]), 1.f, 1.f}, c);
    return s;
}

// The same, with exponentials from the largest of the thread's first elements rather than from a running maximum: any
// point near enough gives as exact a sum, for a multiply-add, an exponential and an add an element.
// The careful way go sums over 2^64 (or not finite; joins of 2^14 such sums could overflow, and would drop one whose maximum
// lies far under another's) and a largest whose product with a factor is 2^23 or more, of which
// rounding would leave too much out.
template <int TYPE, int MODE>
__device__ __forceinline__ Sums share(const typename Row<TYPE>::Elem* p, int n, Factors c) {
    typedef Row<TYPE> R;
    constexpr int VEC = R::VEC, U = DI_LOADS, STEP = DI_THREADS * VEC;
    const int whole = n / VEC * VEC;
    int i = (int) threadIdx.x * VEC;
    if (i + (U - 1) * STEP >= whole) return careful_share<TYPE, MODE>(p, n, c);
    float x[U * VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) R::load(p + i + u * STEP, x + u * VEC);
    float m = x[0];
#pragma unroll
    for (int k = 1; k < U * VEC; ++k) m = fmaxf(m, x[k]);
    const float ua = m * c.a, ub = m * c.b;
    float sa = 0.f, sb = 0.f;
    auto add = [&] {
#pragma unroll
        for (int k = 0; k < U * VEC; ++k) {
            if (MODE == DI_SQUARE) {
                const float e = exp2_of(fmaf(x[k], c.b, -ub));
                sb += e;
                sa = fmaf(e, e, sa);
            } else {
                sa += exp2_of(fmaf(x[k], c.a, -ua));
                if (MODE == DI_BOTH) sb += exp2_of(fmaf(x[k], c.b, -ub));
            }
        }
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
    if (!(sa <= 0x1p64f) || !(sb <= 0x1p64f) || !(fabsf(ua) < 0x1p23f) || !(fabsf(ub) < 0x1p23f)) {
        return careful_share<TYPE, MODE>(p, n, c);
    }
    // what rounding the products of m left out, taken back
    const float fb = exp2_of(-fmaf(m, c.b, -ub));
    return {m, sa * (MODE == DI_SQUARE ? fb * fb : exp2_of(-fmaf(m, c.a, -ua))), MODE == DI_ONE ? 0.f : sb * fb};
}

// Where the teacher's entries of a row lie.
struct Teacher {
    const int32_t* ids;
    const uint8_t* z;
    int type, top;
    __device__ __forceinline__ float logit(int64_t at) const {
        if (type == TRC_HIP_TYPE_F32) return ((const float*) z)[at];
        const uint16_t b = ((const uint16_t*) z)[at];
        return type == TRC_HIP_TYPE_F16 ? half_bits_to_float(b) : __builtin_bit_cast(float, (uint32_t) b << 16);
    }
};

// One of a row's entries: the teacher's logit and the student's.
struct Entry {
    float z, l;
    bool in;
};

struct Term {
    double kl, ce;
};

// What a row's terms need of its entries and its label: with e_j = exp((z_j - zmax) / tau) and the student's logits taken from
// `ref`, the point m of what was summed beside them: sum e (0: no entries), sum e (z_j - zmax) / tau, sum e (l_j - ref), l_label - ref.
struct Entries {
    double e, ez, el, label;
    float ref, zmax;
    // sum_j p_j (log p_j - log q_j) and -log r_label for the sums of the whole row
    __device__ __forceinline__ Term term(const Sums& s, float tau, float alpha) const {
        const double off = (double) ref - (double) s.m;
        return {alpha > 0.f && e != 0.0 ? (ez - (el + e * off) / (double) tau) / e - log(e) + log((double) s.b) : 0.0,
                alpha < 1.f ? log((double) s.a) - (label + off) : 0.0};
    }
};

// What the gradient needs of a row.
__device__ __forceinline__ void put_stats(float* st, const Sums& s, const Entries& q) {
    st[0] = base_of(s.m);
    st[1] = 1.f / s.a;
    st[2] = 1.f / s.b;
    st[3] = q.zmax;
    st[4] = q.e == 0.0 ? 0.f : (float) (1.0 / q.e);
}

// Rows that are not counted are not read. gridDim.y parts of `len` elements each; the first one's first wave has the entries,
// on their way while the row is summed. One part makes the row's terms, several leave sums and what comes of the entries.
template <int TYPE, int MODE>
__global__ __launch_bounds__(DI_THREADS) void k_distill_rows(const uint8_t* __restrict__ logits, size_t nb1, int64_t V,
                                                              const int32_t* __restrict__ labels, Teacher teacher, Factors c,
                                                              float tau, float alpha, int64_t len, float* __restrict__ stats,
                                                              Term* __restrict__ terms, Sums* __restrict__ parts,
                                                              Entries* __restrict__ of_entries) {
    typedef Row<TYPE> R;
    const int64_t row = blockIdx.x;
    const int lane = (int) threadIdx.x & 63, wave = (int) threadIdx.x >> 6;
    const int32_t y = labels[row];
    if (y < 0) {
        if (blockIdx.y == 0 && threadIdx.x < DI_STATS) stats[row * DI_STATS + threadIdx.x] = 0.f;
        if (blockIdx.y == 0 && threadIdx.x == 0) terms[row] = {0.0, 0.0};
        return;
    }
    const typename R::Elem* const l = (const typename R::Elem*) (logits + row * nb1);
    const int64_t at = row * teacher.top;
    auto entry = [&](int j) {
        const int32_t id = j < teacher.top ? teacher.ids[at + j] : -1;
        const bool in = id >= 0 && id < V;
        return Entry{in ? teacher.logit(at + j) : -INFINITY, in ? R::get(l[id]) : 0.f, in};
    };
    const bool kl = alpha > 0.f, mine = wave == 0 && blockIdx.y == 0;
    Entry first = {-INFINITY, 0.f, false};
    float ly = 0.f;
    if (kl && mine) first = entry(lane);
    if (alpha < 1.f && mine) ly = y < V ? R::get(l[y]) : NAN;
    const int64_t lo = (int64_t) blockIdx.y * len;
    Sums s = wave_join<MODE>(share<TYPE, MODE>(l + lo, (int) (min(lo + len, V) - lo), c), c);
    __shared__ Sums w[DI_THREADS / 64];
    if (lane == 0) w[wave] = s;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int k = 0; k < DI_THREADS / 64; ++k) s = k == 0 ? w[0] : join<MODE>(s, w[k], c);
    if (gridDim.y > 1 && lane == 0) parts[row * gridDim.y + blockIdx.y] = s;
    if (!mine) return;
    if (MODE == DI_ONE) s.b = s.a;  // the only sum, whichever is wanted
    Entries q = {0.0, 0.0, 0.0, 0.0, base_of(s.m), 0.f};
    q.label = (double) ly - (double) q.ref;
    if (kl) {
        float m = first.z;
        bool some = first.in;
        for (int j = lane + 64; j < teacher.top; j += 64) {
            const Entry e = entry(j);
            m = fmaxf(m, e.z);
            some = some || e.in;
        }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
        q.zmax = base_of(m);
        auto take = [&](const Entry& n) {
            if (!n.in) return;
            const double x = (double) (n.z - q.zmax) / (double) tau, e = (double) exp2_of((float) (x * (double) LOG2E));
            if (e == 0.0) return;
            q.e += e;
            q.ez += e * x;
            q.el += e * ((double) n.l - (double) q.ref);
        };
        take(first);
        for (int j = lane + 64; j < teacher.top; j += 64) take(entry(j));
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            q.e += __shfl_xor(q.e, d, 64);
            q.ez += __shfl_xor(q.ez, d, 64);
            q.el += __shfl_xor(q.el, d, 64);
        }
        if (q.e == 0.0 && __any(some)) q.e = NAN;  // (a teacher to whom every entry is impossible)
    }
    if (lane != 0) return;
    if (gridDim.y > 1) {
        of_entries[row] = q;
    } else {
        put_stats(stats + row * DI_STATS, s, q);
        terms[row] = q.term(s, tau, alpha);
    }
}

// One workgroup: the sums of rows in parts, `each` threads (a power of two up to 64) a row, then the terms' means, each
// thread's rows and then the threads in a fixed order.
template <int MODE>
__global__ __launch_bounds__(DI_JOIN) void k_distill_mean(const int32_t* __restrict__ labels, int64_t T, Factors c, float tau, float alpha,
                                                           int n_parts, int each, const Sums* __restrict__ parts,
                                                           const Entries* __restrict__ of_entries,
                                                           const Term* __restrict__ terms, float* __restrict__ stats, float* __restrict__ loss) {
    double kl = 0.0, ce = 0.0;
    int n = 0;
    const int sub = (int) threadIdx.x & (each - 1);
    for (int64_t t0 = 0; t0 < T; t0 += DI_JOIN / each) {
        const int64_t t = t0 + threadIdx.x / each;
        const bool counted = t < T && labels[t] >= 0;
        Term q = {0.0, 0.0};
        if (n_parts > 1) {
            // (read whether or not the row is counted, so as not to wait for its label first)
            const int64_t row = min(t, T - 1);
            const Entries e = of_entries[row];
            const Sums* const p = parts + row * n_parts;
            Sums s = {-INFINITY, 0.f, 0.f};
            for (int i = sub; i < n_parts; i += 4 * each) {
                Sums x[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] = p[min(i + k * each, n_parts - 1)];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (i + k * each < n_parts) s = join<MODE>(s, x[k], c);
            }
            for (int d = 1; d < each; d <<= 1) s = join<MODE>(s, {__shfl_xor(s.m, d, 64), __shfl_xor(s.a, d, 64), __shfl_xor(s.b, d, 64)}, c);
            if (MODE == DI_ONE) s.b = s.a;
            if (counted && sub == 0) {
                put_stats(stats + t * DI_STATS, s, e);
                q = e.term(s, tau, alpha);
            }
        } else if (counted) {
            q = terms[t];
        }
        kl += q.kl;
        ce += q.ce;
        n += counted && sub == 0;
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        kl += __shfl_xor(kl, d, 64);
        ce += __shfl_xor(ce, d, 64);
        n += __shfl_xor(n, d, 64);
    }
    __shared__ double wk[DI_JOIN / 64], wc[DI_JOIN / 64];
    __shared__ int wn[DI_JOIN / 64];
    if ((threadIdx.x & 63) == 0) {
        wk[threadIdx.x >> 6] = kl;
        wc[threadIdx.x >> 6] = ce;
        wn[threadIdx.x >> 6] = n;
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < DI_JOIN / 64; ++w) {
        kl += wk[w];
        ce += wc[w];
        n += wn[w];
    }
    if (n > 0) {
        kl /= n;
        ce /= n;
    }
    // (a term of weight 0 was not computed, so that it is 0 and not infinite)
    loss[0] = (float) ((double) alpha * tau * tau * kl + (1.0 - (double) alpha) * ce);
    loss[1] = (float) kl;
    loss[2] = (float) ce;
    loss[3] = (float) n;
}

// Entries of one token add up, and one of them stores the sum: an open table in LDS, of twice the entries or more, gives each
// token an entry that owns it. (Which one does not show: its sum takes all of them in their order. Without the table each
// entry looked at all: 8192 rows of 32000 with 1024 entries 1078 us, 274 so, 61 of 131071 264 and 11, with 64 entries as before.)
constexpr int DI_OTHER = INT32_MIN;   // on an id: another entry owns the token
constexpr int DI_SHARED = 1 << 30;    // this one does, and there are others
constexpr int DI_TOKEN = DI_SHARED - 1;
__device__ __forceinline__ int owner_of(int* table, int bits, const int32_t* ids, int32_t id, int j) {
    uint32_t slot = (uint32_t) id * 2654435761u >> (32 - bits);
    for (;;) {
        const int old = j < 0 ? table[slot] : atomicCAS(&table[slot], -1, j);
        if (old == -1) return j;
        if ((__hip_atomic_load(&ids[old], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) & DI_TOKEN) == id) return old;
        slot = (slot + 1) & ((1u << bits) - 1);
    }
}

// A row's entries (and its label) are taken out of the row before the gradient may overwrite it, and put over what the
// whole row's pass has stored there.
template <int TYPE, int MODE>
__global__ __launch_bounds__(DI_THREADS) void k_distill_back(const uint8_t* logits, size_t nb1, int64_t V,
                                                              const int32_t* __restrict__ labels, Teacher teacher, Factors c, float tau,
                                                              float alpha, const float* __restrict__ stats, const float* __restrict__ loss,
                                                              const float* __restrict__ dloss, int64_t len, int bits, uint8_t* dlogits, size_t dnb1) {
    typedef Row<TYPE> R;
    constexpr int VEC = R::VEC, U = DI_LOADS, STEP = DI_THREADS * VEC;
    extern __shared__ float entries[];  // ids, probabilities and the student's logits, top + 1 of each, and the table
    const int64_t row = gridDim.x - 1 - blockIdx.x;  // the last rows first: the caches may hold them yet
    const int32_t y = labels[row];
    const int64_t lo = (int64_t) blockIdx.y * len;
    const typename R::Elem* const p = (const typename R::Elem*) (logits + row * nb1) + lo;
    typename R::Elem* const d = (typename R::Elem*) (dlogits + row * dnb1) + lo;
    const int n = (int) (min(lo + len, V) - lo), whole = n / VEC * VEC;
    int i = (int) threadIdx.x * VEC;
    if (y < 0) {  // not counted: zeros, whatever the logits hold
        float z[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) z[k] = 0.f;
        for (; i < whole; i += STEP) R::store(d + i, z);
        if (whole + (int) threadIdx.x < n) d[whole + threadIdx.x] = R::put(0.f);
        return;
    }
    const float* const st = stats + row * DI_STATS;
    const float m = st[0], unit = dloss[0] / loss[3];
    const float wk = alpha > 0.f && st[4] != 0.f ? unit * alpha * tau : 0.f;
    const float wc = alpha < 1.f ? (y < V ? unit * (1.f - alpha) : NAN) : 0.f;  // (a label past the vocabulary: NaN, as the loss is)
    // factors on the exponentials of `both`
    const float qb = wk * st[2], qa = wc != 0.f ? wc * st[1] : 0.f;
    const int top = wk != 0.f ? teacher.top : 0;
    int32_t* const ids = (int32_t*) entries;
    float *const prob = entries + (teacher.top + 1), *const at_id = prob + (teacher.top + 1);
    int* const table = (int*) (at_id + (teacher.top + 1));
    for (int j = (int) threadIdx.x; j <= top; j += DI_THREADS) {
        const int64_t e = row * teacher.top + j;
        const int32_t id = j < top ? teacher.ids[e] : wc != 0.f ? y : -1;
        const bool in = id >= lo && id < lo + n;
        ids[j] = in ? id : -1;
        prob[j] = in && j < top ? exp2_of((teacher.logit(e) - st[3]) * (LOG2E / tau)) * st[4] : 0.f;
        at_id[j] = in ? R::get(p[id - lo]) : 0.f;
    }
    for (int k = (int) threadIdx.x; k < 1 << bits; k += DI_THREADS) table[k] = -1;
    __syncthreads();
    for (int j = (int) threadIdx.x; j < top; j += DI_THREADS) {
        const int32_t id = ids[j] & DI_TOKEN;
        if (ids[j] == -1) continue;
        const int owner = owner_of(table, bits, ids, id, j);
        if (owner == j) continue;
        atomicOr(&ids[owner], DI_SHARED);
        ids[j] = id | DI_OTHER;
    }
    __syncthreads();
    // the label's own entry is only for a token that has no other
    if (threadIdx.x == 0 && ids[top] >= 0 && owner_of(table, bits, ids, ids[top], -1) >= 0) ids[top] = -1;
    auto gradient = [&](float x) {
        float a, b;
        both<MODE>(x - m, c, a, b);
        return MODE == DI_ONE ? (qa + qb) * a : fmaf(qa, a, qb * b);
    };
    for (; i + (U - 1) * STEP < whole; i += U * STEP) {
        float x[U][VEC];
#pragma unroll
        for (int u = 0; u < U; ++u) R::load(p + i + u * STEP, x[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) x[u][k] = gradient(x[u][k]);
            R::store(d + i + u * STEP, x[u]);
        }
    }
    for (; i < whole; i += STEP) {
        float x[VEC];
        R::load(p + i, x);
#pragma unroll
        for (int k = 0; k < VEC; ++k) x[k] = gradient(x[k]);
        R::store(d + i, x);
    }
    if (whole + (int) threadIdx.x < n) d[whole + threadIdx.x] = R::put(gradient(R::get(p[whole + threadIdx.x])));
    // every store of the pass is done before any of these, which may be to the same places
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int j = (int) threadIdx.x; j <= top; j += DI_THREADS) {
        if (ids[j] < 0) continue;
        const int32_t id = ids[j] & DI_TOKEN;
        float sum = prob[j];
        if (ids[j] & DI_SHARED) {
            sum = 0.f;
            for (int k = 0; k < top; ++k) sum += (ids[k] & DI_TOKEN) == id ? prob[k] : 0.f;
        }
        float g = gradient(at_id[j]) - wk * sum;
        if (id == y) g -= wc;
        d[id - lo] = R::put(g);
    }
}

// Parts of a row, and their length: whole rows while there are rows for every CU several times over, else parts of
// 4096 elements or more.
int64_t part_length(int64_t V, int64_t T) {
    const int64_t wanted = ((int64_t) device_cus() * 8 + T - 1) / T;
    const int64_t most = V / 4096;
    int64_t parts = wanted < most ? wanted : most;
    if (parts > DI_MAX_PARTS) parts = DI_MAX_PARTS;
    if (parts < 2) return V;
    return ((V + parts - 1) / parts + 7) / 8 * 8;
}

struct Call {
    const trc_hip_tensor* l;
    const int32_t* labels;
    Teacher teacher;
    float tau, alpha;
    Factors c;
};

template <int TYPE, int MODE>
int forward(const Call& q, float* stats, float* loss, hipStream_t s) {
    const int64_t V = q.l->ne[0], T = q.l->ne[1], len = part_length(V, T), n = (V + len - 1) / len;
    uint8_t* ws = nullptr;
    int rc = qm_stream_workspace(s, &ws);
    if (rc != TRC_HIP_OK) return rc;
    Term* const terms = (Term*) ws;
    Entries* const of_entries = (Entries*) (terms + T);
    Sums* const parts = (Sums*) (of_entries + (n > 1 ? T : 0));
    if ((size_t) T * sizeof(Term) + (n > 1 ? (size_t) T * sizeof(Entries) + (size_t) (n * T) * sizeof(Sums) : 0) > qm_workspace_bytes()) {
        return fail(TRC_HIP_E_SHAPE, "trc_hip_distill_loss: %lld rows in %lld parts", (long long) T, (long long) n);
    }
    hipLaunchKernelGGL((k_distill_rows<TYPE, MODE>), dim3((unsigned) T, (unsigned) n), dim3(DI_THREADS), 0, s, (const uint8_t*) q.l->data,
                       q.l->nb[1], V, q.labels, q.teacher, q.c, q.tau, q.alpha, len, stats, terms, parts, of_entries);
    rc = check_launch("distill_loss (rows)");
    if (rc != TRC_HIP_OK) return rc;
    const int each = n == 1 || T > 256 ? 1 : T > 64 ? 4 : 16;  // (few rows have many parts)
    hipLaunchKernelGGL(k_distill_mean<MODE>, dim3(1), dim3(DI_JOIN), 0, s, q.labels, T, q.c, q.tau, q.alpha, (int) n, each,
                       parts, of_entries, terms, stats, loss);
    return check_launch("distill_loss (mean)");
}

template <int TYPE, int MODE>
int backward(const Call& q, const float* stats, const float* loss, const float* dloss, const trc_hip_tensor& d, hipStream_t s) {
    const int64_t V = q.l->ne[0], T = q.l->ne[1], len = part_length(V, T), n = (V + len - 1) / len;
    int bits = 1;
    while ((1 << bits) < 2 * q.teacher.top) ++bits;
    hipLaunchKernelGGL((k_distill_back<TYPE, MODE>), dim3((unsigned) T, (unsigned) n), dim3(DI_THREADS),
                       (q.teacher.top + 1) * 12 + (4 << bits), s,
                       (const uint8_t*) q.l->data, q.l->nb[1], V, q.labels, q.teacher, q.c, q.tau, q.alpha, stats, loss, dloss, len, bits,
                       (uint8_t*) d.data, d.nb[1]);
    return check_launch("distill_loss_back");
}

// What of a row is summed: tau counts where the KL does, 1 where the cross-entropy does.
int mode_of(float tau, float alpha, Factors& c) {
    c = {LOG2E, LOG2E / tau};
    if (alpha == 1.f) c.a = c.b;
    if (alpha == 0.f || alpha == 1.f || tau == 1.f) return DI_ONE;
    return tau == 2.f ? DI_SQUARE : DI_BOTH;
}

// f<TYPE, MODE> for a call's type and mode
#define DI_PICK(f, type, mode)                                                                                       \
    (type == TRC_HIP_TYPE_F32   ? (mode == DI_ONE ? f<TRC_HIP_TYPE_F32, DI_ONE> : mode == DI_BOTH ? f<TRC_HIP_TYPE_F32, DI_BOTH> : f<TRC_HIP_TYPE_F32, DI_SQUARE>) \
     : type == TRC_HIP_TYPE_F16 ? (mode == DI_ONE ? f<TRC_HIP_TYPE_F16, DI_ONE> : mode == DI_BOTH ? f<TRC_HIP_TYPE_F16, DI_BOTH> : f<TRC_HIP_TYPE_F16, DI_SQUARE>) \
                                : (mode == DI_ONE ? f<TRC_HIP_TYPE_BF16, DI_ONE> : mode == DI_BOTH ? f<TRC_HIP_TYPE_BF16, DI_BOTH> : f<TRC_HIP_TYPE_BF16, DI_SQUARE>))

Call call_of(const trc_hip_tensor& l, const int32_t* labels, const trc_hip_tensor& ids, const trc_hip_tensor& teacher, float tau,
             float alpha) {
    return {&l, labels, {(const int32_t*) ids.data, (const uint8_t*) teacher.data, teacher.type, (int) ids.ne[0]}, tau, alpha, {}};
}

}  // namespace

int launch_distill_loss(const trc_hip_tensor& l, const int32_t* labels, const trc_hip_tensor& ids, const trc_hip_tensor& teacher, float tau,
                        float alpha, float* stats, float* loss, hipStream_t s) {
    if (l.ne[1] > DI_MAX_ROWS) {
        return fail(TRC_HIP_E_SHAPE, "trc_hip_distill_loss: %lld rows (at most %lld)", (long long) l.ne[1], (long long) DI_MAX_ROWS);
    }
    Call q = call_of(l, labels, ids, teacher, tau, alpha);
    const int mode = mode_of(tau, alpha, q.c);
    return DI_PICK(forward, l.type, mode)(q, stats, loss, s);
}

int launch_distill_loss_back(const trc_hip_tensor& l, const int32_t* labels, const trc_hip_tensor& ids, const trc_hip_tensor& teacher,
                             const float* stats, const float* loss, const float* dloss, float tau, float alpha, const trc_hip_tensor& d,
                             hipStream_t s) {
    if (l.ne[1] > DI_MAX_ROWS) {
        return fail(TRC_HIP_E_SHAPE, "trc_hip_distill_loss_back: %lld rows (at most %lld)", (long long) l.ne[1], (long long) DI_MAX_ROWS);
    }
    Call q = call_of(l, labels, ids, teacher, tau, alpha);
    const int mode = mode_of(tau, alpha, q.c);
    return DI_PICK(backward, l.type, mode)(q, stats, loss, dloss, d, s);
}

}  // namespace trc_hip
