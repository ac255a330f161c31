// AdamW over many tensors in one launch, its moments as floats or in 8 bits.
//
//   m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd decay) - (lr / (1 - b1^t)) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// (Loshchilov and Hutter, "Decoupled Weight Decay Regularization", 2019; the
// reference's optimizer step, src/optim/trc_optim.cpp, which its trajectories under
// tests/golden/reference_suite pin.) Every operation is rounded on its own, in
// this order (the file is built without contraction), so the 8-bit codes below are the
// same whoever computes them.
//
// 8 bits: a block of 256 elements shares two float scales, its largest |m| and its
// largest u = sqrt(v). The codes are square roots of the ratios to them,
//   m = sm sign(c) (c / 127)^2, c in -127..127      u = su (c / 255)^2, c in 0..255
// which gives small values finer steps, as block-wise non-linear codes do (Dettmers et al.,
// "8-bit Optimizers via Block-wise Quantization", 2021). A value is off by half a step of its code
// at most, (c + 1/4) / 127^2 of the block's largest |m| and (c + 1/4) / 255^2 of its largest u: of
// values near the largest 1/127 and 1/255, of values near 1/254 of it up to 14 and 7 %. Values under the
// first step (1/127^2 and 1/255^2 of the largest) have no relative bound: an m under a quarter of it is held as 0, a
// u above 0 as the first step at least. u is held rather than v because it is what divides,
// and has twice the range: c is never 0 where u > 0, so a small v never turns into 0 / eps. A block whose largest value is below the smallest
// normal float is held as zeros; a block that meets a value that is not finite is not
// finite from then on.
#include <cmath>
#include <vector>

#include "common.h"

namespace trc_hip {

namespace {

constexpr int AW_BLOCK = TRC_HIP_ADAMW_BLOCK;  // a wave: 64 lanes of four elements
constexpr int AW_THREADS = 256;
constexpr int AW_CHUNK = 2048;  // elements of one workgroup
static_assert(AW_BLOCK == 64 * 4 && AW_CHUNK % (AW_THREADS * 4) == 0, "a wave per block");

// vectors whose address is only as aligned as one element
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t h4u __attribute__((ext_vector_type(4), aligned(2)));
typedef uint8_t b4u __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u32u __attribute__((aligned(1)));

struct AwTensor {
    float* p;
    const void* g;
    void *m, *v;
    float *ms, *vs;  // the blocks' scales (8 bits)
    float *mf, *vf;  // where the moments are read out to
    int64_t n;
    int64_t first;   // its first chunk
    float decay;
    int32_t gtype;
};

struct AwHyper {
    double decay;  // lr wd
    float b1, c1, b2, c2, eps, rate, root, gscale;
};

struct Plan {
    int dev;
    int bits;
    bool readable;   // every tensor has mf and vf
    int64_t chunks;
    AwTensor* tensors;  // device
    uint32_t* owner;    // device: the tensor of each chunk
};

// A step reads and writes everything once, past the caches (but for k_adamw's gradients, which are read by plain loads):
// the 243 million elements of a 4096-wide layer take 1200 us, and 1270 with plain accesses throughout.
__device__ __forceinline__ f4u once(const f4u* p) { return __builtin_nontemporal_load(p); }
__device__ __forceinline__ h4u once(const h4u* p) { return __builtin_nontemporal_load(p); }
__device__ __forceinline__ uint32_t once(const u32u* p) { return __builtin_nontemporal_load(p); }
__device__ __forceinline__ void store_once(f4u* p, f4 x) { __builtin_nontemporal_store(x, p); }
__device__ __forceinline__ void store_once(u32u* p, uint32_t x) { __builtin_nontemporal_store(x, p); }

__device__ __forceinline__ f4 load_grad(const void* g, int type, int64_t i) {
    if (type == TRC_HIP_TYPE_F32) return *(const f4u*) ((const float*) g + i);
    const h4u h = *(const h4u*) ((const uint16_t*) g + i);
    f4 r;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        r[k] = type == TRC_HIP_TYPE_F16 ? half_bits_to_float(h[k]) : __builtin_bit_cast(float, (uint32_t) h[k] << 16);
    }
    return r;
}
__device__ __forceinline__ float load_grad1(const void* g, int type, int64_t i) {
    if (type == TRC_HIP_TYPE_F32) return ((const float*) g)[i];
    const uint16_t h = ((const uint16_t*) g)[i];
    return type == TRC_HIP_TYPE_F16 ? half_bits_to_float(h) : __builtin_bit_cast(float, (uint32_t) h << 16);
}

// One element's step; u = sqrt(v) of the new v comes back too.
__device__ __forceinline__ void update(const AwHyper& h, float decay, float& p, float g, float& m, float& v, float& u) {
    g = g * h.gscale;
    m = m * h.b1 + g * h.c1;
    v = v * h.b2 + (g * g) * h.c2;
    u = sqrtf(v);
    p = p * decay;
    p = p - (m / (u * h.root + h.eps)) * h.rate;
}

__global__ __launch_bounds__(AW_THREADS) void k_adamw(const AwTensor* __restrict__ tensors,
                                                       const uint32_t* __restrict__ owner, AwHyper h) {
    const AwTensor t = tensors[owner[blockIdx.x]];
    const float decay = (float) (1.0 - h.decay * (double) t.decay);
    const int64_t base = ((int64_t) blockIdx.x - t.first) * AW_CHUNK;
    float* const pm = (float*) t.m;
    float* const pv = (float*) t.v;
#pragma unroll
    for (int it = 0; it < AW_CHUNK / (AW_THREADS * 4); ++it) {
        const int64_t i = base + (it * AW_THREADS + (int) threadIdx.x) * 4;
        if (i + 4 <= t.n) {
            f4 p = once((const f4u*) (t.p + i)), m = once((const f4u*) (pm + i)), v = once((const f4u*) (pv + i));
            const f4 g = load_grad(t.g, t.gtype, i);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float pk = p[k], mk = m[k], vk = v[k], u;
                update(h, decay, pk, g[k], mk, vk, u);
                p[k] = pk;
                m[k] = mk;
                v[k] = vk;
            }
            store_once((f4u*) (t.p + i), p);
            store_once((f4u*) (pm + i), m);
            store_once((f4u*) (pv + i), v);
        } else {
            for (int64_t j = i; j < t.n; ++j) {
                float u;
                update(h, decay, t.p[j], load_grad1(t.g, t.gtype, j), pm[j], pv[j], u);
            }
        }
    }
}

// The largest of a wave's values, in every lane. Magnitudes compare as their bits,
// with infinities and NaNs above all others.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t max_with(uint32_t x) {
    const uint32_t y = (uint32_t) __builtin_amdgcn_update_dpp(0, (int) x, CTRL, ROWS, 0xf, true);
    return x > y ? x : y;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    x = max_with<0x111, 0xf>(x);  // from the lane before in the row of 16, then 2, 4 and 8 before
    x = max_with<0x112, 0xf>(x);
    x = max_with<0x114, 0xf>(x);
    x = max_with<0x118, 0xf>(x);
    x = max_with<0x142, 0xa>(x);  // the last lanes of rows 0 and 2 to rows 1 and 3, of row 1 to rows 2 and 3
    x = max_with<0x143, 0xc>(x);
    return (uint32_t) __builtin_amdgcn_readlane((int) x, 63);
}

__device__ __forceinline__ float inverse_scale(float s) {
    return s >= 0x1p-126f || s != s ? 1.f / s : 0.f;
}

constexpr float M_UNIT = (float) (1.0 / (127.0 * 127.0)), U_UNIT = (float) (1.0 / (255.0 * 255.0));

__device__ __forceinline__ float decode_m(int8_t c, float s) {
    const float x = (float) c;
    return (fabsf(x) * x * s) * M_UNIT;
}
__device__ __forceinline__ float decode_u(uint8_t c, float s) {
    const float x = (float) c;
    return (x * x * s) * U_UNIT;
}

// One block of up to 256 elements by a wave, with every operation as it is defined.
__device__ __forceinline__ void exact_block(const AwTensor& t, const AwHyper& h, float decay, int64_t at) {
    const int lane = (int) threadIdx.x & 63;
    int8_t* const pm = (int8_t*) t.m;
    uint8_t* const pv = (uint8_t*) t.v;
    const int64_t i = at + lane * 4;
    const float sm = t.ms[at / AW_BLOCK], su = t.vs[at / AW_BLOCK];
    float p[4], g[4], m[4], u[4];
    int8_t cm[4];
    uint8_t cv[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {  // (elements past the end read the last one and are not stored)
        const int64_t j = min(i + k, t.n - 1);
        p[k] = t.p[j];
        g[k] = load_grad1(t.g, t.gtype, j);
        cm[k] = pm[j];
        cv[k] = pv[j];
    }
    uint32_t top_m = 0, top_u = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        m[k] = decode_m(cm[k], sm);
        u[k] = decode_u(cv[k], su);
        float v = u[k] * u[k];
        update(h, decay, p[k], g[k], m[k], v, u[k]);
        if (i + k < t.n) {
            top_m = max(top_m, __builtin_bit_cast(uint32_t, m[k]) & 0x7fffffffu);
            top_u = max(top_u, __builtin_bit_cast(uint32_t, u[k]) & 0x7fffffffu);
        }
    }
    float nm = __builtin_bit_cast(float, wave_max(top_m)), nu = __builtin_bit_cast(float, wave_max(top_u));
    const float im = inverse_scale(nm), iu = inverse_scale(nu);
    if (im == 0.f && nm < 1.f) nm = 0.f;
    if (iu == 0.f && nu < 1.f) nu = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float rm = rintf(sqrtf(fabsf(m[k]) * im) * 127.f), ru = u[k] * iu;
        const float rv = fmaxf(rintf(sqrtf(ru) * 255.f), ceilf(ru));  // (1 at least, where ru is above 0)
        if (i + k >= t.n) continue;
        t.p[i + k] = p[k];
        pm[i + k] = (int8_t) (int) copysignf(rm, m[k]);
        pv[i + k] = (uint8_t) (int) rv;
    }
    if (lane == 0) {
        t.ms[at / AW_BLOCK] = nm;
        t.vs[at / AW_BLOCK] = nu;
    }
}

// What a lane has of a whole block.
struct Block8 {
    f4u p;
    f4u g32;
    h4u g16;
    uint32_t m, v;
    float sm, su;
};

template <int GTYPE>
__device__ __forceinline__ void load_block(Block8& b, const AwTensor& t, int64_t at) {
    const int64_t i = at + ((int) threadIdx.x & 63) * 4;
    b.p = once((const f4u*) (t.p + i));
    if (GTYPE == TRC_HIP_TYPE_F32) {
        b.g32 = once((const f4u*) ((const float*) t.g + i));
    } else {
        b.g16 = once((const h4u*) ((const uint16_t*) t.g + i));
    }
    b.m = once((const u32u*) ((const uint8_t*) t.m + i));
    b.v = once((const u32u*) ((const uint8_t*) t.v + i));
    b.sm = t.ms[at / AW_BLOCK];
    b.su = t.vs[at / AW_BLOCK];
}

// The square root of 0, of an infinity or NaN, or of 2^-96 and more, correctly rounded: the instruction's is
// one unit off at most, and the signs of two residues tell which neighbour is nearest.
__device__ __forceinline__ float sqrt_from_2em96(float x) {
    const float s = __builtin_amdgcn_sqrtf(x);
    const float lower = __builtin_bit_cast(float, __builtin_bit_cast(int, s) - 1);
    const float upper = __builtin_bit_cast(float, __builtin_bit_cast(int, s) + 1);
    const float dl = __builtin_fmaf(-lower, s, x), du = __builtin_fmaf(-upper, s, x);
    float r = dl <= 0.f ? lower : s;
    return du > 0.f ? upper : r;
}

// A whole block. The arithmetic bounds this kernel, not memory, so it takes what is as good as the exact
// operations wherever that can be told: the square roots of the codes come from the instruction alone, within
// 2 units of the last place, which decides a code unless it is within 1e-4 of the middle of two. A wave that
// meets one such code, or a v above 0 and under 2^-96, leaves the block to exact_block()
// (returns whether it has to be left to that).
template <int GTYPE>
__device__ __forceinline__ bool fast_block(const Block8& b, const AwTensor& t, const AwHyper& h, float decay, int64_t at) {
    const int lane = (int) threadIdx.x & 63;
    const int64_t i = at + lane * 4;
    f4 p, m, u;
    uint32_t top_m = 0, top_u = 0, least = 0xffffffffu;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        float g = GTYPE == TRC_HIP_TYPE_F32   ? b.g32[k]
                  : GTYPE == TRC_HIP_TYPE_F16 ? half_bits_to_float(b.g16[k])
                                              : __builtin_bit_cast(float, (uint32_t) b.g16[k] << 16);
        float mk = decode_m((int8_t) (b.m >> 8 * k), b.sm), uk = decode_u((uint8_t) (b.v >> 8 * k), b.su);
        // (update(), but for the square root)
        g = g * h.gscale;
        mk = mk * h.b1 + g * h.c1;
        const float vk = (uk * uk) * h.b2 + (g * g) * h.c2;
        least = min(least, __builtin_bit_cast(uint32_t, vk) - 1u);  // 0 is above all others here
        uk = sqrt_from_2em96(vk);
        p[k] = b.p[k] * decay - (mk / (uk * h.root + h.eps)) * h.rate;
        m[k] = mk;
        u[k] = uk;
        top_m = max(top_m, __builtin_bit_cast(uint32_t, mk) & 0x7fffffffu);
        top_u = max(top_u, __builtin_bit_cast(uint32_t, uk) & 0x7fffffffu);
    }
    float nm = __builtin_bit_cast(float, wave_max(top_m)), nu = __builtin_bit_cast(float, wave_max(top_u));
    const float im = inverse_scale(nm), iu = inverse_scale(nu);
    if (im == 0.f && nm < 1.f) nm = 0.f;
    if (iu == 0.f && nu < 1.f) nu = 0.f;
    float off = 0.f;  // the largest distance of a ratio from its code
    int cm[4];
    uint32_t cv = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float tm = __builtin_amdgcn_sqrtf(fabsf(m[k]) * im) * 127.f, rm = __builtin_rintf(tm);
        const float ru = u[k] * iu, tu = __builtin_amdgcn_sqrtf(ru) * 255.f, rv = __builtin_rintf(tu);
        off = fmaxf(off, fmaxf(fabsf(tm - rm), fabsf(tu - rv)));
        cm[k] = (int) __builtin_copysignf(rm, m[k]);
        cv = __builtin_amdgcn_cvt_pk_u8_f32(fmaxf(rv, __builtin_ceilf(ru)), k, cv);
    }
    // (a NaN or an infinity is left to the exact operations too)
    const bool doubt = !(off < 0.4999f) || least < 0x0f7fffffu || top_u >= 0x7f800000u || top_m >= 0x7f800000u;
    if (__any(doubt)) return true;
    store_once((f4u*) (t.p + i), p);
    const uint32_t lo = __builtin_amdgcn_perm((uint32_t) cm[1], (uint32_t) cm[0], 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm((uint32_t) cm[3], (uint32_t) cm[2], 0x04000c0cu);
    store_once((u32u*) ((uint8_t*) t.m + i), lo | hi);
    store_once((u32u*) ((uint8_t*) t.v + i), cv);
    if (lane == 0) {
        t.ms[at / AW_BLOCK] = nm;
        t.vs[at / AW_BLOCK] = nu;
    }
    return false;
}

// A wave's two blocks; returns which of them are left.
template <int GTYPE>
__device__ __forceinline__ int chunk8(const AwTensor& t, const AwHyper& h, float decay, int64_t at) {
    constexpr int STEP = AW_THREADS * 4;
    static_assert(AW_CHUNK == 2 * STEP, "two blocks a wave");
    if (at + AW_BLOCK > t.n) return 3;
    Block8 b0, b1;
    load_block<GTYPE>(b0, t, at);
    if (at + STEP + AW_BLOCK > t.n) return fast_block<GTYPE>(b0, t, h, decay, at) ? 3 : 2;
    load_block<GTYPE>(b1, t, at + STEP);
    const bool left = fast_block<GTYPE>(b0, t, h, decay, at);
    return (left ? 1 : 0) | (fast_block<GTYPE>(b1, t, h, decay, at + STEP) ? 2 : 0);
}

__global__ __launch_bounds__(AW_THREADS) void k_adamw8(const AwTensor* __restrict__ tensors,
                                                        const uint32_t* __restrict__ owner, AwHyper h) {
    const AwTensor t = tensors[owner[blockIdx.x]];
    const float decay = (float) (1.0 - h.decay * (double) t.decay);
    const int wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    const int64_t at = ((int64_t) blockIdx.x - t.first) * AW_CHUNK + wave * AW_BLOCK;
    const int left = t.gtype == TRC_HIP_TYPE_F32   ? chunk8<TRC_HIP_TYPE_F32>(t, h, decay, at)
                     : t.gtype == TRC_HIP_TYPE_F16 ? chunk8<TRC_HIP_TYPE_F16>(t, h, decay, at)
                                                   : chunk8<TRC_HIP_TYPE_BF16>(t, h, decay, at);
    for (int k = 0; k < 2; ++k) {
        const int64_t block = at + k * (AW_THREADS * 4);
        if ((left >> k & 1) != 0 && block < t.n) exact_block(t, h, decay, block);
    }
}

__global__ __launch_bounds__(AW_THREADS) void k_adamw_moments(const AwTensor* __restrict__ tensors,
                                                               const uint32_t* __restrict__ owner, int bits) {
    const AwTensor t = tensors[owner[blockIdx.x]];
    const int64_t base = ((int64_t) blockIdx.x - t.first) * AW_CHUNK;
#pragma unroll
    for (int it = 0; it < AW_CHUNK / (AW_THREADS * 4); ++it) {
        const int64_t i = base + (it * AW_THREADS + (int) threadIdx.x) * 4;
        if (i >= t.n) return;
        if (bits == 32) {
            for (int64_t j = i; j < t.n && j < i + 4; ++j) {
                t.mf[j] = ((const float*) t.m)[j];
                t.vf[j] = ((const float*) t.v)[j];
            }
            continue;
        }
        const float sm = t.ms[i / AW_BLOCK], su = t.vs[i / AW_BLOCK];
        if (i + 4 <= t.n) {
            const b4u cm = *(const b4u*) ((const uint8_t*) t.m + i), cv = *(const b4u*) ((const uint8_t*) t.v + i);
            f4 m, v;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float u = decode_u(cv[k], su);
                m[k] = decode_m((int8_t) cm[k], sm);
                v[k] = u * u;
            }
            store_once((f4u*) (t.mf + i), m);
            store_once((f4u*) (t.vf + i), v);
        } else {
            for (int64_t j = i; j < t.n; ++j) {
                const float u = decode_u(((const uint8_t*) t.v)[j], su);
                t.mf[j] = decode_m(((const int8_t*) t.m)[j], sm);
                t.vf[j] = u * u;
            }
        }
    }
}

bool at_least(const void* p, size_t align) { return p != nullptr && ((uintptr_t) p & (align - 1)) == 0; }

}  // namespace

int adamw_create(const trc_hip_adamw_tensor* ts, int64_t count, int bits, void** plan) {
    std::vector<AwTensor> host;
    std::vector<uint32_t> owner;
    int64_t chunks = 0;
    bool readable = true;
    for (int64_t i = 0; i < count; ++i) {
        const trc_hip_adamw_tensor& t = ts[i];
        const char* const who = "trc_hip_adamw_create";
        if (t.n < 0) return fail(TRC_HIP_E_SHAPE, "%s: tensor %lld has %lld elements", who, (long long) i, (long long) t.n);
        if (t.grad_type != TRC_HIP_TYPE_F32 && t.grad_type != TRC_HIP_TYPE_F16 && t.grad_type != TRC_HIP_TYPE_BF16) {
            return fail(TRC_HIP_E_INVALID, "%s: tensor %lld: gradient type %d is not F32, F16 or BF16", who, (long long) i,
                        t.grad_type);
        }
        if (t.n == 0) continue;
        const size_t ga = t.grad_type == TRC_HIP_TYPE_F32 ? 4 : 2, sa = bits == 32 ? 4 : 1;
        if (!at_least(t.param, 4) || !at_least(t.grad, ga) || !at_least(t.m, sa) || !at_least(t.v, sa) ||
            (bits == 8 && (!at_least(t.m_scale, 4) || !at_least(t.v_scale, 4))) || ((uintptr_t) t.m_out & 3u) != 0 ||
            ((uintptr_t) t.v_out & 3u) != 0) {
            return fail(TRC_HIP_E_ALIGN, "%s: tensor %lld: a pointer is NULL or not aligned to its elements", who,
                        (long long) i);
        }
        readable = readable && t.m_out != nullptr && t.v_out != nullptr;
        const int64_t c = (t.n - 1) / AW_CHUNK + 1;
        if (chunks + c > max_groups(AW_THREADS)) {
            return fail(TRC_HIP_E_SHAPE, "%s: over %lld elements in one plan", who,
                        (long long) (max_groups(AW_THREADS) * AW_CHUNK));
        }
        owner.insert(owner.end(), (size_t) c, (uint32_t) host.size());
        host.push_back({t.param, t.grad, t.m, t.v, t.m_scale, t.v_scale, t.m_out, t.v_out, t.n, chunks, t.decay, t.grad_type});
        chunks += c;
    }
    Plan* const p = new Plan{0, bits, readable, chunks, nullptr, nullptr};
    int rc = hip_error(hipGetDevice(&p->dev), "hipGetDevice");
    if (rc == TRC_HIP_OK && chunks > 0) {
        const size_t tb = host.size() * sizeof(AwTensor);
        uint8_t* d = nullptr;
        rc = hip_error(hipMalloc((void**) &d, tb + owner.size() * sizeof(uint32_t)), "trc_hip_adamw_create: hipMalloc");
        if (rc == TRC_HIP_OK) {
            p->tensors = (AwTensor*) d;
            p->owner = (uint32_t*) (d + tb);
            rc = hip_error(hipMemcpy(d, host.data(), tb, hipMemcpyHostToDevice), "trc_hip_adamw_create: hipMemcpy");
            if (rc == TRC_HIP_OK) {
                rc = hip_error(hipMemcpy(p->owner, owner.data(), owner.size() * sizeof(uint32_t), hipMemcpyHostToDevice),
                               "trc_hip_adamw_create: hipMemcpy");
            }
            if (rc != TRC_HIP_OK) (void) hipFree(d);
        }
    }
    if (rc != TRC_HIP_OK) {
        delete p;
        return rc;
    }
    *plan = p;
    return TRC_HIP_OK;
}

// The plan's tables are on one device; a launch from another would read them there.
static int same_device(const char* who, const Plan& p) {
    int dev = 0;
    const int rc = hip_error(hipGetDevice(&dev), "hipGetDevice");
    if (rc != TRC_HIP_OK) return rc;
    if (dev != p.dev) {
        return fail(TRC_HIP_E_INVALID, "%s: the plan is of device %d, the current one is %d", who, p.dev, dev);
    }
    return TRC_HIP_OK;
}

int adamw_step(void* plan, const trc_hip_adamw_hyper& q, hipStream_t s) {
    const Plan& p = *(const Plan*) plan;
    const int rc = same_device("trc_hip_adamw_step", p);
    if (rc != TRC_HIP_OK || p.chunks == 0) return rc;
    const double t = (double) q.step;
    AwHyper h;
    h.b1 = (float) q.beta1;
    h.c1 = (float) (1.0 - q.beta1);
    h.b2 = (float) q.beta2;
    h.c2 = (float) (1.0 - q.beta2);
    h.eps = (float) q.eps;
    h.decay = q.lr * q.weight_decay;
    h.rate = (float) (q.lr / (1.0 - std::pow(q.beta1, t)));
    h.root = (float) (1.0 / std::sqrt(1.0 - std::pow(q.beta2, t)));
    h.gscale = (float) q.grad_scale;
    hipLaunchKernelGGL(p.bits == 32 ? k_adamw : k_adamw8, dim3((unsigned) p.chunks), dim3(AW_THREADS), 0, s, p.tensors,
                       p.owner, h);
    return check_launch("adamw_step");
}

int adamw_moments(void* plan, hipStream_t s) {
    const Plan& p = *(const Plan*) plan;
    int rc = same_device("trc_hip_adamw_moments", p);
    if (rc != TRC_HIP_OK || p.chunks == 0) return rc;
    if (!p.readable) {
        return fail(TRC_HIP_E_INVALID, "trc_hip_adamw_moments: the plan was made without m_out and v_out of every tensor");
    }
    hipLaunchKernelGGL(k_adamw_moments, dim3((unsigned) p.chunks), dim3(AW_THREADS), 0, s, p.tensors, p.owner, p.bits);
    return check_launch("adamw_moments");
}

int adamw_destroy(void* plan) {
    Plan* const p = (Plan*) plan;
    const int rc = p->tensors != nullptr ? hip_error(hipFree(p->tensors), "hipFree") : TRC_HIP_OK;
    delete p;
    return rc;
}

}  // namespace trc_hip
