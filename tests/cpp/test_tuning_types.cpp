// The tuning calls of include/traincpp/trc_hip.h in each of their types: HipAdamW's 8-bit step against its definition, bit
// for bit and from the first step on, and adapters in F32, F16 and BF16 with their gradients against 64 bits.
#include "traincpp/traincpp.h"

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <vector>

using namespace traincpp;

namespace {

int g_failures = 0;
#define EXPECT(cond)                                                         \
    do {                                                                     \
        if (!(cond)) {                                                       \
            std::printf("    FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); \
            ++g_failures;                                                    \
        }                                                                    \
    } while (0)

template <class T>
void set(Tensor* t, const std::vector<T>& v) {
    tensor_set(t, v.data(), 0, v.size() * sizeof(T));
}
std::vector<float> get(const Tensor* t) {
    std::vector<float> v((size_t) tensor_nelements(t));
    tensor_get(t, v.data(), 0, v.size() * 4);
    return v;
}
std::vector<float> wave(size_t n, double f, double a) {
    std::vector<float> v(n);
    for (size_t i = 0; i < n; ++i) v[i] = (float) (a * std::sin(f * (double) (i + 1)));
    return v;
}
bool same(const std::vector<float>& a, const std::vector<float>& b) {
    return a.size() == b.size() && std::memcmp(a.data(), b.data(), a.size() * 4) == 0;
}

// ---- the 8-bit step, each operation rounded to 32 bits: blocks of 256 share the scales sm and su,
//   m = sm sign(c) (c / 127)^2     sqrt(v) = su (c / 255)^2, c at least 1 where v > 0
constexpr size_t BLOCK = 256;

struct Moments {
    std::vector<float> cm, cu, sm, su;  // codes and scales
    explicit Moments(size_t n) : cm(n), cu(n), sm((n + BLOCK - 1) / BLOCK), su(sm.size()) {}
    float m(size_t i) const { return std::fabs(cm[i]) * cm[i] * sm[i / BLOCK] * (float) (1.0 / (127.0 * 127.0)); }
    float u(size_t i) const { return cu[i] * cu[i] * su[i / BLOCK] * (float) (1.0 / (255.0 * 255.0)); }
};

void step8(std::vector<float>& p, const std::vector<float>& g, Moments& s, const HipAdamWParams& q, float decay, int step) {
    const float b1 = (float) q.beta1, c1 = (float) (1.0 - q.beta1), b2 = (float) q.beta2, c2 = (float) (1.0 - q.beta2);
    const float eps = (float) q.eps, rate = (float) (q.lr / (1.0 - std::pow(q.beta1, step)));
    const float root = (float) (1.0 / std::sqrt(1.0 - std::pow(q.beta2, step)));
    const float shrink = (float) (1.0 - q.lr * q.weight_decay * (double) decay);
    for (size_t at = 0; at < p.size(); at += BLOCK) {
        const size_t n = std::min(BLOCK, p.size() - at);
        float m[BLOCK], u[BLOCK], top_m = 0, top_u = 0;
        for (size_t k = 0; k < n; ++k) {
            const float gk = g[at + k] * (float) q.grad_scale, old = s.u(at + k);
            m[k] = s.m(at + k) * b1 + gk * c1;
            u[k] = std::sqrt((old * old) * b2 + (gk * gk) * c2);
            p[at + k] = p[at + k] * shrink - (m[k] / (u[k] * root + eps)) * rate;
            top_m = std::fmax(top_m, std::fabs(m[k]));
            top_u = std::fmax(top_u, u[k]);
        }
        s.sm[at / BLOCK] = top_m >= 0x1p-126f ? top_m : 0.f;
        s.su[at / BLOCK] = top_u >= 0x1p-126f ? top_u : 0.f;
        const float im = top_m >= 0x1p-126f ? 1.f / top_m : 0.f, iu = top_u >= 0x1p-126f ? 1.f / top_u : 0.f;
        for (size_t k = 0; k < n; ++k) {
            s.cm[at + k] = std::copysign(std::rint(std::sqrt(std::fabs(m[k]) * im) * 127.f), m[k]) + 0.f;  // (a code has one zero)
            const float ru = u[k] * iu;
            s.cu[at + k] = std::fmax(std::rint(std::sqrt(ru) * 255.f), ru > 0 ? 1.f : 0.f);
        }
    }
}

void optimizer8(Device* dev) {
    const int64_t sizes[4] = {1000, 7, 4096, 256};
    const float decay[4] = {1.f, 0.f, 1.f, 0.5f};
    Context* ctx = context_new(1 << 20);
    Tensor *p[4], *g[4];
    std::vector<std::vector<float>> want;
    std::vector<Moments> state;
    for (int i = 0; i < 4; ++i) {
        p[i] = new_tensor_1d(ctx, TYPE_F32, sizes[i]);
        g[i] = new_tensor_1d(ctx, TYPE_F32, sizes[i]);
        want.push_back(wave((size_t) sizes[i], 0.7, 1.0));
        state.emplace_back((size_t) sizes[i]);
    }
    Buffer* buf = buffer_alloc_ctx_tensors(ctx, dev->default_buffer_type());
    for (int i = 0; i < 4; ++i) set(p[i], want[(size_t) i]);
    HipAdamWParams q;
    q.lr = 1e-2;
    q.weight_decay = 0.1;
    {
        HipAdamW o(p, g, 4, 8, decay);
        for (int s = 1; s <= 4; ++s) {
            q.grad_scale = s == 3 ? 0.25 : 1.0;
            for (int i = 0; i < 4; ++i) {
                const std::vector<float> v = wave((size_t) sizes[i], 0.31 + s, s == 2 ? 10.0 : 0.1);
                set(g[i], v);
                step8(want[(size_t) i], v, state[(size_t) i], q, decay[i], s);
            }
            o.step(q);
            for (size_t i = 0; i < 4; ++i) {
                EXPECT(same(get(p[i]), want[i]));
                std::vector<float> m(want[i].size()), v(m.size()), wm(m.size()), wv(m.size());
                o.moments(i, m.data(), v.data());
                for (size_t k = 0; k < m.size(); ++k) {
                    wm[k] = state[i].m(k);
                    wv[k] = state[i].u(k) * state[i].u(k);
                }
                EXPECT(same(m, wm) && same(v, wv));
            }
        }
    }
    buffer_free(buf);
    context_free(ctx);
    std::printf("    optimizer, 8 bits: done\n");
}

// ---- adapters

// Multiples of 1/64 under 1, which every type holds; as the bits of `type`.
std::vector<double> weights(size_t n, uint64_t seed) {
    std::vector<double> v(n);
    for (double& x : v) {
        seed = seed * 6364136223846793005ull + 1442695040888963407ull;
        x = (double) ((int64_t) (seed >> 33) % 127 - 63) / 64;
    }
    return v;
}
void set_weights(Tensor* t, const std::vector<double>& v) {
    if (t->type == TYPE_F32) return set(t, std::vector<float>(v.begin(), v.end()));
    std::vector<uint16_t> h;
    for (double x : v) {
        const float f = (float) x;
        uint32_t b;
        std::memcpy(&b, &f, 4);
        const uint32_t sign = b >> 16 & 0x8000, rest = b & 0x7fffffff;
        h.push_back((uint16_t) (t->type == TYPE_BF16 ? b >> 16 : rest == 0 ? sign : sign | ((rest - (112u << 23)) >> 13)));
    }
    set(t, h);
}

// A sum of n terms in 32 bits is within 8 sqrt(n) 2^-24 of the sum of their magnitudes.
void near(const std::vector<float>& got, const std::vector<double>& want, const std::vector<double>& mags, double n) {
    bool ok = got.size() == want.size();
    for (size_t i = 0; ok && i < got.size(); ++i) ok = std::fabs(got[i] - want[i]) <= 8 * std::sqrt(n) * 0x1p-24 * mags[i] + 1e-30;
    EXPECT(ok);
}

void adapters(Device* dev, Type type) {
    const size_t K = 200, M = 136, R = 12, n = 2;
    const std::vector<int32_t> start{0, 1, 20, 23}, ids{1, 0, -1};
    const size_t T = 23;
    Context* ctx = context_new(1 << 20);
    HipLoraSet s;
    s.a = new_tensor_3d(ctx, type, K, R, n);
    s.b = new_tensor_3d(ctx, type, R, M, n);
    s.scale = new_tensor_1d(ctx, TYPE_F32, n);
    s.start = new_tensor_1d(ctx, TYPE_I32, 4);
    s.adapter = new_tensor_1d(ctx, TYPE_I32, 3);
    Tensor* x = new_tensor_2d(ctx, TYPE_F32, K, T);
    Tensor* base = new_tensor_2d(ctx, TYPE_F32, M, T);
    Tensor* h = new_tensor_2d(ctx, TYPE_F32, R, T);
    Tensor* y = new_tensor_2d(ctx, TYPE_F32, M, T);
    Tensor* dy = new_tensor_2d(ctx, TYPE_F32, M, T);
    Tensor* g = new_tensor_2d(ctx, TYPE_F32, R, T);
    Tensor* dx = new_tensor_2d(ctx, TYPE_F32, K, T);
    Tensor* da = new_tensor_3d(ctx, TYPE_F32, K, R, n);
    Tensor* db = new_tensor_3d(ctx, TYPE_F32, R, M, n);
    Buffer* buf = buffer_alloc_ctx_tensors(ctx, dev->default_buffer_type());
    const std::vector<double> a = weights(K * R * n, 3), b = weights(R * M * n, 4);
    const std::vector<float> scale{0.5f, 1.75f}, xv = wave(K * T, 0.9, 1.0), bv = wave(M * T, 0.37, 2.0), dv = wave(M * T, 1.3, 0.5);
    set_weights(s.a, a);
    set_weights(s.b, b);
    set(s.scale, scale);
    set(s.start, start);
    set(s.adapter, ids);
    set(x, xv);
    set(base, bv);
    set(dy, dv);
    hip_lora(s, x, base, h, y);
    const std::vector<float> hv = get(h);

    struct Sum {
        std::vector<double> v, m;
        explicit Sum(size_t n) : v(n), m(n) {}
        void add(size_t i, double x, double mag) { v[i] += x, m[i] += mag; }
    };
    Sum wh(R * T), wy(M * T), wg(R * T), wx(K * T), wa(K * R * n), wb(R * M * n);
    for (size_t q = 0; q < ids.size(); ++q) {
        for (size_t t = (size_t) start[q]; t < (size_t) start[q + 1]; ++t) {
            for (size_t i = 0; i < M; ++i) wy.add(t * M + i, bv[t * M + i], std::fabs(bv[t * M + i]));
            if (ids[q] < 0) continue;
            const double* A = &a[(size_t) ids[q] * K * R];
            const double* B = &b[(size_t) ids[q] * R * M];
            const double sc = scale[(size_t) ids[q]];
            for (size_t r = 0; r < R; ++r) {
                for (size_t k = 0; k < K; ++k) wh.add(t * R + r, A[r * K + k] * xv[t * K + k], std::fabs(A[r * K + k] * xv[t * K + k]));
                for (size_t i = 0; i < M; ++i) {
                    const double z = sc * B[i * R + r] * dv[t * M + i], w = sc * dv[t * M + i] * hv[t * R + r];
                    wg.add(t * R + r, z, std::fabs(z));
                    wb.add((size_t) ids[q] * R * M + i * R + r, w, std::fabs(w));
                }
            }
            for (size_t r = 0; r < R; ++r) {
                const size_t at = t * R + r;
                for (size_t i = 0; i < M; ++i) wy.add(t * M + i, sc * B[i * R + r] * wh.v[at], sc * std::fabs(B[i * R + r]) * wh.m[at]);
                for (size_t k = 0; k < K; ++k) {
                    wx.add(t * K + k, A[r * K + k] * wg.v[at], std::fabs(A[r * K + k]) * wg.m[at]);
                    wa.add((size_t) ids[q] * K * R + r * K + k, wg.v[at] * xv[t * K + k], wg.m[at] * std::fabs(xv[t * K + k]));
                }
            }
        }
    }
    near(hv, wh.v, wh.m, K + 2);
    near(get(y), wy.v, wy.m, K + R + 4);
    hip_lora_back(s, x, h, dy, g, nullptr, dx, da, db);
    near(get(g), wg.v, wg.m, M + 3);
    near(get(dx), wx.v, wx.m, M + R + 5);
    near(get(da), wa.v, wa.m, M + T + 5);
    near(get(db), wb.v, wb.m, T + 5);
    hip_lora_back(s, x, h, dy, g, nullptr, nullptr, da, db, true);  // added to what is there: twice the gradients
    for (Sum* w : {&wa, &wb}) {
        for (double& v : w->v) v *= 2;
        for (double& v : w->m) v *= 2;
    }
    near(get(da), wa.v, wa.m, M + T + 6);
    near(get(db), wb.v, wb.m, T + 6);
    buffer_free(buf);
    context_free(ctx);
    std::printf("    adapters, type %d: done\n", (int) type);
}

}  // namespace

int main() {
    Device* dev = hip_device(0);
    if (dev == nullptr) {
        std::fprintf(stderr, "test_tuning_types: no HIP device\n");
        return 77;
    }
    optimizer8(dev);
    for (Type type : {TYPE_F32, TYPE_F16, TYPE_BF16}) adapters(dev, type);
    std::printf("%s: %d failure(s)\n", g_failures == 0 ? "PASS" : "FAIL", g_failures);
    return g_failures == 0 ? 0 : 1;
}
