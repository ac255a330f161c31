// The optimizer of include/traincpp/trc_hip.h: HipAdamW's steps against a restatement in 64 bits, its moments, and
// its state put into another optimizer, which has to go on bit for bit.
//
//   test_tuning                 all cases
//   test_tuning --abort-host    an adapter call with tensors that are in no HIP buffer (must abort; needs no device)
#include "traincpp/traincpp.h"

#include <cmath>
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

std::vector<float> wave(size_t n, double f, double a) {
    std::vector<float> v(n);
    for (size_t i = 0; i < n; ++i) v[i] = (float) (a * std::sin(f * (double) (i + 1)));
    return v;
}
std::vector<float> get(const Tensor* t) {
    std::vector<float> v((size_t) tensor_nelements(t));
    tensor_get(t, v.data(), 0, v.size() * 4);
    return v;
}
bool same(const std::vector<float>& a, const std::vector<float>& b) {
    return a.size() == b.size() && std::memcmp(a.data(), b.data(), a.size() * 4) == 0;
}

void optimizer(Device* dev, int bits) {
    const int64_t sizes[3] = {1000, 7, 4096};
    const float decay[3] = {1.f, 0.f, 1.f};
    Context* ctx = context_new(1 << 20);
    Tensor *p[2][3], *g[3];
    for (int i = 0; i < 3; ++i) {
        for (int k = 0; k < 2; ++k) p[k][i] = new_tensor_1d(ctx, TYPE_F32, sizes[i]);
        g[i] = new_tensor_1d(ctx, TYPE_F32, sizes[i]);
    }
    Buffer* buf = buffer_alloc_ctx_tensors(ctx, dev->default_buffer_type());
    HipAdamWParams q;
    q.lr = 1e-2;
    q.weight_decay = 0.1;
    {
        HipAdamW a(p[0], g, 3, bits, decay), b(p[1], g, 3, bits, decay);
        std::vector<std::vector<double>> wp(3), wm(3), wv(3);
        for (int i = 0; i < 3; ++i) {
            const std::vector<float> v = wave((size_t) sizes[i], 0.7, 1.0);
            tensor_set(p[0][i], v.data(), 0, v.size() * 4);
            wp[i].assign(v.begin(), v.end());
            wm[i].assign(v.size(), 0.0);
            wv[i].assign(v.size(), 0.0);
        }
        auto step = [&](int s, HipAdamW& o) {
            for (int i = 0; i < 3; ++i) {
                const std::vector<float> v = wave((size_t) sizes[i], 0.31 + s, 0.1);
                tensor_set(g[i], v.data(), 0, v.size() * 4);
            }
            o.step(q);
        };
        for (int s = 1; s <= 3; ++s) {
            step(s, a);
            for (int i = 0; i < 3; ++i) {
                const std::vector<float> v = wave((size_t) sizes[i], 0.31 + s, 0.1);
                for (size_t k = 0; k < v.size(); ++k) {
                    wm[i][k] = q.beta1 * wm[i][k] + (1 - q.beta1) * v[k];
                    wv[i][k] = q.beta2 * wv[i][k] + (1 - q.beta2) * (double) v[k] * v[k];
                    wp[i][k] -= q.lr * q.weight_decay * decay[i] * wp[i][k];
                    wp[i][k] -= q.lr / (1 - std::pow(q.beta1, s)) * wm[i][k] /
                                (std::sqrt(wv[i][k] / (1 - std::pow(q.beta2, s))) + q.eps);
                }
            }
        }
        EXPECT(a.steps() == 3);
        for (int i = 0; i < 3; ++i) {
            const std::vector<float> v = get(p[0][i]);
            std::vector<float> m(v.size()), u(v.size());
            a.moments((size_t) i, m.data(), u.data());
            double ep = 0, em = 0;
            for (size_t k = 0; k < v.size(); ++k) {
                ep = std::fmax(ep, std::fabs(v[k] - wp[i][k]));
                em = std::fmax(em, std::fabs(m[k] - wm[i][k]));
            }
            // 32 bits: some 30 roundings a step of values up to 1; 8 bits: each step moves a parameter by lr at
            // most, and its codes are off by 1 / 254 of their block's largest moment (0.03 here) a step
            EXPECT(ep <= (bits == 32 ? 3 * 30 * 0x1p-24 : 3 * q.lr) && em <= (bits == 32 ? 1e-8 : 3 * 0.03 / 127));
        }
        // another optimizer takes over: same parameters, same state
        std::vector<uint8_t> state(a.state_bytes());
        a.get_state(state.data());
        b.set_state(state.data(), a.steps());
        for (int i = 0; i < 3; ++i) {
            const std::vector<float> v = get(p[0][i]);
            tensor_set(p[1][i], v.data(), 0, v.size() * 4);
        }
        for (int s = 4; s <= 6; ++s) {
            step(s, a);
            b.step(q);
        }
        for (int i = 0; i < 3; ++i) EXPECT(same(get(p[0][i]), get(p[1][i])));
        EXPECT(b.steps() == 6);
    }
    buffer_free(buf);
    context_free(ctx);
    std::printf("    optimizer, %d bits: done\n", bits);
}

void wrong_call() {
    Context* ctx = context_new(1 << 20);
    HipLoraSet s;
    s.a = new_tensor_3d(ctx, TYPE_F32, 64, 8, 1);
    s.b = new_tensor_3d(ctx, TYPE_F32, 8, 32, 1);
    s.scale = new_tensor_1d(ctx, TYPE_F32, 1);
    s.start = new_tensor_1d(ctx, TYPE_I32, 2);
    s.adapter = new_tensor_1d(ctx, TYPE_I32, 1);
    Tensor* x = new_tensor_2d(ctx, TYPE_F32, 64, 4);
    Tensor* h = new_tensor_2d(ctx, TYPE_F32, 8, 4);
    Tensor* y = new_tensor_2d(ctx, TYPE_F32, 32, 4);
    hip_lora(s, x, nullptr, h, y);
}

}  // namespace

int main(int argc, char** argv) {
    if (argc > 1 && std::strcmp(argv[1], "--abort-host") == 0) {
        wrong_call();
        return 0;
    }
    Device* dev = hip_device(0);
    if (dev == nullptr) {
        std::fprintf(stderr, "test_tuning: no HIP device\n");
        return 77;
    }
    optimizer(dev, 32);
    optimizer(dev, 8);
    std::printf("%s: %d failure(s)\n", g_failures == 0 ? "PASS" : "FAIL", g_failures);
    return g_failures == 0 ? 0 : 1;
}
