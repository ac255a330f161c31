// The 8-bit floating point and distillation calls of include/traincpp/trc_hip.h, run together as a tuning step does: every
// result against 64 bits from the operands that the device holds, and the loss's gradient by an adapter against
// differences of the loss.
//
// Tolerances, u = 2^-24: a sum of n terms in 32 bits is within 8 sqrt(n) u of the sum of their magnitudes (and no
// more than n u, where n is small). The loss's rows: see the relative error e_s of a sum of V exponentials in `losses`.
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

typedef std::vector<double> Doubles;
constexpr double U = 0x1p-24;

template <class T>
void set(Tensor* t, const std::vector<T>& v) {
    tensor_set(t, v.data(), 0, v.size() * sizeof(T));
}
template <class T = float>
std::vector<T> get(const Tensor* t) {
    std::vector<T> v((size_t) tensor_nelements(t));
    tensor_get(t, v.data(), 0, v.size() * sizeof(T));
    return v;
}
Doubles wide(const std::vector<float>& v) { return Doubles(v.begin(), v.end()); }
std::vector<float> wave(size_t n, double f, double a) {
    std::vector<float> v(n);
    for (size_t i = 0; i < n; ++i) v[i] = (float) (a * std::sin(f * (double) (i + 1)) * std::cos(0.37 * f * (double) (i * i % 1013)));
    return v;
}

// The value of an e4m3 code.
double e4m3(uint8_t c) {
    const int e = c >> 3 & 15, m = c & 7;
    const double v = e == 0 ? std::ldexp(m, -9) : std::ldexp(8 + m, e - 10);
    return c & 128 ? -v : v;
}

// What quantized rows hold, from their parents (whole rows of blocks).
Doubles values(const HipFp8& f, bool weight) {
    const size_t K = (size_t) f.q->ne[0], R = (size_t) f.q->ne[1], pitch = f.q->nb[1], words = f.scale->nb[1];
    std::vector<uint8_t> q(pitch * (R - 1) + K), s(words * ((size_t) f.scale->ne[1] - 1) + (size_t) f.scale->ne[0]);
    tensor_get(f.q, q.data(), 0, q.size());
    tensor_get(f.scale, s.data(), 0, s.size());
    Doubles v(K * R);
    for (size_t r = 0; r < R; ++r)
        for (size_t k = 0; k < K; ++k)
            v[r * K + k] = std::ldexp(e4m3(q[r * pitch + k]), (int) s[(weight ? r / 128 : r) * words + k / 128] - 127);
    return v;
}

// Within half a step of x: 2^-4 of it, or half the smallest code's step, 2^-10 times the scale, which is at most
// twice amax / 448.
void quantized(const Doubles& x, const Doubles& q, size_t K, size_t R, bool weight) {
    bool ok = true;
    const size_t rows = weight ? 128 : 1;
    for (size_t r0 = 0; r0 < R; r0 += rows)
        for (size_t k0 = 0; k0 < K; k0 += 128) {
            double amax = 0;
            auto each = [&](auto f) {
                for (size_t r = r0; r < std::min(R, r0 + rows); ++r)
                    for (size_t k = k0; k < std::min(K, k0 + 128); ++k) f(r * K + k);
            };
            each([&](size_t i) { amax = std::fmax(amax, std::fabs(x[i])); });
            each([&](size_t i) { ok = ok && std::fabs(q[i] - x[i]) <= std::fmax(0x1p-4 * std::fabs(x[i]), 0x1p-10 * amax / 224); });
        }
    EXPECT(ok);
}

void near(const std::vector<float>& got, const Doubles& want, const Doubles& mags, double n, const char* what) {
    double worst = 0;
    for (size_t i = 0; i < got.size(); ++i)
        worst = std::fmax(worst, std::fabs(got[i] - want[i]) / (std::fmin(8 * std::sqrt(n), 2 * n) * U * mags[i] + 1e-30));
    std::printf("    %s: %.3g of the bound\n", what, worst);
    EXPECT(got.size() == want.size() && worst <= 1);
}

struct Sum {
    Doubles v, m;
    explicit Sum(size_t n) : v(n), m(n) {}
    void add(size_t i, double x, double mag) { v[i] += x, m[i] += mag; }
};

// y [M, T] = W x, or W^T x with `back`
Sum product(const Doubles& w, const Doubles& x, size_t K, size_t M, size_t T, bool back) {
    Sum y((back ? K : M) * T);
    for (size_t t = 0; t < T; ++t)
        for (size_t m = 0; m < M; ++m)
            for (size_t k = 0; k < K; ++k) {
                const double z = w[m * K + k] * x[back ? t * M + m : t * K + k];
                y.add(back ? t * K + k : t * M + m, z, std::fabs(z));
            }
    return y;
}

template <class T>
void put(Tensor* t, const std::vector<T>& v) {
    set(t, v);
}

struct Adapter {
    HipLoraSet set;
    Tensor *da, *db, *h, *g;
    size_t in, out, R = 8;
    Adapter(Context* ctx, size_t i, size_t o, size_t T) : in(i), out(o) {
        set.a = new_tensor_3d(ctx, TYPE_F32, (int64_t) in, (int64_t) R, 1);
        set.b = new_tensor_3d(ctx, TYPE_F32, (int64_t) R, (int64_t) out, 1);
        set.scale = new_tensor_1d(ctx, TYPE_F32, 1);
        set.start = new_tensor_1d(ctx, TYPE_I32, 2);
        set.adapter = new_tensor_1d(ctx, TYPE_I32, 1);
        da = new_tensor_3d(ctx, TYPE_F32, (int64_t) in, (int64_t) R, 1);
        db = new_tensor_3d(ctx, TYPE_F32, (int64_t) R, (int64_t) out, 1);
        h = new_tensor_2d(ctx, TYPE_F32, (int64_t) R, (int64_t) T);
        g = new_tensor_2d(ctx, TYPE_F32, (int64_t) R, (int64_t) T);
    }
    void fill(size_t T) {
        put(set.a, wave(in * R, 0.83, 0.1));
        put(set.b, wave(R * out, 1.31, 0.1));
        put(set.scale, std::vector<float>{1.5f});
        put(set.start, std::vector<int32_t>{0, (int32_t) T});
        put(set.adapter, std::vector<int32_t>{0});
    }
    // the gradients of A, B and the input by dy, from what the device holds
    void check(const Doubles& x, const Doubles& dy, const Doubles* base, Tensor* dx, size_t T, const char* what) const {
        const Doubles A = wide(get(set.a)), B = wide(get(set.b)), hv = wide(get(h));
        Sum wg(R * T), wa(in * R), wb(R * out), wx(in * T);
        for (size_t t = 0; t < T; ++t) {
            for (size_t i = 0; i < out; ++i)
                for (size_t r = 0; r < R; ++r) {
                    const double z = 1.5 * B[i * R + r] * dy[t * out + i], w = 1.5 * dy[t * out + i] * hv[t * R + r];
                    wg.add(t * R + r, z, std::fabs(z));
                    wb.add(i * R + r, w, std::fabs(w));
                }
            for (size_t r = 0; r < R; ++r)
                for (size_t k = 0; k < in; ++k) {
                    wa.add(r * in + k, wg.v[t * R + r] * x[t * in + k], wg.m[t * R + r] * std::fabs(x[t * in + k]));
                    wx.add(t * in + k, wg.v[t * R + r] * A[r * in + k], wg.m[t * R + r] * std::fabs(A[r * in + k]));
                }
            if (base != nullptr)
                for (size_t k = 0; k < in; ++k) wx.add(t * in + k, (*base)[t * in + k], std::fabs((*base)[t * in + k]));
        }
        std::printf("  adapter %s\n", what);
        near(get(da), wa.v, wa.m, (double) (out + T + 5), "dA");
        near(get(db), wb.v, wb.m, (double) (T + 5), "dB");
        if (dx != nullptr) near(get(dx), wx.v, wx.m, (double) (out + R + 6), "dx");
    }
};

struct Loss {
    double loss = 0;
    Doubles d, mags;  // the gradient, and what its terms weigh
};
// The formulas, from logits in 64 bits.
Loss losses(const HipDistillation& q, const Doubles& l, size_t V, size_t T) {
    const std::vector<int32_t> labels = get<int32_t>(q.labels), ids = get<int32_t>(q.ids);
    const Doubles z = wide(get(q.teacher));
    const size_t top = (size_t) q.ids->ne[0];
    const double tau = q.tau, alpha = q.alpha;
    Loss out;
    out.d.assign(V * T, 0.0);
    out.mags.assign(V * T, 0.0);
    size_t n = 0;
    for (int32_t y : labels) n += y >= 0;
    for (size_t t = 0; t < T; ++t) {
        if (labels[t] < 0) continue;
        double m = l[t * V], s1 = 0, st = 0, zm = -1e30, zs = 0;
        for (size_t v = 0; v < V; ++v) m = std::fmax(m, l[t * V + v]);
        for (size_t v = 0; v < V; ++v) s1 += std::exp(l[t * V + v] - m), st += std::exp((l[t * V + v] - m) / tau);
        for (size_t v = 0; v < V; ++v) {
            const double qv = std::exp((l[t * V + v] - m) / tau) / st, rv = std::exp(l[t * V + v] - m) / s1;
            out.d[t * V + v] = out.mags[t * V + v] = (alpha * tau * qv + (1 - alpha) * rv) / (double) n;
        }
        auto in = [&](size_t j) { return ids[t * top + j] >= 0 && (size_t) ids[t * top + j] < V; };
        for (size_t j = 0; j < top; ++j)
            if (in(j)) zm = std::fmax(zm, z[t * top + j]);
        for (size_t j = 0; j < top; ++j)
            if (in(j)) zs += std::exp((z[t * top + j] - zm) / tau);
        for (size_t j = 0; j < top; ++j) {
            if (!in(j)) continue;
            const size_t v = (size_t) ids[t * top + j];
            const double logp = (z[t * top + j] - zm) / tau - std::log(zs), logq = (l[t * V + v] - m) / tau - std::log(st);
            out.loss += alpha * tau * tau * std::exp(logp) * (logp - logq) / (double) n;
            out.d[t * V + v] -= alpha * tau * std::exp(logp) / (double) n;
            out.mags[t * V + v] += alpha * tau * std::exp(logp) / (double) n;
        }
        const size_t y = (size_t) labels[t];
        out.loss += (1 - alpha) * (std::log(s1) + m - l[t * V + y]) / (double) n;
        out.d[t * V + y] -= (1 - alpha) / (double) n;
        out.mags[t * V + y] += (1 - alpha) / (double) n;
    }
    return out;
}

void step(Device* dev, size_t K, size_t D, size_t V, size_t T, float tau, float alpha) {
    std::printf("  %zu %zu %zu, %zu tokens, tau %g, alpha %g\n", K, D, V, T, (double) tau, (double) alpha);
    const size_t top = 20;
    Context* ctx = context_new(1 << 20);
    auto mat = [&](size_t a, size_t b, Type type = TYPE_F32) { return new_tensor_2d(ctx, type, (int64_t) a, (int64_t) b); };
    auto eight = [&](size_t k, size_t r, bool weight) { return hip_fp8_new(ctx, (int64_t) k, (int64_t) r, weight); };
    const HipFp8 w1 = eight(K, D, true), w2 = eight(D, V, true), xq = eight(K, T, false), hq = eight(D, T, false), dq = eight(V, T, false);
    Tensor *w1f = mat(K, D), *w2f = mat(D, V), *x = mat(K, T), *base = mat(D, T), *h = mat(D, T), *dh = mat(D, T), *dx = mat(D, T);
    Tensor *base2 = mat(V, T), *one = mat(V, 1), *dlogits = mat(V, T), *dloss = new_tensor_1d(ctx, TYPE_F32, 1);
    Tensor* h_one = view_2d(ctx, h, (int64_t) D, 1, (T - 1) * D * sizeof(float));
    HipDistillation d;
    d.logits = mat(V, T);
    d.labels = new_tensor_1d(ctx, TYPE_I32, (int64_t) T);
    d.ids = mat(top, T, TYPE_I32);
    d.teacher = mat(top, T);
    d.stats = mat(5, T);
    d.loss = new_tensor_1d(ctx, TYPE_F32, 4);
    d.tau = tau;
    d.alpha = alpha;
    Adapter first(ctx, K, D, T), second(ctx, D, V, T);
    Buffer* buffer = buffer_alloc_ctx_tensors(ctx, dev->default_buffer_type());

    set(w1f, wave(K * D, 0.71, 0.2));
    set(w2f, wave(D * V, 0.53, 0.3));
    set(x, wave(K * T, 0.97, 1.0));
    set(dloss, std::vector<float>{1.0f});
    first.fill(T);
    second.fill(T);
    std::vector<int32_t> labels(T), ids(top * T);
    std::vector<float> z(top * T);
    for (size_t t = 0; t < T; ++t) {
        labels[t] = t % 5 == 2 ? -1 : (int32_t) ((t * 37 + 11) % V);
        for (size_t j = 0; j < top; ++j) {
            ids[t * top + j] = j == 3 ? -1 : j == 7 ? (int32_t) V : j == 9 ? ids[t * top] : (int32_t) ((t * 37 + 11 + j * 13) % V);
            z[t * top + j] = 4.f - 0.3f * (float) j;
        }
    }
    set(d.labels, labels);
    set(d.ids, ids);
    set(d.teacher, z);

    hip_fp8_quantize(w1f, w1);
    hip_fp8_quantize(w2f, w2);
    hip_fp8_quantize(x, xq);
    hip_fp8_mul_mat(w1, xq, base);
    hip_lora(first.set, x, base, first.h, h);
    hip_fp8_quantize(h, hq);
    hip_fp8_mul_mat(w2, hq, base2);
    hip_fp8_matvec(w2, h_one, one);
    hip_lora(second.set, h, base2, second.h, d.logits);
    hip_distill_loss(d);
    hip_distill_loss_back(d, dloss, dlogits);
    hip_fp8_quantize(dlogits, dq);
    hip_fp8_mul_mat_back(w2, dq, dh);
    hip_lora_back(second.set, h, second.h, dlogits, second.g, dh, dx, second.da, second.db);
    hip_lora_back(first.set, x, first.h, dx, first.g, nullptr, nullptr, first.da, first.db);

    // the way forward
    const Doubles v1 = values(w1, true), v2 = values(w2, true), vx = values(xq, false), vh = values(hq, false), vd = values(dq, false);
    quantized(wide(get(w1f)), v1, K, D, true);
    quantized(wide(get(w2f)), v2, D, V, true);
    quantized(wide(get(x)), vx, K, T, false);
    quantized(wide(get(h)), vh, D, T, false);
    quantized(wide(get(dlogits)), vd, V, T, false);
    const Sum y1 = product(v1, vx, K, D, T, false), y2 = product(v2, vh, D, V, T, false);
    near(get(base), y1.v, y1.m, (double) K + 16, "W1 x");
    near(get(base2), y2.v, y2.m, (double) D + 16, "W2 h");
    const Doubles last(y2.v.end() - (long) V, y2.v.end()), last_m(y2.m.end() - (long) V, y2.m.end());
    near(get(one), last, last_m, (double) D + 16, "W2 h, one token");

    // the loss and its gradient
    const Doubles l = wide(get(d.logits));
    const Loss want = losses(d, l, V, T);
    const double spread = *std::max_element(l.begin(), l.end()) - *std::min_element(l.begin(), l.end());
    const double e_s = 2 * (spread / std::fmin(tau, 1.0) + 8 * std::sqrt((double) V) + 8) * U;
    const std::vector<float> loss = get(d.loss), dl = get(dlogits);
    EXPECT(std::fabs(loss[0] - want.loss) <= e_s * (alpha * tau * tau + 1 - alpha) + 2 * U * want.loss);
    double worst = 0;
    for (size_t i = 0; i < dl.size(); ++i) {
        // (the teacher's logits are within 6 of one another)
        const double bound = want.mags[i] * (2 * e_s + (6 / tau + 16 + (double) top) * U) + U * std::fabs(want.d[i]) + 1e-36;
        worst = std::fmax(worst, std::fabs(dl[i] - want.d[i]) / bound);
    }
    std::printf("    dlogits: %.3g of the bound\n", worst);
    EXPECT(worst <= 1);
    for (size_t t = 2; t < T; t += 5)
        for (size_t v = 0; v < V; ++v) EXPECT(dl[t * V + v] == 0.f);

    // the way back
    const Sum back = product(v2, vd, D, V, T, true);
    near(get(dh), back.v, back.m, (double) V + 16, "dh");
    const Doubles dhv = wide(get(dh));
    second.check(wide(get(h)), wide(dl), &dhv, dx, T, "beside W2");
    first.check(wide(get(x)), wide(get(dx)), nullptr, nullptr, T, "beside W1");

    // dB of the second adapter against differences of the loss in 64 bits along dB itself: logits are linear in B, so
    // (L(e) - L(-e)) / 2e is off by e^2 / 6 of the third derivative
    const Doubles hv = wide(get(second.h)), db = wide(get(second.db));
    double norm = 0;
    for (double g : db) norm += g * g;
    norm = std::sqrt(norm);
    auto moved = [&](double e) {
        Doubles lm = l;
        for (size_t t = 0; t < T; ++t)
            for (size_t v = 0; v < V; ++v)
                for (size_t r = 0; r < second.R; ++r) lm[t * V + v] += 1.5 * e * db[v * second.R + r] / norm * hv[t * second.R + r];
        return losses(d, lm, V, T).loss;
    };
    // e = 1e-3: logits move by less than 1e-3 * 1.5 |h| a token; a cumulant of third order of what moves by s is at most
    // s^3 a row, and s = 1.5 sqrt(8) max |h|; the rest is rounding in 64 bits and of dB in 32
    double hmax = 0;
    for (double v : hv) hmax = std::fmax(hmax, std::fabs(v));
    const double e = 1e-3, s = 1.5 * std::sqrt(8.0) * hmax, slope = (moved(e) - moved(-e)) / (2 * e);
    const double bound = e * e / 6 * 8 * s * s * s * (alpha / tau + 1 - alpha) + 1e-9 + 1e-4 * norm;
    std::printf("    slope %.6f, |dB| %.6f\n", slope, norm);
    EXPECT(std::fabs(slope - norm) <= bound);
    EXPECT(norm > 0);
    buffer_free(buffer);
    context_free(ctx);
}

}  // namespace

int main(int argc, char** argv) {
    if (argc > 1 && std::strcmp(argv[1], "--abort-host") == 0) {
        Context* ctx = context_new(1 << 16);
        Tensor* x = new_tensor_2d(ctx, TYPE_F32, 128, 2);
        hip_fp8_quantize(x, hip_fp8_new(ctx, 128, 2, false));  // aborts: in no HIP buffer
        return 0;
    }
    Device* dev = hip_device(0);
    if (dev == nullptr) {
        std::fprintf(stderr, "test_distillation: no HIP device\n");
        return 77;
    }
    step(dev, 200, 256, 1000, 50, 2.0f, 0.8f);
    step(dev, 130, 100, 333, 70, 1.5f, 0.3f);
    step(dev, 1, 1, 65, 3, 1.0f, 0.5f);
    step(dev, 256, 384, 4100, 8, 4.0f, 0.5f);
    std::printf("%s: %d failure(s)\n", g_failures == 0 ? "PASS" : "FAIL", g_failures);
    return g_failures == 0 ? 0 : 1;
}
