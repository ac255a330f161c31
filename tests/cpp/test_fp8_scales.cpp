// An 8-bit weight whose scales are floats, as a checkpoint brings them, through include/traincpp/trc_hip.h: the same bits as from bytes
// where the floats are powers of two, and any floats against 64 bits.
//
// Tolerance, u = 2^-24: products of codes are exact, n of them added in 32 bits (n u of the sum of magnitudes at most),
// scaled (2 u), and a rounding for each block.
#include "traincpp/traincpp.h"

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

constexpr double U = 0x1p-24;

template <class T>
std::vector<T> get(const Tensor* t) {
    std::vector<T> v((size_t) tensor_nelements(t));
    tensor_get(t, v.data(), 0, v.size() * sizeof(T));
    return v;
}
std::vector<float> wave(size_t n, double f, double a) {
    std::vector<float> v(n);
    for (size_t i = 0; i < n; ++i) v[i] = (float) (a * std::sin(f * (double) (i + 1)) * std::cos(0.37 * f * (double) (i * i % 1013)));
    return v;
}
double e4m3(uint8_t c) {
    const int e = c >> 3 & 15, m = c & 7;
    const double v = e == 0 ? std::ldexp(m, -9) : std::ldexp(8 + m, e - 10);
    return c & 128 ? -v : v;
}
// the rows of a view of bytes, its gaps left out
std::vector<uint8_t> bytes(const Tensor* t) {
    const size_t n = (size_t) t->ne[0], rows = (size_t) t->ne[1], pitch = t->nb[1];
    std::vector<uint8_t> raw(pitch * (rows - 1) + n), v(n * rows);
    tensor_get(t, raw.data(), 0, raw.size());
    for (size_t r = 0; r < rows; ++r) std::memcpy(&v[r * n], &raw[r * pitch], n);
    return v;
}

void run(Device* dev, size_t K, size_t M, size_t T) {
    std::printf("  %zu x %zu, %zu tokens\n", K, M, T);
    Context* ctx = context_new(1 << 20);
    auto mat = [&](size_t a, size_t b) { return new_tensor_2d(ctx, TYPE_F32, (int64_t) a, (int64_t) b); };
    const HipFp8 w = hip_fp8_new(ctx, (int64_t) K, (int64_t) M, true), wf = hip_fp8_new(ctx, (int64_t) K, (int64_t) M, true, TYPE_F32);
    const HipFp8 xq = hip_fp8_new(ctx, (int64_t) K, (int64_t) T, false), gq = hip_fp8_new(ctx, (int64_t) M, (int64_t) T, false);
    Tensor *w32 = mat(K, M), *x = mat(K, T), *g = mat(M, T), *few = mat(K, 2);
    Tensor *y = mat(M, T), *dx = mat(K, T), *one = mat(M, 2), *yf = mat(M, T), *dxf = mat(K, T), *onef = mat(M, 2);
    Buffer* buffer = buffer_alloc_ctx_tensors(ctx, dev->default_buffer_type());
    auto set = [](Tensor* t, const auto& v) { tensor_set(t, v.data(), 0, v.size() * sizeof(v[0])); };
    set(w32, wave(K * M, 0.71, 0.2));
    set(x, wave(K * T, 0.97, 1.0));
    set(g, wave(M * T, 0.43, 1e-3));
    set(few, wave(K * 2, 0.59, 2.0));
    hip_fp8_quantize(w32, w);
    hip_fp8_quantize(x, xq);
    hip_fp8_quantize(g, gq);
    const std::vector<uint8_t> codes = bytes(w.q), exps = bytes(w.scale);
    // the same codes, row by row, and scales as floats
    for (size_t m = 0; m < M; ++m) tensor_set(wf.q, &codes[m * K], m * wf.q->nb[1], K);
    std::vector<float> scales(exps.size());
    for (size_t i = 0; i < exps.size(); ++i) scales[i] = std::ldexp(1.0f, exps[i] - 127);
    set(wf.scale, scales);
    EXPECT(wf.scale->type == TYPE_F32 && tensor_nelements(wf.scale) == (int64_t) scales.size());

    auto all = [&](const HipFp8& weight, Tensor* a, Tensor* b, Tensor* c) {
        hip_fp8_mul_mat(weight, xq, a);
        hip_fp8_mul_mat_back(weight, gq, b);
        hip_fp8_matvec(weight, few, c);
    };
    all(w, y, dx, one);
    all(wf, yf, dxf, onef);
    EXPECT(get<float>(y) == get<float>(yf) && get<float>(dx) == get<float>(dxf) && get<float>(one) == get<float>(onef));

    for (size_t i = 0; i < scales.size(); ++i) scales[i] *= 0.6f + 0.1f * (float) (i % 9);
    set(wf.scale, scales);
    all(wf, yf, dxf, onef);
    const size_t kb = (K + 127) / 128, mb = (M + 127) / 128;
    auto wv = [&](size_t m, size_t k) { return e4m3(codes[m * K + k]) * (double) scales[m / 128 * kb + k / 128]; };
    auto check = [&](const HipFp8& in, const Tensor* out, bool back) {
        const std::vector<uint8_t> q = bytes(in.q), s = bytes(in.scale);
        const std::vector<float> got = get<float>(out);
        const size_t n = back ? M : K, rows = back ? K : M, blocks = back ? mb : kb;
        double worst = 0;
        for (size_t t = 0; t < T; ++t)
            for (size_t r = 0; r < rows; ++r) {
                double want = 0, mag = 0;
                for (size_t i = 0; i < n; ++i) {
                    const double z = (back ? wv(i, r) : wv(r, i)) * e4m3(q[t * n + i]) * std::ldexp(1.0, s[t * blocks + i / 128] - 127);
                    want += z, mag += std::fabs(z);
                }
                worst = std::fmax(worst, std::fabs(got[t * rows + r] - want) / ((128.0 + (double) blocks + 16) * U * mag + 1e-38));
            }
        std::printf("    %s: %.3g of the bound\n", back ? "dx" : "y", worst);
        EXPECT(worst <= 1);
    };
    check(xq, yf, false);
    check(gq, dxf, true);
    buffer_free(buffer);
    context_free(ctx);
}

}  // namespace

int main(int argc, char** argv) {
    if (argc > 1 && std::strcmp(argv[1], "--abort-type") == 0) {
        hip_fp8_new(context_new(1 << 16), 128, 2, false, TYPE_F32);  // aborts: activations have bytes
        return 0;
    }
    Device* dev = hip_device(0);
    if (dev == nullptr) {
        std::fprintf(stderr, "test_fp8_scales: no HIP device\n");
        return 77;
    }
    run(dev, 200, 256, 50);
    run(dev, 300, 130, 90);
    run(dev, 1, 1, 3);
    run(dev, 640, 300, 70);
    std::printf("%s: %d failure(s)\n", g_failures == 0 ? "PASS" : "FAIL", g_failures);
    return g_failures == 0 ? 0 : 1;
}
