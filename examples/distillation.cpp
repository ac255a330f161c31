// Tunes low-rank adapters beside weights in 8-bit floating point to answer as a teacher does.
//
//   distillation [steps]
//
// A toy language model of two layers, whose weights W1 and W2 are quantized once and stay so; an adapter of rank 8 learns
// beside each. Of the teacher, whose own output weights differ, only its 16 largest logits of every token are kept. Each
// step:
//
//   h      = W1 x + scale B1 (A1 x)             hip_fp8_mul_mat (x is quantized once), hip_lora
//   logits = W2 h + scale B2 (A2 h)             hip_fp8_quantize, hip_fp8_mul_mat, hip_lora
//   loss, then its gradient by the logits       hip_distill_loss, hip_distill_loss_back
//   gradient by h, and of A2 and B2             hip_fp8_quantize, hip_fp8_mul_mat_back, hip_lora_back
//   gradients of A1 and B1                      hip_lora_back
//   all adapters                                HipAdamW::step
//
// At the end one token alone goes through W2 by hip_fp8_matvec, which has to give what the batch gave it, but for the
// order of the sums.
#include "traincpp/traincpp.h"

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <numeric>
#include <vector>

using namespace traincpp;

namespace {

struct Random {
    uint64_t s;
    double uniform() {  // splitmix64
        uint64_t z = (s += 0x9E3779B97F4A7C15ull);
        z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
        z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
        return (double) ((z ^ (z >> 31)) >> 11) * 0x1p-53;
    }
    float normal() {
        const double u = 1.0 - uniform(), v = uniform();
        return (float) (std::sqrt(-2.0 * std::log(u)) * std::cos(6.283185307179586 * v));
    }
    std::vector<float> normals(int64_t n, float scale) {
        std::vector<float> v((size_t) n);
        for (float& x : v) x = normal() * scale;
        return v;
    }
};

template <class T>
void set(Tensor* t, const std::vector<T>& v) {
    tensor_set(t, v.data(), 0, v.size() * sizeof(T));
}
std::vector<float> get(const Tensor* t) {
    std::vector<float> v((size_t) tensor_nelements(t));
    tensor_get(t, v.data(), 0, v.size() * sizeof(float));
    return v;
}

// y = W x on the host, W [K, M], x [K, T]
std::vector<float> product(const std::vector<float>& w, const std::vector<float>& x, int64_t K, int64_t M, int64_t T) {
    std::vector<float> y((size_t) (M * T));
    for (int64_t t = 0; t < T; ++t)
        for (int64_t m = 0; m < M; ++m)
            y[(size_t) (t * M + m)] = std::inner_product(&w[(size_t) (m * K)], &w[(size_t) (m * K)] + K, &x[(size_t) (t * K)], 0.f);
    return y;
}

}  // namespace

int main(int argc, char** argv) {
    const int steps = argc > 1 ? std::atoi(argv[1]) : 60;
    if (steps < 1) {
        std::fprintf(stderr, "usage: distillation [steps]\n");
        return 2;
    }
    Device* dev = hip_device(0);
    if (dev == nullptr) {
        std::fprintf(stderr, "distillation: no HIP device\n");
        return 2;
    }
    const int64_t K = 200, D = 256, V = 1000, T = 50, R = 8, top = 16;
    Random rng{20240911};
    Context* ctx = context_new(1 << 20);

    const HipFp8 w1 = hip_fp8_new(ctx, K, D, true), w2 = hip_fp8_new(ctx, D, V, true);
    const HipFp8 xq = hip_fp8_new(ctx, K, T, false), hq = hip_fp8_new(ctx, D, T, false), dq = hip_fp8_new(ctx, V, T, false);
    Tensor* w1f = new_tensor_2d(ctx, TYPE_F32, K, D);  // (the weights as they were trained)
    Tensor* w2f = new_tensor_2d(ctx, TYPE_F32, D, V);
    Tensor* x = new_tensor_2d(ctx, TYPE_F32, K, T);
    Tensor* base = new_tensor_2d(ctx, TYPE_F32, D, T);
    Tensor* h = new_tensor_2d(ctx, TYPE_F32, D, T);
    Tensor* dh = new_tensor_2d(ctx, TYPE_F32, D, T);
    Tensor* dloss = new_tensor_1d(ctx, TYPE_F32, 1);
    HipDistillation d;
    d.logits = new_tensor_2d(ctx, TYPE_F32, V, T);
    d.labels = new_tensor_1d(ctx, TYPE_I32, T);
    d.ids = new_tensor_2d(ctx, TYPE_I32, top, T);
    d.teacher = new_tensor_2d(ctx, TYPE_F32, top, T);
    d.stats = new_tensor_2d(ctx, TYPE_F32, 5, T);
    d.loss = new_tensor_1d(ctx, TYPE_F32, 4);
    d.tau = 2.0f;
    d.alpha = 0.8f;

    struct Layer {
        HipLoraSet set;
        Tensor *da, *db, *h, *g;
    } one, two;
    auto adapter = [&](Layer& l, int64_t in, int64_t out) {
        l.set.a = new_tensor_3d(ctx, TYPE_F32, in, R, 1);
        l.set.b = new_tensor_3d(ctx, TYPE_F32, R, out, 1);
        l.set.scale = new_tensor_1d(ctx, TYPE_F32, 1);
        l.set.start = new_tensor_1d(ctx, TYPE_I32, 2);
        l.set.adapter = new_tensor_1d(ctx, TYPE_I32, 1);
        l.da = new_tensor_3d(ctx, TYPE_F32, in, R, 1);
        l.db = new_tensor_3d(ctx, TYPE_F32, R, out, 1);
        l.h = new_tensor_2d(ctx, TYPE_F32, R, T);
        l.g = new_tensor_2d(ctx, TYPE_F32, R, T);
    };
    adapter(one, K, D);
    adapter(two, D, V);
    // one token's way, beside the batch's
    Tensor* h_one = view_2d(ctx, h, D, 1, (size_t) ((T - 1) * D) * sizeof(float));
    Tensor* base_one = new_tensor_2d(ctx, TYPE_F32, V, 1);
    Buffer* buffer = buffer_alloc_ctx_tensors(ctx, dev->default_buffer_type());

    const std::vector<float> w1v = rng.normals(K * D, 0.07f), w2v = rng.normals(D * V, 0.1f), xv = rng.normals(K * T, 1.0f);
    set(w1f, w1v);
    set(w2f, w2v);
    set(x, xv);
    set(dloss, std::vector<float>{1.0f});
    for (Layer* l : {&one, &two}) {
        set(l->set.a, rng.normals(tensor_nelements(l->set.a), 0.06f));  // (B starts as zeros, as a new buffer reads)
        set(l->set.scale, std::vector<float>{2.0f});
        set(l->set.start, std::vector<int32_t>{0, (int32_t) T});
        set(l->set.adapter, std::vector<int32_t>{0});
    }

    // the teacher's answers: its largest logits, the largest of all as the label, and a few tokens (a prompt) not counted
    std::vector<float> w2t = w2v;
    for (float& v : w2t) v += rng.normal() * 0.1f;
    const std::vector<float> teacher = product(w2t, product(w1v, xv, K, D, T), D, V, T);
    std::vector<int32_t> ids((size_t) (top * T)), labels((size_t) T), order((size_t) V);
    std::vector<float> z((size_t) (top * T));
    for (int64_t t = 0; t < T; ++t) {
        const float* const l = &teacher[(size_t) (t * V)];
        std::iota(order.begin(), order.end(), 0);
        std::partial_sort(order.begin(), order.begin() + top, order.end(), [&](int32_t a, int32_t b) { return l[a] > l[b]; });
        for (int64_t j = 0; j < top; ++j) {
            ids[(size_t) (t * top + j)] = order[(size_t) j];
            z[(size_t) (t * top + j)] = l[order[(size_t) j]];
        }
        labels[(size_t) t] = t < 5 ? -1 : order[0];
    }
    set(d.ids, ids);
    set(d.teacher, z);
    set(d.labels, labels);

    hip_fp8_quantize(w1f, w1);
    hip_fp8_quantize(w2f, w2);
    hip_fp8_quantize(x, xq);
    hip_fp8_mul_mat(w1, xq, base);
    Tensor* params[] = {one.set.a, one.set.b, two.set.a, two.set.b};
    Tensor* grads[] = {one.da, one.db, two.da, two.db};
    HipAdamW optimizer(params, grads, 4, 32);
    HipAdamWParams hyper;
    hyper.lr = 5e-3;
    auto forward = [&] {
        hip_lora(one.set, x, base, one.h, h);
        hip_fp8_quantize(h, hq);
        hip_fp8_mul_mat(w2, hq, d.logits);
    };
    for (int step = 0; step <= steps; ++step) {
        forward();
        hip_lora(two.set, h, d.logits, two.h, d.logits);
        hip_distill_loss(d);
        if (step % 10 == 0 || step == steps) {
            const std::vector<float> loss = get(d.loss);
            std::printf("step %3d  loss %.6f  KL %.6f  cross-entropy %.6f\n", step, (double) loss[0], (double) loss[1], (double) loss[2]);
        }
        if (step == steps) break;
        hip_distill_loss_back(d, dloss, d.logits);  // (the gradient takes the logits' place)
        hip_fp8_quantize(d.logits, dq);
        hip_fp8_mul_mat_back(w2, dq, dh);
        hip_lora_back(two.set, h, two.h, d.logits, two.g, dh, dh, two.da, two.db);
        hip_lora_back(one.set, x, one.h, dh, one.g, nullptr, nullptr, one.da, one.db);
        optimizer.step(hyper);
    }

    forward();
    hip_fp8_matvec(w2, h_one, base_one);
    const std::vector<float> all = get(d.logits), single = get(base_one);
    float worst = 0, largest = 0;
    for (int64_t v = 0; v < V; ++v) {
        worst = std::fmax(worst, std::fabs(single[(size_t) v] - all[(size_t) ((T - 1) * V + v)]));
        largest = std::fmax(largest, std::fabs(single[(size_t) v]));
    }
    // (both quantize the token alike and multiply exactly, and add D terms in 32 bits in some order)
    const bool ok = std::isfinite(get(d.loss)[0]) && worst <= 1e-4f * largest;
    std::printf("%s: one token alone differs by %.2g of %.2g\n", ok ? "ok" : "FAILED", (double) worst, (double) largest);
    buffer_free(buffer);
    context_free(ctx);
    return ok ? 0 : 1;
}
