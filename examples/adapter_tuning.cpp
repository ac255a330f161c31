// Tunes low-rank adapters on a quantized weight to prefer chosen answers to rejected ones.
//
//   adapter_tuning [steps] [bits of the optimizer's moments: 8 or 32]
//
// A toy language model: fixed hidden states x of every answer's tokens, and one
// output projection whose Q4_0 weight W stays as it was loaded. Two adapters of rank 8
// learn beside it, one for each half of the pairs, in one batch. Each step:
//
//   base   = W x                                graph: mul_mat with the quantized weight (once: W and x stay)
//   logits = base + scale B (A x)               hip_lora, the requests' adapters side by side
//   loss, then its gradient by the logits       hip_preference_loss, hip_preference_loss_back
//   gradients of A and B                        hip_lora_back
//   A and B                                     HipAdamW::step
//
// The reference model is the same weights without an adapter: the answers' log-probabilities
// before the first step, with every request's adapter at -1. The loss starts at log 2 and falls as the
// adapters learn. Exits with 0 if it ends under a tenth of that, with every chosen answer ahead.
#include "traincpp/traincpp.h"

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
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
};

// IEEE half of a positive normal float in half's range, to nearest.
uint16_t half_of(float x) {
    uint32_t b;
    std::memcpy(&b, &x, 4);
    b += 0x1000 - (112u << 23);
    return (uint16_t) (b >> 13);
}

// Rows as Q4_0 blocks: 32 elements share d, the largest magnitude over 7, and are (q - 8) d; byte i of a
// block holds elements i and i + 16.
std::vector<uint8_t> quantize_q4_0(const std::vector<float>& w) {
    std::vector<uint8_t> out;
    for (size_t i = 0; i < w.size(); i += 32) {
        float top = 1e-4f;
        for (int k = 0; k < 32; ++k) top = std::fmax(top, std::fabs(w[i + k]));
        const float d = top / 7;
        const uint16_t h = half_of(d);
        out.push_back((uint8_t) h);
        out.push_back((uint8_t) (h >> 8));
        auto q = [&](int k) { return (int) std::fmin(15.f, std::fmax(0.f, std::round(w[i + k] / d) + 8)); };
        for (int k = 0; k < 16; ++k) out.push_back((uint8_t) (q(k) | q(k + 16) << 4));
    }
    return out;
}

template <class T>
void set(Tensor* t, const std::vector<T>& v) {
    tensor_set(t, v.data(), 0, v.size() * sizeof(T));
}
std::vector<float> get(const Tensor* t) {
    std::vector<float> v((size_t) tensor_nelements(t));
    tensor_get(t, v.data(), 0, v.size() * sizeof(float));
    return v;
}

}  // namespace

int main(int argc, char** argv) {
    const int steps = argc > 1 ? std::atoi(argv[1]) : 60, bits = argc > 2 ? std::atoi(argv[2]) : 8;
    if (steps < 1 || (bits != 8 && bits != 32)) {
        std::fprintf(stderr, "usage: adapter_tuning [steps] [8 or 32]\n");
        return 2;
    }
    Device* dev = hip_device(0);
    if (dev == nullptr) {
        std::fprintf(stderr, "adapter_tuning: no HIP device\n");
        return 2;
    }
    const int64_t K = 256, V = 1000, R = 8, adapters = 2, pairs = 6;
    Random rng{20240607};

    // answers of 5 to 16 tokens; the first two tokens of each stand for the prompt and are not counted
    std::vector<int32_t> start{0}, labels, adapter;
    for (int64_t s = 0; s < 2 * pairs; ++s) {
        const int n = 5 + (int) (rng.uniform() * 12);
        for (int t = 0; t < n; ++t) labels.push_back(t < 2 ? -1 : (int32_t) (rng.uniform() * (double) V));
        start.push_back(start.back() + n);
        adapter.push_back(s / 2 < pairs / 2 ? 0 : 1);
    }
    const int64_t T = start.back();

    Context* ctx = context_new(1 << 20);
    Tensor* w = new_tensor_2d(ctx, TYPE_Q4_0, K, V);
    Tensor* x = new_tensor_2d(ctx, TYPE_F32, K, T);
    Tensor* base = mul_mat(ctx, w, x);
    Graph* graph = graph_new(ctx);
    graph_build_forward_expand(ctx, graph, base);

    HipLoraSet set_;
    set_.a = new_tensor_3d(ctx, TYPE_F32, K, R, adapters);
    set_.b = new_tensor_3d(ctx, TYPE_F32, R, V, adapters);
    set_.scale = new_tensor_1d(ctx, TYPE_F32, adapters);
    set_.start = new_tensor_1d(ctx, TYPE_I32, 2 * pairs + 1);
    set_.adapter = new_tensor_1d(ctx, TYPE_I32, 2 * pairs);
    HipLoraSet none = set_;  // the same batch without adapters
    none.adapter = new_tensor_1d(ctx, TYPE_I32, 2 * pairs);
    Tensor* da = new_tensor_3d(ctx, TYPE_F32, K, R, adapters);
    Tensor* db = new_tensor_3d(ctx, TYPE_F32, R, V, adapters);
    Tensor* h = new_tensor_2d(ctx, TYPE_F32, R, T);
    Tensor* g = new_tensor_2d(ctx, TYPE_F32, R, T);
    HipPreference p;
    p.logits = new_tensor_2d(ctx, TYPE_F32, V, T);
    p.labels = new_tensor_1d(ctx, TYPE_I32, T);
    p.start = set_.start;
    p.ref = new_tensor_1d(ctx, TYPE_F32, 2 * pairs);
    p.lse = new_tensor_1d(ctx, TYPE_F32, T);
    p.logp = new_tensor_1d(ctx, TYPE_F32, 2 * pairs);
    p.slope = new_tensor_1d(ctx, TYPE_F32, pairs);
    p.loss = new_tensor_1d(ctx, TYPE_F32, 1);
    p.beta = 0.5f;
    Tensor* dloss = new_tensor_1d(ctx, TYPE_F32, 1);
    Buffer* buffer = buffer_alloc_ctx_tensors(ctx, dev->default_buffer_type());

    std::vector<float> wv((size_t) (K * V)), xv((size_t) (K * T)), av((size_t) (K * R * adapters));
    for (float& v : wv) v = rng.normal() * 0.06f;
    for (float& v : xv) v = rng.normal();
    for (float& v : av) v = rng.normal() / 16;
    set(w, quantize_q4_0(wv));
    set(x, xv);
    set(set_.a, av);  // (B starts as zeros, as a new buffer reads)
    set(set_.scale, std::vector<float>((size_t) adapters, 2.0f));
    set(set_.start, start);
    set(set_.adapter, adapter);
    set(none.adapter, std::vector<int32_t>((size_t) (2 * pairs), -1));
    set(p.labels, labels);
    set(dloss, std::vector<float>{1.0f});

    // the shared projection, and the reference model's log-probabilities
    dev->graph_compute(graph);
    hip_lora(none, x, base, h, p.logits);
    hip_preference_loss(p);
    set(p.ref, get(p.logp));

    Tensor* params[] = {set_.a, set_.b};
    Tensor* grads[] = {da, db};
    HipAdamW optimizer(params, grads, 2, bits);
    HipAdamWParams hyper;
    hyper.lr = 5e-3;
    hyper.weight_decay = 0.01;
    float first = 0, last = 0;
    for (int step = 0; step <= steps; ++step) {
        hip_lora(set_, x, base, h, p.logits);
        hip_preference_loss(p);
        last = get(p.loss)[0];
        if (step == 0) first = last;
        if (step % 10 == 0 || step == steps) std::printf("step %3d  loss %.6f\n", step, (double) last);
        if (step == steps) break;
        hip_preference_loss_back(p, dloss, p.logits);  // (the gradient takes the logits' place)
        hip_lora_back(set_, x, h, p.logits, g, nullptr, nullptr, da, db);
        optimizer.step(hyper);
    }

    const std::vector<float> logp = get(p.logp), ref = get(p.ref);
    int ahead = 0;
    for (int64_t i = 0; i < pairs; ++i) ahead += logp[2 * i] - ref[2 * i] > logp[2 * i + 1] - ref[2 * i + 1];
    const bool ok = std::fabs(first - std::log(2.0f)) < 1e-4f && last < 0.1f * first && ahead == pairs;
    std::printf("%s: loss %.4f to %.4f in %d steps, %d of %lld chosen answers ahead\n", ok ? "ok" : "FAILED", (double) first,
                (double) last, steps, ahead, (long long) pairs);
    buffer_free(buffer);
    graph_free(graph);
    context_free(ctx);
    return ok ? 0 : 1;
}
