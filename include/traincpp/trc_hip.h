// Entry points of the MI355X HIP backend (libtraincpp_hip.so, or hip_device.cpp
// built into a traincpp tree). hip_device() is a new sibling of the reference's
// cpu_device()/vulkan_device() (src/core/trc_backends.h:14-22): it returns the
// Device of HIP ordinal `ordinal`, or nullptr when that GPU is not visible.
// Devices are process-lifetime singletons; register them with
// backend_register_device (include/traincpp/trc_backend.h:105) or the
// compile-time device list.
//
// The includes name the traincpp/ directory so that, built inside a traincpp
// tree, they resolve to that tree's own headers.
#pragma once

#include "traincpp/trc_backend.h"
#include "traincpp/trc_gguf.h"

#include <cstdint>

namespace traincpp {

Device* hip_device(int ordinal = 0);
int     hip_device_count();

// Warm-start load of one GGUF tensor in a legacy quant format (Q4_0, Q4_1,
// Q5_0, Q5_1, Q8_0) into a contiguous F32 tensor held in a HIP buffer, with the
// dequantization on the GPU (bit-identical to gguf_tensor_to_f32,
// src/io/trc_gguf.cpp:966-1049). Only the tensor's raw blocks cross PCIe (a
// quarter to a ninth of the F32 bytes); they are read by mmap straight from
// `path`, the file `f` was opened from, at the offsets the public reader
// reports (gguf_data_offset + GgufTensorInfo::offset). f may therefore be
// opened with load_data = false, so the data section is never read into host
// memory. Returns false, having done nothing, when the tensor is not a legacy
// quant type or dst is not such a tensor (use gguf_load_tensor then); prints
// an error and returns false when the name or the file is wrong; aborts on a
// device error.
bool hip_gguf_load_tensor(const char* path, const GgufFile* f, const char* name, Tensor* dst);

// Uploads n_blocks raw blocks of a legacy quant `type` from host memory and
// dequantizes them on the GPU straight into dst (a contiguous F32 tensor in a
// HIP buffer). Returns false, doing nothing, when dst is not in a HIP buffer;
// aborts on a device error. This is the call a reader that already holds the
// blocks makes: the quant branch of the reference's gguf_load_tensor
// (src/io/trc_gguf.cpp:1082-1088) can hand its blocks here instead of
// dequantizing on the host.
bool hip_dequant_into(Tensor* dst, Type type, const void* host_blocks, int64_t n_blocks);

// ---- tuning low-rank adapters on weights that stay as they were loaded ----
//
// These work on tensors in HIP buffers of one device, outside of graphs. They enqueue their work
// on the null stream, so they run in order with graph_compute, tensor_set and tensor_get, and need
// no synchronization between them. Tensors that are not in such buffers, wrong shapes and device
// errors abort, as a graph's do. trc_hip_abi.h (trc_hip_lora and the entries after it) has the formulas,
// the layouts and what may overlap.

// n adapters of one projection and the requests of one batch that use them.
struct HipLoraSet {
    Tensor* a = nullptr;        // [K, R, n] F32, F16 or BF16
    Tensor* b = nullptr;        // [R, M, n] of a's type
    Tensor* scale = nullptr;    // [n] F32
    Tensor* start = nullptr;    // [requests + 1] I32: request q holds tokens start[q] .. start[q+1] - 1
    Tensor* adapter = nullptr;  // [requests] I32: the request's adapter, < 0 for none
};

// h = A x [R, T], dst = base + scale B h [M, T]. base may be nullptr or dst.
void hip_lora(const HipLoraSet& set, const Tensor* x, const Tensor* base, Tensor* h, Tensor* dst);

// g = scale B^T dy [R, T], dx = base + A^T g [K, T] (dx may be nullptr), and the gradients of A and B (F32), added to
// where accumulate is set.
void hip_lora_back(const HipLoraSet& set, const Tensor* x, const Tensor* h, const Tensor* dy, Tensor* g,
                   const Tensor* base, Tensor* dx, Tensor* da, Tensor* db, bool accumulate = false);

// The preference loss of P pairs of sequences over logits [V, T].
struct HipPreference {
    Tensor* logits = nullptr;  // [V, T] F32, F16 or BF16
    Tensor* labels = nullptr;  // [T] I32, negative: not counted
    Tensor* start = nullptr;   // [2 P + 1] I32: pair i is sequences 2 i (chosen) and 2 i + 1 (rejected)
    Tensor* ref = nullptr;     // [2 P] F32: the reference model's log-probabilities of the sequences
    Tensor* lse = nullptr;     // [T] F32, written
    Tensor* logp = nullptr;    // [2 P] F32, written: the sequences' log-probabilities
    Tensor* slope = nullptr;   // [P] F32, written
    Tensor* loss = nullptr;    // [1] F32, written
    float beta = 0.1f;
    float smoothing = 0.0f;
};
void hip_preference_loss(const HipPreference& p);
// The logits' gradient for the loss's gradient dloss [1]; dlogits may be the logits themselves.
void hip_preference_loss_back(const HipPreference& p, const Tensor* dloss, Tensor* dlogits);

// One AdamW step over many tensors in one launch (the reference's AdamW, src/optim/trc_optim.cpp), its moments as floats
// or in 8 bits. The moments belong to the optimizer and start as zeros; the parameters (F32) and gradients
// (F32, F16 or BF16) are contiguous, keep their places and outlive it.
struct HipAdamWParams {
    double lr = 1e-3, beta1 = 0.9, beta2 = 0.999, eps = 1e-8, weight_decay = 0.01;
    double grad_scale = 1.0;  // every gradient is multiplied by it first
};
class HipAdamW {
public:
    // decay[i] (all 1 where it is nullptr) is the factor on tensor i's weight decay: 0 for biases and norms.
    HipAdamW(Tensor* const* params, Tensor* const* grads, size_t count, int bits = 32, const float* decay = nullptr);
    ~HipAdamW();
    HipAdamW(const HipAdamW&) = delete;
    HipAdamW& operator=(const HipAdamW&) = delete;
    void    step(const HipAdamWParams& p);
    int64_t steps() const;
    // Tensor i's moments as floats (either may be nullptr).
    void    moments(size_t i, float* m, float* v) const;
    // The moments as they are held, to be kept in a checkpoint and put back, bit for bit, into an optimizer over tensors
    // of the same sizes and bits.
    size_t  state_bytes() const;
    void    get_state(void* state) const;
    void    set_state(const void* state, int64_t steps);

private:
    struct State;
    State* s_;
};

}  // namespace traincpp
