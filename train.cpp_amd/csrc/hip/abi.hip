// extern "C" entry points of libtrc_hip.so (declared in include/trc_hip_abi.h):
// argument validation, error reporting and the HIP runtime calls. Kernels live
// in dequant.hip, qmatvec.hip, qmm.hip, mul_mat.hip, elementwise.hip, copy.hip, lora.hip,
// preference.hip, adamw.hip, fp8.hip, fp8_mm.hip and distill.hip.
#include "common.h"
#include "fp8.h"

#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <new>

namespace trc_hip {

namespace {
thread_local char g_last_error[512] = "";

// TRC_HIP_FORCE_ERROR=<entry> makes that entry point fail before any device work.
bool forced(const char* entry) {
    const char* v = std::getenv("TRC_HIP_FORCE_ERROR");
    return v != nullptr && std::strcmp(v, entry) == 0;
}

bool is_quant(int type) {
    return block_bytes(type) != 0;
}

size_t basic_type_size(int type) {
    switch (type) {
        case 0: return 4;   // F32
        case 1: return 2;   // F16
        case 24: return 1;  // I8
        case 25: return 2;  // I16
        case 26: return 4;  // I32
        case 27: return 8;  // I64
        case 28: return 8;  // F64
        case 30: return 2;  // BF16
        default: return 0;
    }
}
}  // namespace

int hip_error(hipError_t e, const char* what) {
    if (e == hipSuccess) return TRC_HIP_OK;
    std::snprintf(g_last_error, sizeof(g_last_error), "%s: %s (hipError_t %d)", what,
                  hipGetErrorString(e), (int) e);
    // The runtime also keeps the failure as its "last error"; clear it so that
    // the launch check of a later kernel does not report this stale error.
    (void) hipGetLastError();
    return (int) e;
}

int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
    va_end(ap);
    return code;
}

int check_launch(const char* what) {
    return hip_error(hipGetLastError(), what);
}

int device_cus() {
    constexpr int MAX_DEV = 64;
    static int cached[MAX_DEV] = {};  // 0 = not queried yet; a benign race stores the same value
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0) dev = 0;
    if (dev < MAX_DEV && cached[dev] > 0) return cached[dev];
    int cus = 0;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) cus = 256;
    if (dev < MAX_DEV) cached[dev] = cus;
    return cus;
}

}  // namespace trc_hip

using namespace trc_hip;

#define TRC_FORCED(name)                                                               \
    do {                                                                               \
        if (forced(name)) return fail(TRC_HIP_E_FORCED, "%s: forced failure (TRC_HIP_FORCE_ERROR)", name); \
    } while (0)

extern "C" {

const char* trc_hip_last_error(void) {
    return g_last_error;
}

int trc_hip_device_count(int* count) {
    if (count == nullptr) return fail(TRC_HIP_E_INVALID, "trc_hip_device_count: count is NULL");
    *count = 0;
    TRC_FORCED("trc_hip_device_count");
    int n = 0;
    const hipError_t e = hipGetDeviceCount(&n);
    if (e == hipErrorNoDevice) return TRC_HIP_OK;
    if (e != hipSuccess) return hip_error(e, "hipGetDeviceCount");
    *count = n;
    return TRC_HIP_OK;
}

int trc_hip_init(int ordinal, trc_hip_props* props) {
    TRC_FORCED("trc_hip_init");
    int n = 0;
    if (hipGetDeviceCount(&n) != hipSuccess || n == 0) {
        (void) hipGetLastError();
        return fail(TRC_HIP_E_NO_DEVICE, "trc_hip_init: no HIP device is visible");
    }
    if (ordinal < 0 || ordinal >= n) {
        return fail(TRC_HIP_E_NO_DEVICE, "trc_hip_init: ordinal %d out of range (%d devices)", ordinal, n);
    }
    int st = hip_error(hipSetDevice(ordinal), "hipSetDevice");
    if (st != TRC_HIP_OK) return st;
    // the address of trc_hip_qmatvec_noalloc's fixed workspace on this device
    st = qm_scratch_setup();
    if (st != TRC_HIP_OK) return st;
    if (props == nullptr) return TRC_HIP_OK;
    hipDeviceProp_t p;
    st = hip_error(hipGetDeviceProperties(&p, ordinal), "hipGetDeviceProperties");
    if (st != TRC_HIP_OK) return st;
    std::memset(props, 0, sizeof(*props));
    std::snprintf(props->name, sizeof(props->name), "%s", p.name[0] ? p.name : "AMD GPU");
    std::snprintf(props->arch, sizeof(props->arch), "%s", p.gcnArchName);
    props->ordinal = ordinal;
    props->compute_units = p.multiProcessorCount;
    size_t free_b = 0, total_b = 0;
    st = hip_error(hipMemGetInfo(&free_b, &total_b), "hipMemGetInfo");
    if (st != TRC_HIP_OK) return st;
    props->memory_free = free_b;
    props->memory_total = total_b;
    props->unified_memory = p.integrated ? 1 : 0;
    props->abi_version = TRC_HIP_ABI_VERSION;
    return TRC_HIP_OK;
}

int trc_hip_sync(void* stream) {
    TRC_FORCED("trc_hip_sync");
    return hip_error(hipStreamSynchronize((hipStream_t) stream), "hipStreamSynchronize");
}

int trc_hip_malloc(void** ptr, size_t bytes) {
    if (ptr == nullptr) return fail(TRC_HIP_E_INVALID, "trc_hip_malloc: ptr is NULL");
    *ptr = nullptr;
    TRC_FORCED("trc_hip_malloc");
    if (bytes == 0) return TRC_HIP_OK;
    return hip_error(hipMalloc(ptr, bytes), "hipMalloc");
}

int trc_hip_free(void* ptr) {
    TRC_FORCED("trc_hip_free");
    if (ptr == nullptr) return TRC_HIP_OK;
    return hip_error(hipFree(ptr), "hipFree");
}

int trc_hip_h2d(void* dst, const void* src, size_t bytes, void* stream) {
    TRC_FORCED("trc_hip_h2d");
    if (bytes == 0) return TRC_HIP_OK;
    if (dst == nullptr || src == nullptr) return fail(TRC_HIP_E_INVALID, "trc_hip_h2d: NULL pointer");
    int st = hip_error(hipMemcpyAsync(dst, src, bytes, hipMemcpyHostToDevice, (hipStream_t) stream),
                       "hipMemcpyAsync(H2D)");
    if (st != TRC_HIP_OK) return st;
    return hip_error(hipStreamSynchronize((hipStream_t) stream), "hipStreamSynchronize(H2D)");
}

int trc_hip_d2h(void* dst, const void* src, size_t bytes, void* stream) {
    TRC_FORCED("trc_hip_d2h");
    if (bytes == 0) return TRC_HIP_OK;
    if (dst == nullptr || src == nullptr) return fail(TRC_HIP_E_INVALID, "trc_hip_d2h: NULL pointer");
    int st = hip_error(hipMemcpyAsync(dst, src, bytes, hipMemcpyDeviceToHost, (hipStream_t) stream),
                       "hipMemcpyAsync(D2H)");
    if (st != TRC_HIP_OK) return st;
    return hip_error(hipStreamSynchronize((hipStream_t) stream), "hipStreamSynchronize(D2H)");
}

int trc_hip_memset(void* dst, int value, size_t bytes, void* stream) {
    TRC_FORCED("trc_hip_memset");
    if (bytes == 0) return TRC_HIP_OK;
    if (dst == nullptr) return fail(TRC_HIP_E_INVALID, "trc_hip_memset: NULL pointer");
    return hip_error(hipMemsetAsync(dst, value, bytes, (hipStream_t) stream), "hipMemsetAsync");
}

int trc_hip_fill_f32(float* dst, float value, int64_t count, void* stream) {
    TRC_FORCED("trc_hip_fill_f32");
    if (count < 0) return fail(TRC_HIP_E_INVALID, "trc_hip_fill_f32: negative count");
    if (count == 0) return TRC_HIP_OK;
    if (dst == nullptr || ((uintptr_t) dst & 3u) != 0) {
        return fail(TRC_HIP_E_INVALID, "trc_hip_fill_f32: dst must be a non-NULL 4-byte aligned pointer");
    }
    return launch_fill_f32(dst, value, count, (hipStream_t) stream);
}

int trc_hip_dequant(int type, const void* blocks, int64_t n_blocks, float* dst, void* stream) {
    TRC_FORCED("trc_hip_dequant");
    if (!is_quant(type)) return fail(TRC_HIP_E_INVALID, "trc_hip_dequant: type %d is not Q4_0/Q4_1/Q5_0/Q5_1/Q8_0", type);
    if (n_blocks < 0) return fail(TRC_HIP_E_INVALID, "trc_hip_dequant: negative block count");
    if (n_blocks > 0 && (blocks == nullptr || dst == nullptr)) {
        return fail(TRC_HIP_E_INVALID, "trc_hip_dequant: NULL pointer");
    }
    return launch_dequant(type, blocks, n_blocks, dst, (hipStream_t) stream);
}

}  // extern "C"

namespace {

// The argument rules of both mul_mat entries; `who` names the entry in messages.
int check_mul_mat_args(const char* who, const trc_hip_tensor* a, const trc_hip_tensor* b, const trc_hip_tensor* dst) {
    if (a == nullptr || b == nullptr || dst == nullptr) {
        return fail(TRC_HIP_E_INVALID, "%s: NULL tensor", who);
    }
    const trc_hip_tensor* ts[3] = {a, b, dst};
    for (const trc_hip_tensor* t : ts) {
        if (t->type != TRC_HIP_TYPE_F32) return fail(TRC_HIP_E_INVALID, "%s: tensors must be F32", who);
        for (int i = 0; i < 4; ++i) {
            if (t->ne[i] <= 0) return fail(TRC_HIP_E_SHAPE, "%s: ne[%d] = %lld", who, i, (long long) t->ne[i]);
            if (t->nb[i] % 4 != 0) return fail(TRC_HIP_E_ALIGN, "%s: nb[%d] = %zu is not a multiple of 4", who, i, t->nb[i]);
        }
        if (t->data == nullptr || ((uintptr_t) t->data & 3u) != 0) {
            return fail(TRC_HIP_E_ALIGN, "%s: data must be non-NULL and 4-byte aligned", who);
        }
    }
    // ggml_can_mul_mat (src/ops/trc_ops.cpp:369-375) and the output shape (:380).
    if (a->ne[0] != b->ne[0] || b->ne[2] % a->ne[2] != 0 || b->ne[3] % a->ne[3] != 0 ||
        dst->ne[0] != a->ne[1] || dst->ne[1] != b->ne[1] || dst->ne[2] != b->ne[2] || dst->ne[3] != b->ne[3]) {
        return fail(TRC_HIP_E_SHAPE,
                    "%s: shapes a[%lld,%lld,%lld,%lld] b[%lld,%lld,%lld,%lld] dst[%lld,%lld,%lld,%lld] "
                    "are not a mul_mat",
                    who, (long long) a->ne[0], (long long) a->ne[1], (long long) a->ne[2], (long long) a->ne[3],
                    (long long) b->ne[0], (long long) b->ne[1], (long long) b->ne[2], (long long) b->ne[3],
                    (long long) dst->ne[0], (long long) dst->ne[1], (long long) dst->ne[2], (long long) dst->ne[3]);
    }
    // dst may be cleared before the sums are added into it (and is read and
    // written while the operands are read), so it must not share bytes with an
    // operand (compared by the byte spans the views cover)
    auto span_end = [](const trc_hip_tensor* t) {
        uintptr_t e = (uintptr_t) t->data + 4;
        for (int i = 0; i < 4; ++i) e += (uintptr_t) (t->ne[i] - 1) * t->nb[i];
        return e;
    };
    for (const trc_hip_tensor* t : {a, b}) {
        if ((uintptr_t) dst->data < span_end(t) && (uintptr_t) t->data < span_end(dst)) {
            return fail(TRC_HIP_E_SHAPE, "%s: dst overlaps an operand", who);
        }
    }
    return TRC_HIP_OK;
}

}  // namespace

extern "C" {

int trc_hip_mul_mat_f32(const trc_hip_tensor* a, const trc_hip_tensor* b, const trc_hip_tensor* dst,
                        void* stream) {
    TRC_FORCED("trc_hip_mul_mat_f32");
    const int rc = check_mul_mat_args("trc_hip_mul_mat_f32", a, b, dst);
    if (rc != TRC_HIP_OK) return rc;
    return launch_mul_mat_f32(*a, *b, *dst, (hipStream_t) stream);
}

int trc_hip_mul_mat_acc_f32(const trc_hip_tensor* a, const trc_hip_tensor* b, const trc_hip_tensor* dst,
                            void* stream) {
    TRC_FORCED("trc_hip_mul_mat_acc_f32");
    const int rc = check_mul_mat_args("trc_hip_mul_mat_acc_f32", a, b, dst);
    if (rc != TRC_HIP_OK) return rc;
    // the kernels address one dst plane through 32-bit buffer offsets
    const uint64_t plane = (uint64_t) (dst->ne[0] - 1) * dst->nb[0] + (uint64_t) (dst->ne[1] - 1) * dst->nb[1] + 4;
    if (plane >= (1ull << 31)) {
        return fail(TRC_HIP_E_SHAPE, "trc_hip_mul_mat_acc_f32: a dst plane spans %llu bytes (2 GiB at most)",
                    (unsigned long long) plane);
    }
    return launch_mul_mat_f32(*a, *b, *dst, (hipStream_t) stream, true);
}

}  // extern "C"

namespace {

// Argument checks shared by trc_hip_qmatvec and trc_hip_qmatvec_noalloc.
int qmatvec_args(const char* entry, int type, const void* wq, int64_t K, int64_t M, size_t nb1_w, const float* x,
                 int64_t N, size_t nb1_x, const float* y, size_t nb1_y) {
    if (!is_quant(type)) return fail(TRC_HIP_E_INVALID, "%s: type %d is not a legacy quant type", entry, type);
    if (K <= 0 || M <= 0 || N <= 0 || K % QK != 0) {
        return fail(TRC_HIP_E_SHAPE, "%s: need K > 0, K %% 32 == 0, M > 0, N > 0 (K=%lld M=%lld N=%lld)", entry,
                    (long long) K, (long long) M, (long long) N);
    }
    if (N > TRC_HIP_QMATVEC_MAX_N) {
        return fail(TRC_HIP_E_SHAPE, "%s: N=%lld exceeds %d", entry, (long long) N, TRC_HIP_QMATVEC_MAX_N);
    }
    if (wq == nullptr || x == nullptr || y == nullptr) return fail(TRC_HIP_E_INVALID, "%s: NULL pointer", entry);
    const size_t row_bytes = (size_t) (K / QK) * (size_t) block_bytes(type);
    if (nb1_w < row_bytes && M > 1) return fail(TRC_HIP_E_SHAPE, "%s: nb1_w %zu < row size %zu", entry, nb1_w, row_bytes);
    if ((N > 1 && (nb1_x < (size_t) K * 4 || nb1_y < (size_t) M * 4))) {
        return fail(TRC_HIP_E_SHAPE, "%s: columns of x or y overlap", entry);
    }
    // y is written (and, for some shapes, cleared first) while W and x are read,
    // so it must share no byte with either (compared by the spans they cover)
    const uintptr_t w0 = (uintptr_t) wq, w1 = w0 + (uintptr_t) (M - 1) * nb1_w + row_bytes;
    const uintptr_t x0 = (uintptr_t) x, x1 = x0 + (uintptr_t) (N - 1) * nb1_x + (uintptr_t) K * 4;
    const uintptr_t y0 = (uintptr_t) y, y1 = y0 + (uintptr_t) (N - 1) * nb1_y + (uintptr_t) M * 4;
    if ((y0 < w1 && w0 < y1) || (y0 < x1 && x0 < y1)) {
        return fail(TRC_HIP_E_SHAPE, "%s: y overlaps W or x", entry);
    }
    return TRC_HIP_OK;
}

}  // namespace

extern "C" {

int trc_hip_qmatvec(int type, const void* wq, int64_t K, int64_t M, size_t nb1_w, const float* x, int64_t N,
                    size_t nb1_x, float* y, size_t nb1_y, void* stream) {
    TRC_FORCED("trc_hip_qmatvec");
    const int rc = qmatvec_args("trc_hip_qmatvec", type, wq, K, M, nb1_w, x, N, nb1_x, y, nb1_y);
    if (rc != TRC_HIP_OK) return rc;
    return launch_qmatvec(type, wq, K, M, nb1_w, x, N, nb1_x, y, nb1_y, (hipStream_t) stream, QmScratch::PER_STREAM);
}

int trc_hip_qmatvec_noalloc(int type, const void* wq, int64_t K, int64_t M, size_t nb1_w, const float* x, int64_t N,
                            size_t nb1_x, float* y, size_t nb1_y, void* stream) {
    TRC_FORCED("trc_hip_qmatvec_noalloc");
    const int rc = qmatvec_args("trc_hip_qmatvec_noalloc", type, wq, K, M, nb1_w, x, N, nb1_x, y, nb1_y);
    if (rc != TRC_HIP_OK) return rc;
    return launch_qmatvec(type, wq, K, M, nb1_w, x, N, nb1_x, y, nb1_y, (hipStream_t) stream, QmScratch::STATIC);
}

int trc_hip_qmatvec_release_stream(void* stream) {
    TRC_FORCED("trc_hip_qmatvec_release_stream");
    return qm_release_stream((hipStream_t) stream);
}

int trc_hip_cpy(const trc_hip_tensor* src, const trc_hip_tensor* dst, void* stream) {
    TRC_FORCED("trc_hip_cpy");
    if (src == nullptr || dst == nullptr) return fail(TRC_HIP_E_INVALID, "trc_hip_cpy: NULL tensor");
    if (src->type != dst->type) return fail(TRC_HIP_E_INVALID, "trc_hip_cpy: types differ (%d vs %d)", src->type, dst->type);
    const size_t es = basic_type_size(src->type);
    if (es == 0) return fail(TRC_HIP_E_INVALID, "trc_hip_cpy: type %d has no per-element size", src->type);
    for (int i = 0; i < 4; ++i) {
        if (src->ne[i] != dst->ne[i] || src->ne[i] <= 0) return fail(TRC_HIP_E_SHAPE, "trc_hip_cpy: shapes differ");
        if (src->nb[i] % es != 0 || dst->nb[i] % es != 0) return fail(TRC_HIP_E_ALIGN, "trc_hip_cpy: strides not element aligned");
    }
    if (src->data == nullptr || dst->data == nullptr) return fail(TRC_HIP_E_INVALID, "trc_hip_cpy: NULL data");
    if (((uintptr_t) src->data % es) != 0 || ((uintptr_t) dst->data % es) != 0) {
        return fail(TRC_HIP_E_ALIGN, "trc_hip_cpy: data not element aligned");
    }
    return launch_cpy(*src, *dst, es, (hipStream_t) stream);
}

int trc_hip_add_f32(const trc_hip_tensor* a, const trc_hip_tensor* b, const trc_hip_tensor* dst, void* stream) {
    TRC_FORCED("trc_hip_add_f32");
    if (a == nullptr || b == nullptr || dst == nullptr) return fail(TRC_HIP_E_INVALID, "trc_hip_add_f32: NULL tensor");
    if (a->data == nullptr || b->data == nullptr || dst->data == nullptr) {
        return fail(TRC_HIP_E_INVALID, "trc_hip_add_f32: NULL data");
    }
    return launch_add_f32(*a, *b, *dst, (hipStream_t) stream);
}

int trc_hip_mul_f32(const trc_hip_tensor* a, const trc_hip_tensor* b, const trc_hip_tensor* dst, void* stream) {
    TRC_FORCED("trc_hip_mul_f32");
    if (a == nullptr || b == nullptr || dst == nullptr) return fail(TRC_HIP_E_INVALID, "trc_hip_mul_f32: NULL tensor");
    if (a->data == nullptr || b->data == nullptr || dst->data == nullptr) {
        return fail(TRC_HIP_E_INVALID, "trc_hip_mul_f32: NULL data");
    }
    return launch_mul_f32(*a, *b, *dst, (hipStream_t) stream);
}

int trc_hip_repeat_f32(const trc_hip_tensor* a, const trc_hip_tensor* dst, void* stream) {
    TRC_FORCED("trc_hip_repeat_f32");
    if (a == nullptr || dst == nullptr) return fail(TRC_HIP_E_INVALID, "trc_hip_repeat_f32: NULL tensor");
    if (a->data == nullptr || dst->data == nullptr) return fail(TRC_HIP_E_INVALID, "trc_hip_repeat_f32: NULL data");
    return launch_repeat_f32(*a, *dst, (hipStream_t) stream);
}

int trc_hip_sqr_f32(const trc_hip_tensor* a, const trc_hip_tensor* dst, void* stream) {
    TRC_FORCED("trc_hip_sqr_f32");
    if (a == nullptr || dst == nullptr) return fail(TRC_HIP_E_INVALID, "trc_hip_sqr_f32: NULL tensor");
    if (a->data == nullptr || dst->data == nullptr) return fail(TRC_HIP_E_INVALID, "trc_hip_sqr_f32: NULL data");
    return launch_sqr_f32(*a, *dst, (hipStream_t) stream);
}

int trc_hip_scale_f32(const trc_hip_tensor* a, const trc_hip_tensor* dst, float s, void* stream) {
    TRC_FORCED("trc_hip_scale_f32");
    if (a == nullptr || dst == nullptr) return fail(TRC_HIP_E_INVALID, "trc_hip_scale_f32: NULL tensor");
    if (a->data == nullptr || dst->data == nullptr) return fail(TRC_HIP_E_INVALID, "trc_hip_scale_f32: NULL data");
    return launch_scale_f32(*a, *dst, s, (hipStream_t) stream);
}

int trc_hip_sum_f32(const trc_hip_tensor* a, const trc_hip_tensor* dst, void* stream) {
    TRC_FORCED("trc_hip_sum_f32");
    if (a == nullptr || dst == nullptr) return fail(TRC_HIP_E_INVALID, "trc_hip_sum_f32: NULL tensor");
    if (a->data == nullptr || dst->data == nullptr) return fail(TRC_HIP_E_INVALID, "trc_hip_sum_f32: NULL data");
    return launch_sum_f32(*a, *dst, (hipStream_t) stream);
}

int trc_hip_acc_f32(const trc_hip_tensor* a, const trc_hip_tensor* b, const trc_hip_tensor* dst, size_t nb1,
                    size_t nb2, size_t nb3, size_t offset, int inplace, void* stream) {
    TRC_FORCED("trc_hip_acc_f32");
    if (a == nullptr || b == nullptr || dst == nullptr) return fail(TRC_HIP_E_INVALID, "trc_hip_acc_f32: NULL tensor");
    if (a->data == nullptr || b->data == nullptr || dst->data == nullptr) {
        return fail(TRC_HIP_E_INVALID, "trc_hip_acc_f32: NULL data");
    }
    return launch_acc_f32(*a, *b, *dst, nb1, nb2, nb3, offset, inplace, (hipStream_t) stream);
}

int trc_hip_repeat_back_f32(const trc_hip_tensor* a, const trc_hip_tensor* dst, void* stream) {
    TRC_FORCED("trc_hip_repeat_back_f32");
    if (a == nullptr || dst == nullptr) return fail(TRC_HIP_E_INVALID, "trc_hip_repeat_back_f32: NULL tensor");
    if (a->data == nullptr || dst->data == nullptr) return fail(TRC_HIP_E_INVALID, "trc_hip_repeat_back_f32: NULL data");
    return launch_repeat_back_f32(*a, *dst, (hipStream_t) stream);
}

}  // extern "C"

namespace {

// The bytes a tensor covers, from its first element to its last.
struct Span {
    uintptr_t lo, hi;
};
Span span_of(const trc_hip_tensor& t) {
    Span s{(uintptr_t) t.data, (uintptr_t) t.data + basic_type_size(t.type)};
    for (int i = 0; i < 4; ++i) s.hi += (uintptr_t) (t.ne[i] - 1) * t.nb[i];
    return s;
}

// A tensor of `type` and shape ne0 x ne1 x ne2 x 1, its elements side by side along ne0;
// `apart`: its rows and planes do not overlap (it is written).
int check_shape(const char* who, const char* name, const trc_hip_tensor* t, int type, int64_t ne0, int64_t ne1, int64_t ne2,
                bool apart) {
    if (t == nullptr) return fail(TRC_HIP_E_INVALID, "%s: %s is NULL", who, name);
    const size_t es = basic_type_size(type);
    if (t->type != type) return fail(TRC_HIP_E_INVALID, "%s: %s has type %d, not %d", who, name, t->type, type);
    if (t->ne[0] != ne0 || t->ne[1] != ne1 || t->ne[2] != ne2 || t->ne[3] != 1) {
        return fail(TRC_HIP_E_SHAPE, "%s: %s is [%lld,%lld,%lld,%lld], not [%lld,%lld,%lld,1]", who, name,
                    (long long) t->ne[0], (long long) t->ne[1], (long long) t->ne[2], (long long) t->ne[3], (long long) ne0,
                    (long long) ne1, (long long) ne2);
    }
    if (t->data == nullptr || (uintptr_t) t->data % es != 0) {
        return fail(TRC_HIP_E_ALIGN, "%s: %s's data must be non-NULL and %zu-byte aligned", who, name, es);
    }
    if ((ne0 > 1 && t->nb[0] != es) || (ne1 > 1 && t->nb[1] % es != 0) || (ne2 > 1 && t->nb[2] % es != 0)) {
        return fail(TRC_HIP_E_ALIGN, "%s: %s's strides must be whole elements, and neighbours along ne[0]", who, name);
    }
    if (apart && ((ne1 > 1 && t->nb[1] < (size_t) ne0 * es) || (ne2 > 1 && t->nb[2] < (size_t) (ne1 - 1) * t->nb[1] + (size_t) ne0 * es))) {
        return fail(TRC_HIP_E_SHAPE, "%s: rows of %s overlap", who, name);
    }
    return TRC_HIP_OK;
}

// What is written may share no byte with another operand, unless they are the same view.
int check_apart(const char* who, const trc_hip_tensor* out, const char* name, const trc_hip_tensor* other,
                const char* other_name, bool same_is_fine) {
    if (out == nullptr || other == nullptr) return TRC_HIP_OK;
    const Span a = span_of(*out), b = span_of(*other);
    if (a.lo >= b.hi || b.lo >= a.hi) return TRC_HIP_OK;
    if (same_is_fine && out->data == other->data && (out->ne[1] == 1 || out->nb[1] == other->nb[1])) return TRC_HIP_OK;
    return fail(TRC_HIP_E_SHAPE, "%s: %s overlaps %s", who, name, other_name);
}

#define TRC_TRY(call)                             \
    do {                                          \
        const int trc_rc = (call);                \
        if (trc_rc != TRC_HIP_OK) return trc_rc;  \
    } while (0)

bool is_float(int type) {
    return type == TRC_HIP_TYPE_F32 || type == TRC_HIP_TYPE_F16 || type == TRC_HIP_TYPE_BF16;
}

// The rules that trc_hip_lora and trc_hip_lora_back share; T is the batch's tokens.
int check_lora_set(const char* who, const trc_hip_lora_set* set, int64_t T) {
    const trc_hip_tensor &a = set->a, &b = set->b;
    if (!is_float(a.type)) return fail(TRC_HIP_E_INVALID, "%s: type %d of a is not F32, F16 or BF16", who, a.type);
    const int64_t K = a.ne[0], R = a.ne[1], n = a.ne[2], M = b.ne[1], requests = set->adapter.ne[0];
    if (K <= 0 || M <= 0 || T <= 0 || n <= 0 || n > 65535 || requests <= 0 || R <= 0 || R > TRC_HIP_LORA_MAX_RANK ||
        requests > (1 << 30) || T > INT32_MAX || M > (1 << 24) || K > (1 << 24)) {
        return fail(TRC_HIP_E_SHAPE,
                    "%s: K = %lld, M = %lld, T = %lld, rank %lld (at most %d), %lld adapters, %lld requests", who,
                    (long long) K, (long long) M, (long long) T, (long long) R, TRC_HIP_LORA_MAX_RANK, (long long) n,
                    (long long) requests);
    }
    TRC_TRY(check_shape(who, "a", &a, a.type, K, R, n, false));
    TRC_TRY(check_shape(who, "b", &b, a.type, R, M, n, false));
    if ((R > 1 && a.nb[1] > ((size_t) 1 << 24)) || (M > 1 && b.nb[1] > ((size_t) 1 << 24))) {
        return fail(TRC_HIP_E_SHAPE, "%s: rows of a or b over 16 MiB apart", who);
    }
    TRC_TRY(check_shape(who, "scale", &set->scale, TRC_HIP_TYPE_F32, n, 1, 1, false));
    TRC_TRY(check_shape(who, "start", &set->start, TRC_HIP_TYPE_I32, requests + 1, 1, 1, false));
    return check_shape(who, "adapter", &set->adapter, TRC_HIP_TYPE_I32, requests, 1, 1, false);
}

int check_lora_out(const char* who, const trc_hip_lora_set* set, const trc_hip_tensor* out, const char* name) {
    TRC_TRY(check_apart(who, out, name, &set->a, "a", false));
    TRC_TRY(check_apart(who, out, name, &set->b, "b", false));
    TRC_TRY(check_apart(who, out, name, &set->scale, "scale", false));
    TRC_TRY(check_apart(who, out, name, &set->start, "start", false));
    return check_apart(who, out, name, &set->adapter, "adapter", false);
}

// The kernels address a tile's rows of an activation through 32-bit offsets.
int check_row_stride(const char* who, const char* name, const trc_hip_tensor* t) {
    if (t != nullptr && t->ne[1] > 1 && t->nb[1] > ((size_t) 1 << 27)) {
        return fail(TRC_HIP_E_SHAPE, "%s: rows of %s over 128 MiB apart", who, name);
    }
    return TRC_HIP_OK;
}

// A contiguous vector or matrix: rows back to back.
int check_packed(const char* who, const char* name, const trc_hip_tensor* t) {
    if (t->ne[1] > 1 && t->nb[1] != (size_t) t->ne[0] * basic_type_size(t->type)) {
        return fail(TRC_HIP_E_SHAPE, "%s: %s must be contiguous", who, name);
    }
    return TRC_HIP_OK;
}

// The rules that the preference loss and its gradient share.
int check_preference(const char* who, const trc_hip_tensor* logits, const trc_hip_tensor* labels,
                     const trc_hip_tensor* start, const trc_hip_tensor* lse, const trc_hip_tensor* slope, float beta) {
    if (logits == nullptr || slope == nullptr) return fail(TRC_HIP_E_INVALID, "%s: NULL tensor", who);
    if (!is_float(logits->type)) return fail(TRC_HIP_E_INVALID, "%s: type %d of logits is not F32, F16 or BF16", who, logits->type);
    const int64_t V = logits->ne[0], T = logits->ne[1], P = slope->ne[0];
    // (the kernels count a row's elements in 32 bits, and some thousands past its end)
    if (V <= 0 || V > (1 << 30) || T <= 0 || T > INT32_MAX || P <= 0 || P > INT32_MAX / 2) {
        return fail(TRC_HIP_E_SHAPE, "%s: V = %lld, T = %lld, %lld pairs", who, (long long) V, (long long) T, (long long) P);
    }
    if (!(beta == beta)) return fail(TRC_HIP_E_INVALID, "%s: beta is NaN", who);
    TRC_TRY(check_shape(who, "logits", logits, logits->type, V, T, 1, false));
    TRC_TRY(check_shape(who, "labels", labels, TRC_HIP_TYPE_I32, T, 1, 1, false));
    TRC_TRY(check_shape(who, "start", start, TRC_HIP_TYPE_I32, 2 * P + 1, 1, 1, false));
    TRC_TRY(check_shape(who, "lse", lse, TRC_HIP_TYPE_F32, T, 1, 1, false));
    return check_shape(who, "slope", slope, TRC_HIP_TYPE_F32, P, 1, 1, false);
}

}  // namespace

extern "C" {

int trc_hip_lora(const trc_hip_lora_set* set, const trc_hip_tensor* x, const trc_hip_tensor* base, const trc_hip_tensor* h,
                 const trc_hip_tensor* dst, void* stream) {
    const char* const who = "trc_hip_lora";
    TRC_FORCED("trc_hip_lora");
    if (set == nullptr || x == nullptr) return fail(TRC_HIP_E_INVALID, "%s: NULL argument", who);
    const int64_t K = set->a.ne[0], R = set->a.ne[1], M = set->b.ne[1], T = x->ne[1];
    TRC_TRY(check_lora_set(who, set, T));
    TRC_TRY(check_shape(who, "x", x, TRC_HIP_TYPE_F32, K, T, 1, false));
    TRC_TRY(check_shape(who, "h", h, TRC_HIP_TYPE_F32, R, T, 1, true));
    TRC_TRY(check_packed(who, "h", h));
    TRC_TRY(check_shape(who, "dst", dst, TRC_HIP_TYPE_F32, M, T, 1, true));
    if (base != nullptr) TRC_TRY(check_shape(who, "base", base, TRC_HIP_TYPE_F32, M, T, 1, false));
    TRC_TRY(check_row_stride(who, "x", x));
    TRC_TRY(check_row_stride(who, "base", base));
    TRC_TRY(check_row_stride(who, "dst", dst));
    TRC_TRY(check_lora_out(who, set, h, "h"));
    TRC_TRY(check_lora_out(who, set, dst, "dst"));
    TRC_TRY(check_apart(who, h, "h", x, "x", false));
    TRC_TRY(check_apart(who, h, "h", base, "base", false));
    TRC_TRY(check_apart(who, dst, "dst", x, "x", false));
    TRC_TRY(check_apart(who, dst, "dst", h, "h", false));
    TRC_TRY(check_apart(who, dst, "dst", base, "base", true));
    return launch_lora(*set, *x, base, *h, *dst, (hipStream_t) stream);
}

int trc_hip_lora_back(const trc_hip_lora_set* set, const trc_hip_tensor* x, const trc_hip_tensor* h, const trc_hip_tensor* dy,
                      const trc_hip_tensor* g, const trc_hip_tensor* base, const trc_hip_tensor* dx, const trc_hip_tensor* da,
                      const trc_hip_tensor* db, int accumulate, void* stream) {
    const char* const who = "trc_hip_lora_back";
    TRC_FORCED("trc_hip_lora_back");
    if (set == nullptr || x == nullptr) return fail(TRC_HIP_E_INVALID, "%s: NULL argument", who);
    const int64_t K = set->a.ne[0], R = set->a.ne[1], n = set->a.ne[2], M = set->b.ne[1], T = x->ne[1];
    TRC_TRY(check_lora_set(who, set, T));
    TRC_TRY(check_shape(who, "x", x, TRC_HIP_TYPE_F32, K, T, 1, false));
    TRC_TRY(check_shape(who, "h", h, TRC_HIP_TYPE_F32, R, T, 1, false));
    TRC_TRY(check_packed(who, "h", h));
    TRC_TRY(check_shape(who, "dy", dy, TRC_HIP_TYPE_F32, M, T, 1, false));
    TRC_TRY(check_shape(who, "g", g, TRC_HIP_TYPE_F32, R, T, 1, true));
    TRC_TRY(check_packed(who, "g", g));
    if (dx != nullptr) TRC_TRY(check_shape(who, "dx", dx, TRC_HIP_TYPE_F32, K, T, 1, true));
    if (base != nullptr) {
        if (dx == nullptr) return fail(TRC_HIP_E_INVALID, "%s: base without dx", who);
        TRC_TRY(check_shape(who, "base", base, TRC_HIP_TYPE_F32, K, T, 1, false));
    }
    TRC_TRY(check_shape(who, "da", da, TRC_HIP_TYPE_F32, K, R, n, true));
    TRC_TRY(check_shape(who, "db", db, TRC_HIP_TYPE_F32, R, M, n, true));
    TRC_TRY(check_row_stride(who, "x", x));
    TRC_TRY(check_row_stride(who, "dy", dy));
    TRC_TRY(check_row_stride(who, "base", base));
    TRC_TRY(check_row_stride(who, "dx", dx));
    const trc_hip_tensor* const outs[4] = {g, dx, da, db};
    const char* const names[4] = {"g", "dx", "da", "db"};
    for (int i = 0; i < 4; ++i) {
        if (outs[i] == nullptr) continue;
        TRC_TRY(check_lora_out(who, set, outs[i], names[i]));
        TRC_TRY(check_apart(who, outs[i], names[i], x, "x", false));
        TRC_TRY(check_apart(who, outs[i], names[i], h, "h", false));
        TRC_TRY(check_apart(who, outs[i], names[i], dy, "dy", false));
        TRC_TRY(check_apart(who, outs[i], names[i], base, "base", outs[i] == dx));
        for (int j = i + 1; j < 4; ++j) TRC_TRY(check_apart(who, outs[i], names[i], outs[j], names[j], false));
    }
    return launch_lora_back(*set, *x, *h, *dy, *g, base, dx, *da, *db, accumulate != 0, (hipStream_t) stream);
}

int trc_hip_preference_loss(const trc_hip_tensor* logits, const trc_hip_tensor* labels, const trc_hip_tensor* start,
                            const trc_hip_tensor* ref, float beta, float smoothing, const trc_hip_tensor* lse,
                            const trc_hip_tensor* logp, const trc_hip_tensor* slope, const trc_hip_tensor* loss,
                            void* stream) {
    const char* const who = "trc_hip_preference_loss";
    TRC_FORCED("trc_hip_preference_loss");
    TRC_TRY(check_preference(who, logits, labels, start, lse, slope, beta));
    const int64_t P = slope->ne[0];
    if (!(smoothing >= 0.f && smoothing <= 1.f)) return fail(TRC_HIP_E_INVALID, "%s: smoothing %g is not in 0 .. 1", who, smoothing);
    TRC_TRY(check_shape(who, "ref", ref, TRC_HIP_TYPE_F32, 2 * P, 1, 1, false));
    TRC_TRY(check_shape(who, "logp", logp, TRC_HIP_TYPE_F32, 2 * P, 1, 1, false));
    TRC_TRY(check_shape(who, "loss", loss, TRC_HIP_TYPE_F32, 1, 1, 1, false));
    const trc_hip_tensor* const all[8] = {lse, logp, slope, loss, logits, labels, start, ref};
    const char* const names[8] = {"lse", "logp", "slope", "loss", "logits", "labels", "start", "ref"};
    for (int i = 0; i < 4; ++i) {
        for (int j = i + 1; j < 8; ++j) TRC_TRY(check_apart(who, all[i], names[i], all[j], names[j], false));
    }
    return launch_preference_loss(*logits, (const int32_t*) labels->data, (const int32_t*) start->data, P,
                                  (const float*) ref->data, beta, smoothing, (float*) lse->data, (float*) logp->data,
                                  (float*) slope->data, (float*) loss->data, (hipStream_t) stream);
}

int trc_hip_preference_loss_back(const trc_hip_tensor* logits, const trc_hip_tensor* labels, const trc_hip_tensor* start,
                                 const trc_hip_tensor* lse, const trc_hip_tensor* slope, const trc_hip_tensor* dloss,
                                 float beta, const trc_hip_tensor* dlogits, void* stream) {
    const char* const who = "trc_hip_preference_loss_back";
    TRC_FORCED("trc_hip_preference_loss_back");
    TRC_TRY(check_preference(who, logits, labels, start, lse, slope, beta));
    TRC_TRY(check_shape(who, "dloss", dloss, TRC_HIP_TYPE_F32, 1, 1, 1, false));
    TRC_TRY(check_shape(who, "dlogits", dlogits, logits->type, logits->ne[0], logits->ne[1], 1, true));
    const trc_hip_tensor* const all[6] = {logits, labels, start, lse, slope, dloss};
    const char* const names[6] = {"logits", "labels", "start", "lse", "slope", "dloss"};
    for (int j = 0; j < 6; ++j) TRC_TRY(check_apart(who, dlogits, "dlogits", all[j], names[j], j == 0));
    return launch_preference_loss_back(*logits, (const int32_t*) labels->data, (const int32_t*) start->data, slope->ne[0],
                                       (const float*) lse->data, (const float*) slope->data, (const float*) dloss->data, beta,
                                       *dlogits, (hipStream_t) stream);
}

int trc_hip_adamw_create(const trc_hip_adamw_tensor* tensors, int64_t count, int bits, void** plan) {
    const char* const who = "trc_hip_adamw_create";
    if (plan == nullptr) return fail(TRC_HIP_E_INVALID, "%s: plan is NULL", who);
    *plan = nullptr;
    TRC_FORCED("trc_hip_adamw_create");
    if (count < 0 || (count > 0 && tensors == nullptr)) return fail(TRC_HIP_E_INVALID, "%s: no tensors", who);
    if (bits != 32 && bits != 8) return fail(TRC_HIP_E_INVALID, "%s: moments of %d bits (32 or 8)", who, bits);
    try {
        return adamw_create(tensors, count, bits, plan);
    } catch (const std::bad_alloc&) {
        return fail((int) hipErrorOutOfMemory, "%s: out of host memory", who);
    }
}

int trc_hip_adamw_step(void* plan, const trc_hip_adamw_hyper* hyper, void* stream) {
    const char* const who = "trc_hip_adamw_step";
    TRC_FORCED("trc_hip_adamw_step");
    if (plan == nullptr || hyper == nullptr) return fail(TRC_HIP_E_INVALID, "%s: NULL argument", who);
    if (hyper->step < 1) return fail(TRC_HIP_E_INVALID, "%s: step %lld (they count from 1)", who, (long long) hyper->step);
    if (!(hyper->beta1 >= 0.0 && hyper->beta1 < 1.0) || !(hyper->beta2 >= 0.0 && hyper->beta2 < 1.0) || !(hyper->eps >= 0.0)) {
        return fail(TRC_HIP_E_INVALID, "%s: beta1 = %g, beta2 = %g, eps = %g", who, hyper->beta1, hyper->beta2, hyper->eps);
    }
    return adamw_step(plan, *hyper, (hipStream_t) stream);
}

int trc_hip_adamw_moments(void* plan, void* stream) {
    TRC_FORCED("trc_hip_adamw_moments");
    if (plan == nullptr) return fail(TRC_HIP_E_INVALID, "trc_hip_adamw_moments: plan is NULL");
    return adamw_moments(plan, (hipStream_t) stream);
}

int trc_hip_adamw_destroy(void* plan) {
    TRC_FORCED("trc_hip_adamw_destroy");
    return plan != nullptr ? adamw_destroy(plan) : TRC_HIP_OK;
}

}  // extern "C"

namespace {

// A matrix in 8-bit floating point and what is read of it: whole blocks of its rows, whole words of its rows of bytes
// of scales. per_row: its scales are its rows'; else those of 128 rows each.
int check_fp8(const char* who, const char* name, const trc_hip_fp8* m, int64_t K, int64_t R, bool per_row) {
    const trc_hip_tensor &q = m->q, &s = m->scale;
    const int64_t kb = (K + 127) / 128, groups = per_row ? R : (R + 127) / 128;
    TRC_TRY(check_shape(who, name, &q, TRC_HIP_TYPE_I8, K, R, 1, false));
    if ((uintptr_t) q.data % 16 != 0 || q.nb[1] % 128 != 0) {
        return fail(TRC_HIP_E_ALIGN, "%s: codes of %s must be 16-byte aligned, rows whole blocks of 128 bytes", who, name);
    }
    if (q.nb[1] < (size_t) kb * 128 || q.nb[1] > ((size_t) 1 << 23)) {
        return fail(TRC_HIP_E_SHAPE, "%s: rows of %s are %zu bytes apart (whole blocks, 8 MiB at most)", who, name, q.nb[1]);
    }
    if (s.type != TRC_HIP_TYPE_I8 && (per_row || s.type != TRC_HIP_TYPE_F32)) {
        return fail(TRC_HIP_E_INVALID, "%s: type %d of %s's scales", who, s.type, name);
    }
    TRC_TRY(check_shape(who, name, &s, s.type, kb, groups, 1, true));
    if ((uintptr_t) s.data % 4 != 0 || (groups > 1 && s.nb[1] % 4 != 0)) {
        return fail(TRC_HIP_E_ALIGN, "%s: scales of %s must be 4-byte aligned, their rows too", who, name);
    }
    // (a row of bytes has room for whole words, since rows are whole words apart and do not overlap)
    if (groups > 1 && s.nb[1] > ((size_t) 1 << 22)) {
        return fail(TRC_HIP_E_SHAPE, "%s: scales of %s's rows over 4 MiB apart", who, name);
    }
    return TRC_HIP_OK;
}

// What a matrix in 8 bits covers, whole blocks and words included, as contiguous bytes.
trc_hip_tensor bytes_of(const trc_hip_tensor& t, int64_t whole) {
    const int64_t es = (int64_t) basic_type_size(t.type), row = (t.ne[0] * es + whole - 1) / whole * whole;
    const int64_t n = (t.ne[1] - 1) * (int64_t) t.nb[1] + row;
    trc_hip_tensor b{};
    b.data = t.data;
    b.type = TRC_HIP_TYPE_I8;
    b.ne[0] = n;
    b.ne[1] = b.ne[2] = b.ne[3] = 1;
    b.nb[0] = 1;
    return b;
}
int check_fp8_apart(const char* who, const trc_hip_tensor* out, const char* name, const trc_hip_fp8* m, const char* other) {
    const trc_hip_tensor q = bytes_of(m->q, 128), s = bytes_of(m->scale, 4);
    TRC_TRY(check_apart(who, out, name, &q, other, false));
    return check_apart(who, out, name, &s, other, false);
}

// The sizes that the kernels' 32-bit offsets and counts allow for.
int check_fp8_sizes(const char* who, int64_t K, int64_t M, int64_t N) {
    if (K <= 0 || M <= 0 || N <= 0 || K > (1 << 23) || M > (1 << 23) || N > (1 << 23)) {
        return fail(TRC_HIP_E_SHAPE, "%s: K = %lld, M = %lld, N = %lld (1 to 2^23 each)", who, (long long) K, (long long) M, (long long) N);
    }
    return TRC_HIP_OK;
}

// y, rows x N in any float type, apart from the weight; `in` are its columns.
int check_fp8_out(const char* who, const char* name, const trc_hip_tensor* y, int64_t rows, int64_t N, const trc_hip_fp8* w) {
    if (y == nullptr) return fail(TRC_HIP_E_INVALID, "%s: %s is NULL", who, name);
    if (!is_float(y->type)) return fail(TRC_HIP_E_INVALID, "%s: type %d of %s is not F32, F16 or BF16", who, y->type, name);
    TRC_TRY(check_shape(who, name, y, y->type, rows, N, 1, true));
    return check_fp8_apart(who, y, name, w, "w");
}

F8Args fp8_args(const trc_hip_fp8& w, const trc_hip_tensor& y, int64_t N) {
    F8Args a{};
    a.w = (const uint8_t*) w.q.data;
    a.w_nb1 = (int64_t) w.q.nb[1];
    a.K = w.q.ne[0];
    a.M = w.q.ne[1];
    a.N = N;
    a.ws = (const uint8_t*) w.scale.data;
    a.ws_nb1 = (int64_t) w.scale.nb[1];
    a.ws_float = w.scale.type == TRC_HIP_TYPE_F32;
    a.y = (uint8_t*) y.data;
    a.y_nb1 = (int64_t) y.nb[1];
    a.y_type = y.type;
    return a;
}

// The product and its gradient by x: back sums over w's rows.
int fp8_product(const char* who, const trc_hip_fp8* w, const trc_hip_fp8* x, const trc_hip_tensor* y, bool back, hipStream_t s) {
    if (w == nullptr || x == nullptr || y == nullptr) return fail(TRC_HIP_E_INVALID, "%s: NULL argument", who);
    const int64_t K = w->q.ne[0], M = w->q.ne[1], N = x->q.ne[1];
    const char *const xn = back ? "dy" : "x", *const yn = back ? "dx" : "y";
    TRC_TRY(check_fp8_sizes(who, K, M, N));
    TRC_TRY(check_fp8(who, "w", w, K, M, false));
    TRC_TRY(check_fp8(who, xn, x, back ? M : K, N, true));
    TRC_TRY(check_fp8_out(who, yn, y, back ? K : M, N, w));
    TRC_TRY(check_fp8_apart(who, y, yn, x, xn));
    F8Args a = fp8_args(*w, *y, N);
    a.x = (const uint8_t*) x->q.data;
    a.x_nb1 = (int64_t) x->q.nb[1];
    a.xs = (const uint8_t*) x->scale.data;
    a.xs_nb1 = (int64_t) x->scale.nb[1];
    return launch_f8_product(a, back, s);
}

}  // namespace

extern "C" {

int trc_hip_fp8_quantize(const trc_hip_tensor* x, const trc_hip_fp8* out, void* stream) {
    const char* const who = "trc_hip_fp8_quantize";
    TRC_FORCED("trc_hip_fp8_quantize");
    if (x == nullptr || out == nullptr) return fail(TRC_HIP_E_INVALID, "%s: NULL argument", who);
    if (!is_float(x->type)) return fail(TRC_HIP_E_INVALID, "%s: type %d of x is not F32, F16 or BF16", who, x->type);
    const int64_t K = x->ne[0], R = x->ne[1];
    TRC_TRY(check_fp8_sizes(who, K, R, 1));
    TRC_TRY(check_shape(who, "x", x, x->type, K, R, 1, false));
    TRC_TRY(check_fp8(who, "out", out, K, R, out->scale.ne[1] == R));
    if (out->scale.type != TRC_HIP_TYPE_I8) return fail(TRC_HIP_E_INVALID, "%s: the scales must be I8", who);
    // (a workgroup of 256 for each 128 x 128, or for four pieces of 512 of a row)
    if ((out->scale.ne[1] == R ? R * ((K + 511) / 512) / 4 : ((R + 127) / 128) * ((K + 127) / 128)) >= max_groups(256)) {
        return fail(TRC_HIP_E_SHAPE, "%s: %lld rows of %lld", who, (long long) R, (long long) K);
    }
    const trc_hip_tensor q = bytes_of(out->q, 128), s = bytes_of(out->scale, 4);
    TRC_TRY(check_apart(who, &q, "out", x, "x", false));
    TRC_TRY(check_apart(who, &s, "out's scale", x, "x", false));
    TRC_TRY(check_apart(who, &q, "out", &s, "its scale", false));
    return launch_f8_quantize(*x, *out, (hipStream_t) stream);
}

int trc_hip_fp8_mul_mat(const trc_hip_fp8* w, const trc_hip_fp8* x, const trc_hip_tensor* y, void* stream) {
    TRC_FORCED("trc_hip_fp8_mul_mat");
    return fp8_product("trc_hip_fp8_mul_mat", w, x, y, false, (hipStream_t) stream);
}

int trc_hip_fp8_mul_mat_back(const trc_hip_fp8* w, const trc_hip_fp8* dy, const trc_hip_tensor* dx, void* stream) {
    TRC_FORCED("trc_hip_fp8_mul_mat_back");
    return fp8_product("trc_hip_fp8_mul_mat_back", w, dy, dx, true, (hipStream_t) stream);
}

int trc_hip_fp8_matvec(const trc_hip_fp8* w, const trc_hip_tensor* x, const trc_hip_tensor* y, void* stream) {
    const char* const who = "trc_hip_fp8_matvec";
    TRC_FORCED("trc_hip_fp8_matvec");
    if (w == nullptr || x == nullptr || y == nullptr) return fail(TRC_HIP_E_INVALID, "%s: NULL argument", who);
    const int64_t K = w->q.ne[0], M = w->q.ne[1], N = x->ne[1];
    TRC_TRY(check_fp8_sizes(who, K, M, N));
    if (N > TRC_HIP_FP8_MATVEC_MAX_N) {
        return fail(TRC_HIP_E_SHAPE, "%s: %lld tokens (at most %d)", who, (long long) N, TRC_HIP_FP8_MATVEC_MAX_N);
    }
    if (!is_float(x->type)) return fail(TRC_HIP_E_INVALID, "%s: type %d of x is not F32, F16 or BF16", who, x->type);
    TRC_TRY(check_fp8(who, "w", w, K, M, false));
    TRC_TRY(check_shape(who, "x", x, x->type, K, N, 1, false));
    TRC_TRY(check_fp8_out(who, "y", y, M, N, w));
    TRC_TRY(check_apart(who, y, "y", x, "x", false));
    return launch_f8_matvec(fp8_args(*w, *y, N), *x, (hipStream_t) stream);
}

}  // extern "C"

namespace {

// The rules that the distillation loss and its gradient share.
int check_distill(const char* who, const trc_hip_tensor* logits, const trc_hip_tensor* labels, const trc_hip_tensor* ids,
                  const trc_hip_tensor* teacher, const trc_hip_tensor* stats, const trc_hip_tensor* loss, float tau, float alpha) {
    if (logits == nullptr || ids == nullptr || teacher == nullptr) return fail(TRC_HIP_E_INVALID, "%s: NULL tensor", who);
    if (!is_float(logits->type)) return fail(TRC_HIP_E_INVALID, "%s: type %d of logits is not F32, F16 or BF16", who, logits->type);
    if (!is_float(teacher->type)) return fail(TRC_HIP_E_INVALID, "%s: type %d of teacher is not F32, F16 or BF16", who, teacher->type);
    const int64_t V = logits->ne[0], T = logits->ne[1], top = ids->ne[0];
    // (the kernels count a row's elements in 32 bits, and some thousands past its end)
    if (V <= 0 || V > (1 << 30) || T <= 0 || T > INT32_MAX || top <= 0 || top > TRC_HIP_DISTILL_MAX_TOP) {
        return fail(TRC_HIP_E_SHAPE, "%s: V = %lld, T = %lld, %lld entries (at most %d)", who, (long long) V, (long long) T,
                    (long long) top, TRC_HIP_DISTILL_MAX_TOP);
    }
    // (the kernels take log2 e / tau as a factor)
    if (!(tau > 0.f) || !(1.f / tau > 0.f) || !(1.44269504f / tau < INFINITY)) return fail(TRC_HIP_E_INVALID, "%s: tau = %g", who, tau);
    if (!(alpha >= 0.f && alpha <= 1.f)) return fail(TRC_HIP_E_INVALID, "%s: alpha = %g is not in 0 .. 1", who, alpha);
    TRC_TRY(check_shape(who, "logits", logits, logits->type, V, T, 1, false));
    TRC_TRY(check_shape(who, "labels", labels, TRC_HIP_TYPE_I32, T, 1, 1, false));
    TRC_TRY(check_shape(who, "ids", ids, TRC_HIP_TYPE_I32, top, T, 1, false));
    TRC_TRY(check_packed(who, "ids", ids));
    TRC_TRY(check_shape(who, "teacher", teacher, teacher->type, top, T, 1, false));
    TRC_TRY(check_packed(who, "teacher", teacher));
    TRC_TRY(check_shape(who, "stats", stats, TRC_HIP_TYPE_F32, 5, T, 1, false));
    TRC_TRY(check_packed(who, "stats", stats));
    return check_shape(who, "loss", loss, TRC_HIP_TYPE_F32, 4, 1, 1, false);
}

}  // namespace

extern "C" {

int trc_hip_distill_loss(const trc_hip_tensor* logits, const trc_hip_tensor* labels, const trc_hip_tensor* ids,
                         const trc_hip_tensor* teacher, float tau, float alpha, const trc_hip_tensor* stats,
                         const trc_hip_tensor* loss, void* stream) {
    const char* const who = "trc_hip_distill_loss";
    TRC_FORCED("trc_hip_distill_loss");
    TRC_TRY(check_distill(who, logits, labels, ids, teacher, stats, loss, tau, alpha));
    const trc_hip_tensor* const all[6] = {stats, loss, logits, labels, ids, teacher};
    const char* const names[6] = {"stats", "loss", "logits", "labels", "ids", "teacher"};
    for (int i = 0; i < 2; ++i) {
        for (int j = i + 1; j < 6; ++j) TRC_TRY(check_apart(who, all[i], names[i], all[j], names[j], false));
    }
    return launch_distill_loss(*logits, (const int32_t*) labels->data, *ids, *teacher, tau, alpha, (float*) stats->data,
                               (float*) loss->data, (hipStream_t) stream);
}

int trc_hip_distill_loss_back(const trc_hip_tensor* logits, const trc_hip_tensor* labels, const trc_hip_tensor* ids,
                              const trc_hip_tensor* teacher, const trc_hip_tensor* stats, const trc_hip_tensor* loss,
                              const trc_hip_tensor* dloss, float tau, float alpha, const trc_hip_tensor* dlogits, void* stream) {
    const char* const who = "trc_hip_distill_loss_back";
    TRC_FORCED("trc_hip_distill_loss_back");
    TRC_TRY(check_distill(who, logits, labels, ids, teacher, stats, loss, tau, alpha));
    TRC_TRY(check_shape(who, "dloss", dloss, TRC_HIP_TYPE_F32, 1, 1, 1, false));
    TRC_TRY(check_shape(who, "dlogits", dlogits, logits->type, logits->ne[0], logits->ne[1], 1, true));
    const trc_hip_tensor* const all[7] = {logits, labels, ids, teacher, stats, loss, dloss};
    const char* const names[7] = {"logits", "labels", "ids", "teacher", "stats", "loss", "dloss"};
    for (int j = 0; j < 7; ++j) TRC_TRY(check_apart(who, dlogits, "dlogits", all[j], names[j], j == 0));
    return launch_distill_loss_back(*logits, (const int32_t*) labels->data, *ids, *teacher, (const float*) stats->data,
                                    (const float*) loss->data, (const float*) dloss->data, tau, alpha, *dlogits, (hipStream_t) stream);
}

}  // extern "C"
