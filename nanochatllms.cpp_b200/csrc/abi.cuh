// Descriptor checks and small helpers shared by the op-level entry points of the C ABI.
#pragma once
#include "launch.cuh"

namespace gtn {

inline int cuda_status(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return GTN_OK;
    return fail(e == cudaErrorMemoryAllocation ? GTN_ERR_OOM : GTN_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

// cuTensorMapEncodeTiled, reached through the runtime's driver entry point (nullptr: not available).
typedef CUresult (*TmapEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
TmapEncodeFn tmap_encode_fn();

// Multiprocessors of the current device.
int sm_count();

// Reads and clears the device error word; the stream whose kernels are meant has been waited for.
inline int check_dev_err() {
    const unsigned int v = take_device_error();
    if (v)
        return fail(GTN_ERR_DEVICE, "device-side error code %u (1: a bounded wait expired, 2: token id out of range, 8: page, slot or "
                    "length out of range)",
                    v);
    return GTN_OK;
}

// ---- tensor helpers (tensor.h:96-116 bstride) -------------------------------------------------
inline bool valid_dtype(int dt) { return dt >= GTN_I32 && dt <= GTN_Q4; }

inline long bstride(const gtn_tensor* t, int i) {
    const long s = t->strides[i];
    switch (t->dtype) {
        case GTN_Q4: return s == 1 ? 1 : (s / GTN_QBLK) * GTN_Q4_BYTES;
        case GTN_Q8: return s == 1 ? 1 : (s / GTN_QBLK) * GTN_Q8_BYTES;
        case GTN_F16: return s * 2;
        default: return s * 4;
    }
}

inline int check_tensor(const gtn_tensor* t, const char* name) {
    if (!t) return fail(GTN_ERR_ARG, "%s is NULL", name);
    if (!t->data) return fail(GTN_ERR_ARG, "%s has no data", name);
    if (!valid_dtype(t->dtype)) return fail(GTN_ERR_ARG, "%s has invalid dtype %d", name, t->dtype);
    if (t->ndim < 1 || t->ndim > 3) return fail(GTN_ERR_ARG, "%s has %d dims", name, t->ndim);
    for (int i = 0; i < t->ndim; ++i)
        if (t->shape[i] <= 0) return fail(GTN_ERR_ARG, "%s dim %d is %d", name, i, t->shape[i]);
    // Quantized rows of a partial last block: the reference allocates ceil(n/32) blocks per row
    // (tensor.cpp:43-45) but steps rows by floor(n/32) blocks (tensor.h:196-200), so rows beyond
    // the first overlap. Only single-row use is well defined.
    if ((t->dtype == GTN_Q8 || t->dtype == GTN_Q4) && t->ndim >= 2 && t->shape[t->ndim - 1] % GTN_QBLK != 0) {
        long rows = 1;
        for (int i = 0; i < t->ndim - 1; ++i) rows *= t->shape[i];
        if (rows > 1)
            return fail(GTN_ERR_ARG, "%s: quantized rows of %d elements (not a multiple of 32) overlap", name,
                        t->shape[t->ndim - 1]);
    }
    return GTN_OK;
}

inline bool shape_eq(const gtn_tensor* a, const gtn_tensor* b) {
    if (a->ndim != b->ndim) return false;
    for (int i = 0; i < a->ndim; ++i)
        if (a->shape[i] != b->shape[i]) return false;
    return true;
}

inline cudaStream_t S(void* s) { return reinterpret_cast<cudaStream_t>(s); }

#define GTN_CHECK(expr)                 \
    do {                                \
        const int rc_ = (expr);         \
        if (rc_ != GTN_OK) return rc_;  \
    } while (0)
#define GTN_REQUIRE(cond, ...)                              \
    do {                                                    \
        if (!(cond)) return fail(GTN_ERR_ARG, __VA_ARGS__); \
    } while (0)

}  // namespace gtn
