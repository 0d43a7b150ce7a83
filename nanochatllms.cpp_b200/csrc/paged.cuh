// The paged cache as the kernels see it (include/gten_b200.h describes the page layout) and what the
// paged operators share.
#pragma once
#include "abi.cuh"

namespace gtn {

#define GTN_DEVERR_PAGE 8u  // a page id, slot or length read on the device is out of range

constexpr int PAGED_MAX_REQ = 4096;

struct PagedCache {
    uint8_t* k;
    uint8_t* v;
    long page_stride;  // bytes
    int dt, n_pages, ps, ps_shift, kv_heads, d;
};

__host__ __device__ inline long paged_page_bytes(int dt, int ps, int kv_heads, int d) {
    const long n = (long)ps * kv_heads * d;
    return dt == GTN_F16 ? 2 * n : n + n / GTN_QBLK * 2;
}
// Byte offset inside a page of element 0 of (head h, row r), and of its first Q8 delta.
__device__ __forceinline__ long paged_row(const PagedCache& c, int h, int r) {
    return ((long)h * c.ps + r) * c.d * (c.dt == GTN_F16 ? 2 : 1);
}
__device__ __forceinline__ long paged_delta(const PagedCache& c, int h, int r) {
    return (long)c.kv_heads * c.ps * c.d + ((long)h * c.ps + r) * (c.d / GTN_QBLK) * 2;
}
// The element of a page (K or V) as fp32.
__device__ __forceinline__ float paged_elem(const PagedCache& c, const uint8_t* page, int h, int r, int e) {
    if (c.dt == GTN_F16) return h2f(reinterpret_cast<const uint16_t*>(page + paged_row(c, h, r))[e]);
    const float dl = h2f(reinterpret_cast<const uint16_t*>(page + paged_delta(c, h, r))[e / GTN_QBLK]);
    return (float)reinterpret_cast<const int8_t*>(page + paged_row(c, h, r))[e] * dl;
}

// Checks a cache descriptor and fills the kernels' form of it.
int paged_cache_args(const gtn_paged_cache* c, const char* who, PagedCache* out);
// An int32 vector or matrix argument (contiguous rows).
int paged_int_arg(const gtn_tensor* t, int ndim, const char* who, const char* name);
// Every pointer lies in memory that the current device owns (or managed memory). Turns a host pointer or
// another device's tensor into an error before a kernel meets it.
int paged_on_device(const void* const* p, int n, const char* who);
// The device error word, which the kernels write without asking whether there is one.
int paged_error_word(unsigned int** out, const char* who);
// The rows of a tensor (or the pages of a pool): `width` bytes every `stride` bytes (0: one row), in [data, end).
struct PagedSpan {
    const uint8_t *data, *end;
    long width, stride;
};
PagedSpan paged_span(const gtn_tensor* t);
PagedSpan paged_pool_span(const PagedCache& c, const uint8_t* pool);
inline PagedSpan paged_bytes_span(const void* p, long n) { return {(const uint8_t*)p, (const uint8_t*)p + n, n, 0}; }
// Whether two of them may share bytes. Exact for rows of one stride (column ranges of one buffer); rows of different
// strides count as meeting when their ranges do.
bool paged_meet_rows(const PagedSpan& x, const PagedSpan& y);
inline bool paged_meet(const PagedSpan& x, const PagedSpan& y) {
    return x.data < y.end && y.data < x.end && paged_meet_rows(x, y);
}
// out may be q's own memory row for row, else it must lie apart from it.
int paged_apart(const gtn_tensor* q, const gtn_tensor* out, const char* who, const char* name);

// Attributes common to the kernels: nothing is read before the previous kernel in the stream is done.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace gtn
