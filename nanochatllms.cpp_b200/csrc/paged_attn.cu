// gtn_paged_attn: attention of new tokens over a paged cache (causal; or a sliding window and first
// tokens that stay visible), GQA, ragged requests.
#include "paged.cuh"

#include <cmath>

namespace gtn {

struct PagedAttnArgs {
    const uint8_t* q;
    uint8_t* out;
    long qs, os;  // row strides, bytes
    int io;       // dtype of q and out
    PagedCache c;
    const int32_t *table, *q_start, *kv_lens;
    long table_stride;
    int n_req, rows, heads, group, max_pages, window, n_sink;
    float scale_log2;  // scale * log2(e): the softmax runs in base 2
    unsigned int* err;
};

// One warp per (row, query head), the keys in order with a running maximum and sum; lane l holds elements
// l, l + 32, ... of the head.
template <int D>
static __global__ void __launch_bounds__(128) k_paged_attn_rows(PagedAttnArgs a) {
    constexpr int NB = D / GTN_QBLK;
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long u = (long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int t = (int)(u / a.heads), h = (int)(u % a.heads), g = h / a.group;
    if (t >= a.rows || t >= a.q_start[a.n_req]) return;
    int lo = 0, hi = a.n_req - 1;  // the first b with q_start[b + 1] > t
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a.q_start[mid + 1] > t) hi = mid;
        else lo = mid + 1;
    }
    int kv = a.kv_lens[lo];
    if (kv < 0 || kv > (a.max_pages << a.c.ps_shift)) {
        kv = 0;
        if (lane == 0) atomicOr(a.err, GTN_DEVERR_PAGE);
    }
    const int p = kv - (a.q_start[lo + 1] - t);
    const long hb = row_bytes(a.io, D);
    float q[NB], o[NB], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        q[i] = load_elem(a.q + (long)t * a.qs + h * hb, a.io, i * GTN_QBLK + lane);
        o[i] = 0.0f;
    }
    for (int j = 0; j <= p; ++j) {
        if (a.window > 0 && j <= p - a.window && j >= a.n_sink) {
            j = max(j, p - a.window);
            continue;
        }
        const int page = a.table[lo * a.table_stride + (j >> a.c.ps_shift)];
        if (page < 0 || page >= a.c.n_pages) {
            if (lane == 0) atomicOr(a.err, GTN_DEVERR_PAGE);
            continue;
        }
        const int r = j & (a.c.ps - 1);
        const uint8_t* kp = a.c.k + (long)page * a.c.page_stride;
        const uint8_t* vp = a.c.v + (long)page * a.c.page_stride;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NB; ++i) s = fmaf(q[i], paged_elem(a.c, kp, g, r, i * GTN_QBLK + lane), s);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        s *= a.scale_log2;
        const float mn = fmaxf(m, s);
        const float f = exp2f(m - mn), e = exp2f(s - mn);
        l = fmaf(l, f, e);
#pragma unroll
        for (int i = 0; i < NB; ++i) o[i] = fmaf(o[i], f, e * paged_elem(a.c, vp, g, r, i * GTN_QBLK + lane));
        m = mn;
    }
#pragma unroll
    for (int i = 0; i < NB; ++i)
        store_row_elem(a.out + (long)t * a.os + h * hb, a.io, i, lane, D, l > 0.0f || l != l ? o[i] / l : 0.0f);
}

}  // namespace gtn

using namespace gtn;

extern "C" {

int64_t gtn_paged_attn_workspace(int heads, int d_head) {
    if (heads < 1 || (d_head != 64 && d_head != 128)) return 0;
    return 16;
}

int gtn_paged_attn(const gtn_tensor* q, const gtn_paged_cache* cache, const gtn_tensor* block_table,
                   const gtn_tensor* q_start, const gtn_tensor* kv_lens, gtn_tensor* out, float scale, int window,
                   int n_sink, int max_new, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* who = "paged_attn";
    PagedAttnArgs a;
    GTN_CHECK(paged_cache_args(cache, who, &a.c));
    GTN_CHECK(check_tensor(q, "q"));
    GTN_CHECK(check_tensor(out, "out"));
    GTN_CHECK(paged_int_arg(block_table, 2, who, "block_table"));
    GTN_CHECK(paged_int_arg(q_start, 1, who, "q_start"));
    GTN_CHECK(paged_int_arg(kv_lens, 1, who, "kv_lens"));
    const int n = kv_lens->shape[0], d = a.c.d;
    GTN_REQUIRE(n <= PAGED_MAX_REQ, "%s: %d requests (at most %d)", who, n, PAGED_MAX_REQ);
    GTN_REQUIRE(block_table->shape[0] == n && q_start->shape[0] == n + 1, "%s: shapes do not agree on %d requests", who,
                n);
    GTN_REQUIRE((long)block_table->shape[1] * a.c.ps < (1L << 31), "%s: block_table of %d pages a row", who,
                block_table->shape[1]);
    GTN_REQUIRE(q->ndim == 2 && out->ndim == 2 && shape_eq(q, out), "%s: q and out must be 2-D, of one shape", who);
    GTN_REQUIRE(q->dtype == out->dtype && (q->dtype == GTN_F16 || q->dtype == GTN_Q8), "%s: q / out dtypes %d, %d", who,
                q->dtype, out->dtype);
    GTN_REQUIRE(q->shape[1] % d == 0, "%s: q of %d columns, d_head %d", who, q->shape[1], d);
    const int heads = q->shape[1] / d;
    GTN_REQUIRE(heads % a.c.kv_heads == 0, "%s: heads %d not a multiple of kv heads %d", who, heads, a.c.kv_heads);
    GTN_REQUIRE((long)q->shape[0] * heads < (1L << 31), "%s: %d rows of %d heads", who, q->shape[0], heads);
    const gtn_tensor* rt[] = {q, out};
    for (const gtn_tensor* t : rt) {
        GTN_REQUIRE(t->strides[1] == 1 && t->strides[0] >= t->shape[1], "%s: row strides", who);
        if (t->dtype == GTN_F16)
            GTN_REQUIRE((uintptr_t)t->data % 16 == 0 && t->strides[0] % 8 == 0, "%s: fp16 rows must be 16-byte aligned",
                        who);
        else
            GTN_REQUIRE((uintptr_t)t->data % 2 == 0 && t->strides[0] % GTN_QBLK == 0, "%s: Q8 row alignment", who);
    }
    GTN_REQUIRE(std::isfinite(scale) && scale >= 0.0f, "%s: scale", who);
    GTN_REQUIRE(window >= 0 && n_sink >= 0, "%s: window %d, n_sink %d", who, window, n_sink);
    GTN_REQUIRE(max_new >= 0, "%s: max_new", who);
    const int64_t ws_need = gtn_paged_attn_workspace(heads, d);
    GTN_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0, "%s: workspace must be 16-byte aligned device memory", who);
    GTN_REQUIRE(workspace_bytes >= ws_need, "%s: workspace of %ld bytes, %ld needed", who, (long)workspace_bytes,
                (long)ws_need);
    const void* ptrs[] = {q->data, out->data, a.c.k, a.c.v, block_table->data, q_start->data, kv_lens->data, workspace};
    GTN_CHECK(paged_on_device(ptrs, 8, who));
    a.q = (const uint8_t*)q->data;
    a.out = (uint8_t*)out->data;
    a.qs = bstride(q, 0);
    a.os = bstride(out, 0);
    a.io = q->dtype;
    a.table = (const int32_t*)block_table->data;
    a.q_start = (const int32_t*)q_start->data;
    a.kv_lens = (const int32_t*)kv_lens->data;
    a.table_stride = block_table->strides[0];
    a.n_req = n;
    a.rows = q->shape[0];
    a.heads = heads;
    a.group = heads / a.c.kv_heads;
    a.max_pages = block_table->shape[1];
    a.window = window;
    a.n_sink = n_sink;
    a.scale_log2 = (scale > 0.0f ? scale : 1.0f / std::sqrt((float)d)) * 1.4426950408889634f;
    a.err = device_error_word();
    const unsigned grid = (unsigned)(((long)a.rows * heads + 3) / 4);
    const cudaError_t e = d == 64 ? launch_pdl(k_paged_attn_rows<64>, dim3(grid), dim3(128), 0, S(stream), a)
                                  : launch_pdl(k_paged_attn_rows<128>, dim3(grid), dim3(128), 0, S(stream), a);
    return cuda_status(e, who);
}

}  // extern "C"
