// gtn_paged_attn: attention of new tokens over a paged cache (causal; or a sliding window and first
// tokens that stay visible), GQA, ragged requests.
#include "paged_chunk.cuh"

#include <algorithm>
#include <cmath>

namespace gtn {

// Workers of the decode kernel: the warps that are resident at once; of the chunk kernel: one CTA per SM.
constexpr int DECODE_CTAS = 3;  // per SM, at most
static long decode_workers() { return (long)sm_count() * DECODE_CTAS * PD_WARPS; }
static int64_t join_bytes(long workers) { return (workers * (int64_t)sizeof(PagedJoin) + 15) / 16 * 16; }
static int64_t decode_ws_bytes(int d) {
    return decode_workers() * 2 * 16 * (d + 2) * (int64_t)sizeof(float) + join_bytes(decode_workers());
}
static int64_t chunk_ws_bytes(int d) {
    return (int64_t)sm_count() * 2 * CH_ROWS * (d + 2) * (int64_t)sizeof(float) + join_bytes(sm_count());
}

// The three launches of a call. `chunk_ctas` of the join: 0 without a chunk kernel.
template <int D, int ROWS>
static cudaError_t launch_join(const PagedAttnArgs& dec, const PagedAttnArgs& chunk, int chunk_ctas, int workers, int rows,
                               cudaStream_t st) {
    const int n = chunk_ctas * (CH_ROWS / 32);
    const int warps = join_threads(n > 0) / 32;
    const dim3 grid(n + (workers + warps - 1) / warps * rows), block(32 * warps);
    if (n == 0) return launch_pdl(k_paged_join<ROWS, 0, D>, grid, block, 0, st, dec, chunk, n, workers, rows);
    if constexpr (ROWS > 1) return launch_pdl(k_paged_join<ROWS, CH_ROWS, D>, grid, block, 0, st, dec, chunk, n, workers, rows);
    return cudaErrorInvalidValue;
}

template <int DT, int D, int ROWS>
static cudaError_t launch_decode(PagedAttnArgs a, const PagedPick& p, int most_rows, const PagedAttnArgs& chunk,
                                 int chunk_ctas, cudaStream_t st) {
    using C = DecodeCfg<DT, D, ROWS>;
    static_assert(C::OCC <= DECODE_CTAS, "workspace");
    const int ctas = sm_count() * C::OCC, workers = ctas * PD_WARPS;
    a.workers_mul = (unsigned)((1ull << 32) / (unsigned)workers + 1);
    a.join = reinterpret_cast<PagedJoin*>(a.part + (long)workers * 2 * paged_slot<ROWS, D>());
    cudaError_t e = ensure_smem(k_paged_decode<DT, D, ROWS>, C::SMEM);
    if (e != cudaSuccess) return e;
    e = launch_pdl(k_paged_decode<DT, D, ROWS>, dim3(ctas), dim3(32 * PD_WARPS), C::SMEM, st, a, p);
    if (e != cudaSuccess) return e;
    return launch_join<D, ROWS>(a, chunk, chunk_ctas, workers, std::min(most_rows, ROWS), st);
}

template <int ROWS>
static cudaError_t decode(const PagedAttnArgs& a, const PagedPick& p, int most, const PagedAttnArgs& chunk, int cc,
                          cudaStream_t st) {
    if (a.c.d == 64)
        return a.c.dt == GTN_F16 ? launch_decode<GTN_F16, 64, ROWS>(a, p, most, chunk, cc, st) : launch_decode<GTN_Q8, 64, ROWS>(a, p, most, chunk, cc, st);
    return a.c.dt == GTN_F16 ? launch_decode<GTN_F16, 128, ROWS>(a, p, most, chunk, cc, st) : launch_decode<GTN_Q8, 128, ROWS>(a, p, most, chunk, cc, st);
}

// A pool of fp16 pages as [page][kv head and row][d] for boxes of `box` rows x 64 columns.
static bool page_map(const PagedCache& c, uint8_t* pool, int box, CUtensorMap* m) {
    const TmapEncodeFn fn = tmap_encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)c.d, (cuuint64_t)c.kv_heads * c.ps, (cuuint64_t)c.n_pages};
    const cuuint64_t strides[2] = {(cuuint64_t)c.d * 2, (cuuint64_t)c.page_stride};
    const cuuint32_t bx[3] = {64, (cuuint32_t)box, 1}, es[3] = {1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, pool, dims, strides, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DT, int D>
static cudaError_t launch_chunk(PagedAttnArgs& a, const PagedPick& p, cudaStream_t st) {
    using C = ChunkCfg<DT, D>;
    const int ctas = sm_count();
    a.workers_mul = (unsigned)((1ull << 32) / (unsigned)ctas + 1);
    a.join = reinterpret_cast<PagedJoin*>(a.part + (long)ctas * 2 * paged_slot<CH_ROWS, D>());
    cudaError_t e = ensure_smem(k_paged_chunk<DT, D>, C::SMEM);
    if (e != cudaSuccess) return e;
    CUtensorMap km{}, vm{};
    const int box = std::min(a.c.ps, CH_KEYS);
    if (DT == GTN_F16 && (!page_map(a.c, a.c.k, box, &km) || !page_map(a.c, a.c.v, box, &vm))) return cudaErrorInvalidValue;
    return launch_pdl(k_paged_chunk<DT, D>, dim3(ctas), dim3(CH_THREADS), C::SMEM, st, a, p, km, vm, box);
}

static cudaError_t chunk(PagedAttnArgs& a, const PagedPick& p, cudaStream_t st) {
    if (a.c.d == 64) return a.c.dt == GTN_F16 ? launch_chunk<GTN_F16, 64>(a, p, st) : launch_chunk<GTN_Q8, 64>(a, p, st);
    return a.c.dt == GTN_F16 ? launch_chunk<GTN_F16, 128>(a, p, st) : launch_chunk<GTN_Q8, 128>(a, p, st);
}

}  // namespace gtn

using namespace gtn;

extern "C" {

int64_t gtn_paged_attn_workspace(int heads, int d_head) {
    if (heads < 1 || (d_head != 64 && d_head != 128)) return 0;
    return decode_ws_bytes(d_head) + chunk_ws_bytes(d_head);
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
    GTN_REQUIRE(q->ndim == 2 && out->ndim == 2 && shape_eq(q, out), "%s: q and out must be 2-D, of one shape", who);
    GTN_REQUIRE(q->dtype == out->dtype && (q->dtype == GTN_F16 || q->dtype == GTN_Q8), "%s: q / out dtypes %d, %d", who,
                q->dtype, out->dtype);
    GTN_REQUIRE(q->shape[1] % d == 0, "%s: q of %d columns, d_head %d", who, q->shape[1], d);
    const int heads = q->shape[1] / d;
    GTN_REQUIRE(heads % a.c.kv_heads == 0, "%s: heads %d not a multiple of kv heads %d", who, heads, a.c.kv_heads);
    // what the kernels count in 32 bits: rows by the group (paged_group), units on the line
    const long group = heads / a.c.kv_heads, rows = q->shape[0], cap = (long)block_table->shape[1] * a.c.ps;
    GTN_REQUIRE(rows <= (1 << 20) && (rows * group + CH_ROWS) * group < (1L << 32) && rows * heads < (1L << 31),
                "%s: %ld rows of %d heads", who, rows, heads);
    GTN_REQUIRE(cap < (1L << 30), "%s: block_table of %d pages a row", who, block_table->shape[1]);
    // With a bound on the new tokens that a decode tile holds, the decode kernel takes every request, in tiles as high as
    // the bound: rows / height tiles and one more a request, unless a call could then have more units than 32 bits count.
    const long most = max_new > 0 ? max_new * group : 0x7fffffffL, per_tile = (cap / 16 + 2) * a.c.kv_heads;
    const int height = most == 1 && a.c.dt == GTN_Q8 ? 1 : most <= 8 ? 8 : 16;
    const long all_units = (rows * group / height + (height > 1 ? n : 0)) * per_tile;
    const bool small = most <= 16 && all_units < 0x7fffffffL;
    const long few_units = small ? all_units : n * per_tile;  // else one tile a request
    const long many_units = small ? 0 : (rows * group / CH_ROWS + n) * (cap / CH_KEYS + 2) * a.c.kv_heads;
    GTN_REQUIRE(few_units < 0x7fffffffL && many_units < 0x7fffffffL,
                "%s: %ld rows of %d requests over tables of %ld keys are too many for one call", who, rows, n, cap);
    const gtn_tensor* rt[] = {q, out};
    for (const gtn_tensor* t : rt) {
        GTN_REQUIRE(t->strides[1] == 1 && t->strides[0] >= t->shape[1], "%s: row strides", who);
        if (t->dtype == GTN_F16)
            GTN_REQUIRE((uintptr_t)t->data % 16 == 0 && t->strides[0] % 8 == 0, "%s: fp16 rows must be 16-byte aligned",
                        who);
        else
            GTN_REQUIRE((uintptr_t)t->data % 2 == 0 && t->strides[0] % GTN_QBLK == 0, "%s: Q8 row alignment", who);
    }
    GTN_CHECK(paged_apart(q, out, who, "out"));
    GTN_REQUIRE(std::isfinite(scale) && scale >= 0.0f, "%s: scale", who);
    GTN_REQUIRE(window >= 0 && n_sink >= 0, "%s: window %d, n_sink %d", who, window, n_sink);
    GTN_REQUIRE(max_new >= 0, "%s: max_new", who);
    const int64_t ws_need = gtn_paged_attn_workspace(heads, d);
    GTN_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0, "%s: workspace must be 16-byte aligned device memory", who);
    GTN_REQUIRE(workspace_bytes >= ws_need, "%s: workspace of %ld bytes, %ld needed", who, (long)workspace_bytes,
                (long)ws_need);
    // what is written lies apart from what is read (the pools are only read and may be one)
    const PagedSpan io[] = {paged_span(out),         paged_bytes_span(workspace, ws_need), paged_span(block_table),
                            paged_span(q_start),     paged_span(kv_lens),                  paged_pool_span(a.c, a.c.k),
                            paged_pool_span(a.c, a.c.v)};
    for (int i = 0; i < 2; ++i)
        for (int j = i + 1; j < 7; ++j)
            GTN_REQUIRE(!paged_meet(io[i], io[j]), "%s: %s overlaps %s", who, i ? "workspace" : "out",
                        j == 1 ? "workspace" : j < 5 ? "the lengths or the table" : "the cache");
    GTN_REQUIRE(!paged_meet(io[1], paged_span(q)), "%s: workspace overlaps q", who);
    const void* ptrs[] = {q->data, out->data, a.c.k, a.c.v, block_table->data, q_start->data, kv_lens->data, workspace};
    GTN_CHECK(paged_error_word(&a.err, who));
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
    a.group = (int)group;
    a.group_mul = group > 1 ? (unsigned)(((1ull << 32) + group - 1) / group) : 0;
    a.cap = cap;
    a.most = (unsigned)few_units;
    a.window = window < cap ? window : 0;  // a window of all keys is none (and positions minus it stay in 32 bits)
    a.n_sink = n_sink;
    a.scale_log2 = (scale > 0.0f ? scale : 1.0f / std::sqrt((float)d)) * 1.4426950408889634f;
    a.part = (float*)workspace;
    // Requests of at most `cut` rows per kv head (tokens x query heads of it) go to the decode kernel, whose tiles are
    // 8 or 16 rows high, the others to the chunk kernel (16 requests of two tokens x 8 heads over 500 to 1,900 keys:
    // 20.5 us against 26.6). With a bound on the new tokens that says so, only the decode kernel is launched (single
    // tokens behind a window of 4,096 keys: 58.6 us, 65.5 without the bound). A single request without a bound runs on the
    // chunk kernel alone: the other's empty launch would cost more than its choice gives (one token of TinyLlama at
    // 1,990 keys: 12.3 us on the decode kernel, 20.3 on this way). Single rows over a Q8 cache have a kernel
    // of their own (paged_decode.cuh: 61.5 us against 76.1).
    PagedPick p;
    p.below = true;
    p.chained = false;
    p.cut = a.group <= 8 ? 8 : a.group <= 16 ? 16 : 0;
    cudaError_t e = cudaSuccess;
    if (small) {
        p.cut = 0x7fffffff;
        if (height == 1)
            e = d == 64 ? launch_decode<GTN_Q8, 64, 1>(a, p, 1, a, 0, S(stream))
                        : launch_decode<GTN_Q8, 128, 1>(a, p, 1, a, 0, S(stream));
        else
            e = height == 8 ? decode<8>(a, p, (int)most, a, 0, S(stream)) : decode<16>(a, p, (int)most, a, 0, S(stream));
    } else {
        PagedAttnArgs c = a;
        c.most = (unsigned)many_units;
        c.part = (float*)((uint8_t*)workspace + decode_ws_bytes(d));
        if (n == 1) p.cut = 0;
        PagedPick rest = p;
        rest.below = false;
        e = chunk(c, rest, S(stream));
        p.chained = true;
        if (e == cudaSuccess) {
            if (p.cut == 0)
                e = d == 64 ? launch_join<64, 8>(a, c, sm_count(), 0, 1, S(stream))
                            : launch_join<128, 8>(a, c, sm_count(), 0, 1, S(stream));
            else if (p.cut == 8)
                e = decode<8>(a, p, 8, c, sm_count(), S(stream));
            else
                e = decode<16>(a, p, 16, c, sm_count(), S(stream));
        }
    }
    return cuda_status(e, who);
}

}  // extern "C"
