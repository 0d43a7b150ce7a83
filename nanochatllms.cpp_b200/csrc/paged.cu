// Paged serving operators: the step planner (gtn_paged_plan) and the cache append with rotary positions
// (gtn_paged_append). The attention over the pages is in paged_attn.cu.
#include "paged.cuh"

#include <cmath>

namespace gtn {

int paged_cache_args(const gtn_paged_cache* c, const char* who, PagedCache* out) {
    GTN_REQUIRE(c, "%s: cache is NULL", who);
    GTN_REQUIRE(c->k && c->v, "%s: cache has no data", who);
    GTN_REQUIRE(c->dtype == GTN_F16 || c->dtype == GTN_Q8, "%s: cache dtype %d (F16 or Q8)", who, c->dtype);
    const long need = gtn_paged_page_bytes(c->dtype, c->page_size, c->kv_heads, c->d_head);
    GTN_REQUIRE(need > 0, "%s: page_size %d, kv_heads %d, d_head %d unsupported", who, c->page_size, c->kv_heads,
                c->d_head);
    GTN_REQUIRE(c->n_pages > 0 && (long)c->n_pages * c->page_size < (1L << 31), "%s: n_pages %d", who, c->n_pages);
    const long stride = c->page_stride ? c->page_stride : need;
    GTN_REQUIRE(stride >= need && stride % 16 == 0 && stride < (1L << 31), "%s: page_stride %ld (pages of %ld bytes)",
                who, (long)c->page_stride, need);
    GTN_REQUIRE((((uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0, "%s: pools must be 16-byte aligned", who);
    out->k = (uint8_t*)c->k;
    out->v = (uint8_t*)c->v;
    out->page_stride = stride;
    out->dt = c->dtype;
    out->n_pages = c->n_pages;
    out->ps = c->page_size;
    out->ps_shift = __builtin_ctz((unsigned)c->page_size);
    out->kv_heads = c->kv_heads;
    out->d = c->d_head;
    return GTN_OK;
}

int paged_int_arg(const gtn_tensor* t, int ndim, const char* who, const char* name) {
    GTN_CHECK(check_tensor(t, name));
    GTN_REQUIRE(t->dtype == GTN_I32 && t->ndim == ndim, "%s: %s must be int32, %d-D", who, name, ndim);
    GTN_REQUIRE((uintptr_t)t->data % 4 == 0, "%s: %s must be 4-byte aligned", who, name);
    GTN_REQUIRE(t->shape[ndim - 1] == 1 || t->strides[ndim - 1] == 1, "%s: %s must be contiguous", who, name);
    GTN_REQUIRE(ndim == 1 || t->strides[0] >= t->shape[1], "%s: %s rows overlap", who, name);
    return GTN_OK;
}

int paged_on_device(const void* const* p, int n, const char* who) {
    int dev = 0;
    GTN_CHECK(cuda_status(cudaGetDevice(&dev), who));
    for (int i = 0; i < n; ++i) {
        cudaPointerAttributes a;
        GTN_CHECK(cuda_status(cudaPointerGetAttributes(&a, p[i]), who));
        GTN_REQUIRE(a.type == cudaMemoryTypeManaged || (a.type == cudaMemoryTypeDevice && a.device == dev),
                    "%s: tensor data %p is not memory of the current device %d", who, p[i], dev);
    }
    return GTN_OK;
}

int paged_error_word(unsigned int** out, const char* who) {
    *out = device_error_word();
    return *out ? GTN_OK : fail(GTN_ERR_CUDA, "%s: the current device has no error word", who);
}

PagedSpan paged_span(const gtn_tensor* t) {
    const uint8_t* p = (const uint8_t*)t->data;
    const long width = row_bytes(t->dtype, t->shape[t->ndim - 1]);
    const long rows = t->ndim > 1 ? t->shape[0] : 1, stride = rows > 1 ? bstride(t, 0) : 0;
    return {p, p + (rows - 1) * stride + width, width, stride};
}

PagedSpan paged_pool_span(const PagedCache& c, const uint8_t* pool) {
    const long width = paged_page_bytes(c.dt, c.ps, c.kv_heads, c.d);
    return {pool, pool + (c.n_pages - 1) * c.page_stride + width, width, c.n_pages > 1 ? c.page_stride : 0};
}

bool paged_meet_rows(const PagedSpan& x, const PagedSpan& y) {
    const long stride = x.stride ? x.stride : y.stride;
    if (stride == 0 || (y.stride && y.stride != stride)) return true;
    long off = (y.data - x.data) % stride;  // of y's columns behind x's
    if (off < 0) off += stride;
    return off < x.width || off + y.width > stride;
}

int paged_apart(const gtn_tensor* q, const gtn_tensor* out, const char* who, const char* name) {
    const bool same = q->data == out->data && q->dtype == out->dtype &&
                      (q->strides[0] == out->strides[0] || q->shape[0] == 1);
    GTN_REQUIRE(same || !paged_meet(paged_span(q), paged_span(out)), "%s: %s overlaps an input", who, name);
    return GTN_OK;
}

// ---- planner -----------------------------------------------------------------------------------
// need_b = ceil((ctx + new) / ps) - ceil(ctx / ps) pages, granted while the inclusive prefix of need
// stays within n_free; q_start = prefix of new. Every CTA runs both prefix sums over all requests itself
// (at most 8 requests a thread; a second kernel for them would cost more than the few microseconds of
// one CTA) and then writes its share of the table entries and of the rows.
// Bound by latency, not by its bytes: 64 decoding requests 7.5 us, 1,000 requests with some 26,000 rows 8.2 us (graph replay,
// B200), of which the launch is some 3 and the two scans, with their dependent loads, the rest.
constexpr int PLAN_THREADS = 512;
constexpr int PLAN_ROWS = 1024;  // rows per CTA

struct PlanArgs {
    const int32_t *ctx, *nw, *free_pages, *n_free;
    int32_t *table, *q_start, *kv_lens, *pos, *slots, *n_used;
    long table_stride;
    int n, n_cap, max_pages, rows, ps_shift;
    unsigned int* err;
};

// Exclusive prefix over the CTA's threads of one value each; *total receives the sum. red: 17 values of
// shared memory.
__device__ __forceinline__ long long plan_scan(long long x, long long* red, long long* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long s = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += y;
    }
    __syncthreads();  // red may still be read from an earlier scan
    if (lane == 31) red[warp] = s;
    __syncthreads();
    if (warp == 0) {
        long long w = lane < PLAN_THREADS / 32 ? red[lane] : 0;
        const long long own = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        if (lane < PLAN_THREADS / 32) red[lane] = w - own;
        if (lane == 31) red[16] = w;
    }
    __syncthreads();
    *total = red[16];
    return red[warp] + s - x;
}

static __global__ void __launch_bounds__(PLAN_THREADS) k_paged_plan(PlanArgs a) {
    __shared__ int s_qend[PAGED_MAX_REQ];  // end row of each request
    __shared__ int s_off[PAGED_MAX_REQ];   // pages of the granted requests before it; -1 - that if not granted
    __shared__ long long red[17];
    __shared__ int s_used;
    pdl_wait();
    const int tid = threadIdx.x, per = (a.n + PLAN_THREADS - 1) / PLAN_THREADS, b0 = tid * per;
    const int psm = (1 << a.ps_shift) - 1;
    int ctx[8], nw[8];
    long long rows = 0, rows_all;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bool in = i < per && b0 + i < a.n;
        ctx[i] = in ? a.ctx[b0 + i] : 0;
        nw[i] = in ? a.nw[b0 + i] : 0;
        rows += nw[i] > 0 ? nw[i] : 0;
    }
    const int n_free = min(a.n_cap, *a.n_free);
    long long end = plan_scan(rows, red, &rows_all);
    int need[8];
    bool fits[8];
    long long pages = 0, pages_all;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        end += nw[i] > 0 ? nw[i] : 0;
        const long long kv = (long long)ctx[i] + nw[i];
        fits[i] = ctx[i] >= 0 && nw[i] >= 0 && kv <= ((long long)a.max_pages << a.ps_shift) && end <= a.rows;
        need[i] = fits[i] ? (int)((kv + psm) >> a.ps_shift) - (int)(((long long)ctx[i] + psm) >> a.ps_shift) : 0;
        pages += need[i];
        if (i < per && b0 + i < a.n) {
            const int e = (int)(end < 0x7fffffffLL ? end : 0x7fffffffLL);
            s_qend[b0 + i] = e;
            if (blockIdx.x == 0) a.q_start[b0 + i + 1] = e;
        }
    }
    if (blockIdx.x == 0 && tid == 0) a.q_start[0] = 0;
    long long off = plan_scan(pages, red, &pages_all);
    if (tid == 0) s_used = 0;
    __syncthreads();
    int used = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bool grant = fits[i] && (need[i] == 0 || off + need[i] <= n_free);
        if (i < per && b0 + i < a.n) {
            s_off[b0 + i] = grant ? (int)min(off, 0x7ffffffeLL) : -1;
            if (blockIdx.x == 0) a.kv_lens[b0 + i] = grant ? ctx[i] + nw[i] : 0;
            if (grant) used += need[i];
        }
        off += need[i];
    }
    if (blockIdx.x == 0 && used) atomicAdd(&s_used, used);
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) *a.n_used = s_used;
    // new table entries: request b by CTA b mod grid, one warp each
    const int lane = tid & 31, warp = tid >> 5;
    for (int b = blockIdx.x * (PLAN_THREADS / 32) + warp; b < a.n; b += gridDim.x * (PLAN_THREADS / 32)) {
        const int o = s_off[b];
        if (o < 0) continue;
        const int c = a.ctx[b], have = (c + psm) >> a.ps_shift;
        const int nd = (int)(((long long)c + a.nw[b] + psm) >> a.ps_shift) - have;
        for (int i = lane; i < nd; i += 32) a.table[b * a.table_stride + have + i] = a.free_pages[o + i];
    }
    // rows: the request by binary search in the row ends, the page from the old table entries or, for a
    // page that this step hands out, from the free list
    for (int t = blockIdx.x * PLAN_ROWS + tid; t < min(a.rows, (int)(blockIdx.x + 1) * PLAN_ROWS); t += PLAN_THREADS) {
        int pos = -1, slot = -1;
        if (t < rows_all) {
            int lo = 0, hi = a.n - 1;  // the first b with s_qend[b] > t
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (s_qend[mid] > t) hi = mid;
                else lo = mid + 1;
            }
            const int c = a.ctx[lo];
            pos = c + (t - (lo > 0 ? s_qend[lo - 1] : 0));
            const int o = s_off[lo];
            if (o >= 0) {
                const int have = (c + psm) >> a.ps_shift, col = pos >> a.ps_shift;
                const int page = col < have ? a.table[lo * a.table_stride + col] : a.free_pages[o + col - have];
                // an id that no pool can hold has no slot: its cells would not fit 31 bits and come out as another page's
                if ((unsigned)page <= 0x7fffffffu >> a.ps_shift) slot = (page << a.ps_shift) + (pos & psm);
                else atomicOr(a.err, GTN_DEVERR_PAGE);
            }
        }
        a.pos[t] = pos;
        a.slots[t] = slot;
    }
}

// ---- append ------------------------------------------------------------------------------------
struct AppendArgs {
    const uint8_t *q, *k, *v;
    long qs, ks, vs, os;  // row strides, bytes
    const int32_t *pos, *slots;
    uint8_t* out;
    PagedCache c;
    int heads, sdt, odt, half;
    unsigned int* err;
};
struct RopeFreq {
    double f[64];  // base^(-2j / rd)
};

constexpr int APP_THREADS = 256;

// The angle in 64 bits, reduced to [-pi, pi] before the fp32 sine (an fp32 angle is off by pos * 2^-24 radians).
__device__ __forceinline__ float2 rope_cs(int pos, double freq) {
    const double x = (double)pos * freq;
    const double r = fma(-rint(x * 0.15915494309189535), 6.283185307179586, x);
    float sn, cn;
    sincosf((float)r, &sn, &cn);
    return make_float2(cn, sn);
}

// Eight elements of a row in dtype DT, from a 16-byte aligned place (Q8: element e0 of the row's blocks).
template <int DT>
__device__ __forceinline__ void app_load8(const uint8_t* head, int e0, float (&x)[8], uint2* raw, uint16_t* dl) {
    if (DT == GTN_F16) {
        const uint4 v = *reinterpret_cast<const uint4*>(head + 2 * e0);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = h2f((uint16_t)w[i]);
            x[2 * i + 1] = h2f((uint16_t)(w[i] >> 16));
        }
    } else if (DT == GTN_F32) {
        const float4 a = *reinterpret_cast<const float4*>(head + 4 * e0), b = *reinterpret_cast<const float4*>(head + 4 * e0 + 16);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
        const uint8_t* blk = head + e0 / GTN_QBLK * GTN_Q8_BYTES;
        *dl = ld_u16(blk);
        const uint8_t* p = blk + 2 + e0 % GTN_QBLK;  // even addresses
        *raw = make_uint2(ld_u16(p) | ((uint32_t)ld_u16(p + 2) << 16), ld_u16(p + 4) | ((uint32_t)ld_u16(p + 6) << 16));
        const float d = h2f(*dl);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = (float)(int8_t)(raw->x >> (8 * i)) * d;
            x[4 + i] = (float)(int8_t)(raw->y >> (8 * i)) * d;
        }
    }
}

// One CTA per row; a thread takes two groups of eight elements of a head: those that rotate into each other (i
// and i + half / 8, for i < half / 8), or two neighbours of the rest. D / 16 adjacent lanes hold a head, so the
// absmax of a 32-element block is a few shuffles. 1,948 rows of Zephyr, fp16, over changing inputs: 16.4 us, 2.9 TB/s;
// MiniCPM's 1,879 rows from fp32 into Q8: 20.2 us, 3.5 TB/s; 16 rows: 4.1 us, a launch. Of what must be moved that is 44%
// and 53% of a copy's rate: a row's second turn is partly empty and loads only when the first has stored. Five CTAs per SM
// (registers) were the best. For rows that are 16-byte aligned and a rotated width of whole groups; k_paged_append_any takes
// the others (the same rows, back to back in L2: 25.8 us, 37.7 us and 4.5 us there, against 10.7, 14.6 and 2.5 here).
template <int D, int SDT>
static __global__ void __launch_bounds__(APP_THREADS, 5) k_paged_append(AppendArgs a, const __grid_constant__ RopeFreq fr) {
    constexpr int TPH = D / 16, NB = D / GTN_QBLK;  // threads and blocks of a head
    __shared__ float2 cs[64];
    pdl_wait();
    pdl_trigger();
    const int t = blockIdx.x, tid = threadIdx.x;
    const int kvh = a.c.kv_heads, hg = a.half >> 3, heads = a.heads + 2 * kvh;
    const long hb = row_bytes(SDT, D);
    const int i = tid % TPH, g0 = i < hg ? i : 2 * hg + 2 * (i - hg), g1 = i < hg ? i + hg : g0 + 1;  // the groups
    float x[2][8];
    uint2 raw[2];
    uint16_t dl[2];
    auto load = [&](int hh) {
        const uint8_t* src = hh < a.heads         ? a.q + (long)t * a.qs + hh * hb
                             : hh < a.heads + kvh ? a.k + (long)t * a.ks + (hh - a.heads) * hb
                                                  : a.v + (long)t * a.vs + (hh - a.heads - kvh) * hb;
        app_load8<SDT>(src, 8 * g0, x[0], &raw[0], &dl[0]);
        app_load8<SDT>(src, 8 * g1, x[1], &raw[1], &dl[1]);
    };
    if (tid / TPH < heads) load(tid / TPH);  // on its way while the position and the angles are found
    const int pos = a.pos[t], slot = a.slots[t];
    if (pos < 0) return;
    if (tid < a.half) cs[tid] = rope_cs(pos, fr.f[tid]);
    const int page = slot >> a.c.ps_shift, r = slot & (a.c.ps - 1);
    const bool store = slot >= 0 && page < a.c.n_pages;
    if (slot >= 0 && !store && tid == 0) atomicOr(a.err, GTN_DEVERR_PAGE);
    __syncthreads();
    // a head's lanes go the same way, the heads of a warp need not (types, turns): shuffles name the head's lanes alone
    const unsigned mates = ((1u << TPH) - 1) << (tid & 31 & ~(TPH - 1));
    for (int hh = tid / TPH; hh < heads; hh += APP_THREADS / TPH) {
        if (hh >= APP_THREADS / TPH) load(hh);
        const int part = hh < a.heads ? 0 : hh < a.heads + kvh ? 1 : 2, h = hh - (part == 0 ? 0 : part == 1 ? a.heads : a.heads + kvh);
        const bool live = part == 0 || store;
        if (part != 2 && i < hg) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float2 w = cs[8 * i + e];
                const float p = x[0][e], q = x[1][e];
                x[0][e] = fmaf(p, w.x, -(q * w.y));
                x[1][e] = fmaf(p, w.y, q * w.x);
            }
        }
        const int odt = part == 0 ? a.odt : a.c.dt;
        uint8_t* pg = (part == 1 ? a.c.k : a.c.v) + (long)page * a.c.page_stride;
        uint8_t* dst = part == 0 ? a.out + (long)t * a.os + h * row_bytes(a.odt, D) : pg + paged_row(a.c, h, r);
        if (odt == GTN_F16) {
            if (!live) continue;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = (uint32_t)f2h(x[k][2 * e]) | ((uint32_t)f2h(x[k][2 * e + 1]) << 16);
                *reinterpret_cast<uint4*>(dst + 16 * (k ? g1 : g0)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            continue;
        }
        // the activation quantizer (warp_quant_block): absmax of each block over the head's lanes
        float mx[2] = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) mx[k] = fmaxf(mx[k], fabsf(x[k][e]));
        float m0 = 0.0f, m1 = 0.0f;  // of this lane's two groups' blocks
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float m = fmaxf(g0 >> 2 == b ? mx[0] : 0.0f, g1 >> 2 == b ? mx[1] : 0.0f);
#pragma unroll
            for (int o = 1; o < TPH; o <<= 1) m = fmaxf(m, __shfl_xor_sync(mates, m, o));
            if (g0 >> 2 == b) m0 = m;
            if (g1 >> 2 == b) m1 = m;
        }
        if (!live) continue;
        const bool pass = SDT == GTN_Q8 && part == 2;  // V blocks pass unchanged
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int g = k ? g1 : g0;
            const float delta = (k ? m1 : m0) / 127.0f, inv = delta != 0.0f ? 1.0f / delta : 0.0f;
            uint32_t w[2] = {0u, 0u};
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e >> 2] |= (uint32_t)(uint8_t)(int8_t)roundf(x[k][e] * inv) << (8 * (e & 3));
            uint16_t dh = f2h(delta);
            if (pass) {
                w[0] = raw[k].x;
                w[1] = raw[k].y;
                dh = dl[k];
            }
            if (part == 0) {
                uint8_t* blk = dst + (g >> 2) * GTN_Q8_BYTES;
                uint16_t* y = reinterpret_cast<uint16_t*>(blk + 2 + 8 * (g & 3));
                if ((g & 3) == 0) *reinterpret_cast<uint16_t*>(blk) = dh;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
            } else {
                *reinterpret_cast<uint2*>(dst + 8 * g) = make_uint2(w[0], w[1]);
                if ((g & 3) == 0) reinterpret_cast<uint16_t*>(pg + paged_delta(a.c, h, r))[g >> 2] = dh;
            }
        }
    }
}

// Any alignment of the rows and any rotated width. One CTA per row, one warp per head; lane l holds elements l,
// l + 32, ... of its head, so that a 32-element block is one element per lane (the activation quantizer's layout).
template <int D>
static __global__ void __launch_bounds__(APP_THREADS) k_paged_append_any(AppendArgs a, const __grid_constant__ RopeFreq fr) {
    constexpr int NB = D / GTN_QBLK;
    __shared__ float2 cs[64];
    __shared__ float buf[APP_THREADS / 32][D];
    pdl_wait();
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int pos = a.pos[t], slot = a.slots[t];
    if (pos < 0) return;
    if (tid < a.half) cs[tid] = rope_cs(pos, fr.f[tid]);
    __syncthreads();
    const int kvh = a.c.kv_heads, page = slot >> a.c.ps_shift, r = slot & (a.c.ps - 1);
    const bool store = slot >= 0 && page < a.c.n_pages;
    if (slot >= 0 && !store && tid == 0) atomicOr(a.err, GTN_DEVERR_PAGE);
    const long hb = row_bytes(a.sdt, D);
    for (int hh = warp; hh < a.heads + 2 * kvh; hh += APP_THREADS / 32) {
        const bool is_q = hh < a.heads, is_k = !is_q && hh < a.heads + kvh;
        if (!is_q && !store) continue;
        const int h = is_q ? hh : (is_k ? hh - a.heads : hh - a.heads - kvh);
        const uint8_t* src = (is_q ? a.q + (long)t * a.qs : is_k ? a.k + (long)t * a.ks : a.v + (long)t * a.vs) + h * hb;
        float x[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) x[i] = load_elem(src, a.sdt, i * GTN_QBLK + lane);
        if ((is_q || is_k) && a.half > 0) {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < NB; ++i) buf[warp][i * GTN_QBLK + lane] = x[i];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const int e = i * GTN_QBLK + lane;
                if (e < a.half) {
                    const float2 w = cs[e];
                    x[i] = fmaf(x[i], w.x, -(buf[warp][e + a.half] * w.y));
                } else if (e < 2 * a.half) {
                    const float2 w = cs[e - a.half];
                    x[i] = fmaf(buf[warp][e - a.half], w.y, x[i] * w.x);
                }
            }
        }
        if (is_q) {
            uint8_t* dst = a.out + (long)t * a.os + h * row_bytes(a.odt, D);
#pragma unroll
            for (int i = 0; i < NB; ++i) store_row_elem(dst, a.odt, i, lane, D, x[i]);
            continue;
        }
        uint8_t* pg = (is_k ? a.c.k : a.c.v) + (long)page * a.c.page_stride;
        uint8_t* dst = pg + paged_row(a.c, h, r);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            if (a.c.dt == GTN_F16) {
                reinterpret_cast<uint16_t*>(dst)[i * GTN_QBLK + lane] = f2h(x[i]);
                continue;
            }
            uint16_t dh;
            int8_t qv;
            if (!is_k && a.sdt == GTN_Q8) {  // V blocks pass unchanged
                dh = ld_u16(src + i * GTN_Q8_BYTES);
                qv = (int8_t)src[i * GTN_Q8_BYTES + 2 + lane];
            } else {
                qv = warp_quant_block(x[i], lane, GTN_QBLK, &dh);
            }
            dst[i * GTN_QBLK + lane] = (uint8_t)qv;
            if (lane == 0) reinterpret_cast<uint16_t*>(pg + paged_delta(a.c, h, r))[i] = dh;
        }
    }
}

}  // namespace gtn

using namespace gtn;

extern "C" {

int64_t gtn_paged_page_bytes(int dtype, int page_size, int kv_heads, int d_head) {
    if (dtype != GTN_F16 && dtype != GTN_Q8) return 0;
    if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1))) return 0;
    if ((d_head != 64 && d_head != 128) || kv_heads < 1 || kv_heads > 1024) return 0;
    return paged_page_bytes(dtype, page_size, kv_heads, d_head);
}

int gtn_check(void* stream) {
    GTN_CHECK(cuda_status(cudaStreamSynchronize(S(stream)), "check"));
    return check_dev_err();
}

int gtn_paged_plan(const gtn_tensor* ctx_lens, const gtn_tensor* new_lens, const gtn_tensor* free_pages,
                   const gtn_tensor* n_free, int page_size, gtn_tensor* block_table, gtn_tensor* q_start,
                   gtn_tensor* kv_lens, gtn_tensor* pos, gtn_tensor* slots, gtn_tensor* n_used, void* stream) {
    const char* who = "paged_plan";
    GTN_CHECK(paged_int_arg(ctx_lens, 1, who, "ctx_lens"));
    GTN_CHECK(paged_int_arg(new_lens, 1, who, "new_lens"));
    // a list that has run out may be empty (then without memory): requests that need no page go on
    const bool none = free_pages && free_pages->dtype == GTN_I32 && free_pages->ndim == 1 && free_pages->shape[0] == 0;
    if (!none) GTN_CHECK(paged_int_arg(free_pages, 1, who, "free_pages"));
    GTN_CHECK(paged_int_arg(n_free, 1, who, "n_free"));
    GTN_CHECK(paged_int_arg(block_table, 2, who, "block_table"));
    GTN_CHECK(paged_int_arg(q_start, 1, who, "q_start"));
    GTN_CHECK(paged_int_arg(kv_lens, 1, who, "kv_lens"));
    GTN_CHECK(paged_int_arg(pos, 1, who, "pos"));
    GTN_CHECK(paged_int_arg(slots, 1, who, "slots"));
    GTN_CHECK(paged_int_arg(n_used, 1, who, "n_used"));
    const int n = ctx_lens->shape[0];
    GTN_REQUIRE(n <= PAGED_MAX_REQ, "%s: %d requests (at most %d)", who, n, PAGED_MAX_REQ);
    GTN_REQUIRE(new_lens->shape[0] == n && kv_lens->shape[0] == n && block_table->shape[0] == n &&
                    q_start->shape[0] == n + 1,
                "%s: shapes do not agree on %d requests", who, n);
    GTN_REQUIRE(pos->shape[0] == slots->shape[0], "%s: pos and slots differ in rows", who);
    GTN_REQUIRE(page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0, "%s: page_size %d", who,
                page_size);
    // (lengths of granted requests then fit 31 bits; paged_attn has the same limit)
    GTN_REQUIRE((long)block_table->shape[1] * page_size < (1L << 30), "%s: block_table of %d pages a row", who,
                block_table->shape[1]);
    const gtn_tensor* io[] = {block_table, q_start, kv_lens, pos, slots, n_used, ctx_lens, new_lens, free_pages, n_free};
    PagedSpan span[10];
    for (int i = 0; i < 10; ++i) span[i] = none && io[i] == free_pages ? paged_bytes_span(nullptr, 0) : paged_span(io[i]);
    for (int i = 0; i < 6; ++i)
        for (int j = i + 1; j < 10; ++j)
            GTN_REQUIRE(!paged_meet(span[i], span[j]), "%s: tensors that are written overlap others", who);
    const void* ptrs[] = {ctx_lens->data, new_lens->data, none ? n_free->data : free_pages->data, n_free->data, block_table->data,
                          q_start->data,  kv_lens->data,  pos->data,        slots->data,  n_used->data};
    PlanArgs a;
    GTN_CHECK(paged_error_word(&a.err, who));
    GTN_CHECK(paged_on_device(ptrs, 10, who));
    a.ctx = (const int32_t*)ctx_lens->data;
    a.nw = (const int32_t*)new_lens->data;
    a.free_pages = (const int32_t*)free_pages->data;
    a.n_free = (const int32_t*)n_free->data;
    a.table = (int32_t*)block_table->data;
    a.q_start = (int32_t*)q_start->data;
    a.kv_lens = (int32_t*)kv_lens->data;
    a.pos = (int32_t*)pos->data;
    a.slots = (int32_t*)slots->data;
    a.n_used = (int32_t*)n_used->data;
    a.table_stride = block_table->strides[0];
    a.n = n;
    a.n_cap = free_pages->shape[0];
    a.max_pages = block_table->shape[1];
    a.rows = pos->shape[0];
    a.ps_shift = __builtin_ctz((unsigned)page_size);
    return cuda_status(launch_pdl(k_paged_plan, dim3((a.rows + PLAN_ROWS - 1) / PLAN_ROWS), dim3(PLAN_THREADS), 0,
                                  S(stream), a),
                       who);
}

int gtn_paged_append(const gtn_tensor* q, const gtn_tensor* k, const gtn_tensor* v, const gtn_tensor* pos,
                     const gtn_tensor* slots, const gtn_paged_cache* cache, gtn_tensor* q_out, float rope_pct,
                     float rope_base, void* stream) {
    const char* who = "paged_append";
    AppendArgs a;
    GTN_CHECK(paged_cache_args(cache, who, &a.c));
    GTN_CHECK(check_tensor(q, "q"));
    GTN_CHECK(check_tensor(k, "k"));
    GTN_CHECK(check_tensor(v, "v"));
    GTN_CHECK(check_tensor(q_out, "q_out"));
    GTN_CHECK(paged_int_arg(pos, 1, who, "pos"));
    GTN_CHECK(paged_int_arg(slots, 1, who, "slots"));
    GTN_REQUIRE(q->ndim == 2 && k->ndim == 2 && v->ndim == 2 && q_out->ndim == 2, "%s: 2-D rows", who);
    const int rows = q->shape[0], d = a.c.d, kvd = a.c.kv_heads * d;
    GTN_REQUIRE(q->shape[1] % d == 0, "%s: q of %d columns, d_head %d", who, q->shape[1], d);
    GTN_REQUIRE(k->shape[0] == rows && k->shape[1] == kvd && v->shape[0] == rows && v->shape[1] == kvd,
                "%s: k / v must be [%d, %d]", who, rows, kvd);
    GTN_REQUIRE(q_out->shape[0] == rows && q_out->shape[1] == q->shape[1], "%s: q_out shape", who);
    GTN_REQUIRE(pos->shape[0] == rows && slots->shape[0] == rows, "%s: pos / slots must have %d entries", who, rows);
    GTN_REQUIRE(q->dtype == k->dtype && k->dtype == v->dtype, "%s: q, k, v dtypes differ", who);
    GTN_REQUIRE(q->dtype == GTN_F16 || q->dtype == GTN_F32 || q->dtype == GTN_Q8, "%s: q dtype %d", who, q->dtype);
    GTN_REQUIRE(q_out->dtype == GTN_F16 || q_out->dtype == GTN_Q8, "%s: q_out dtype %d", who, q_out->dtype);
    const gtn_tensor* rt[] = {q, k, v, q_out};
    for (const gtn_tensor* t : rt) {
        GTN_REQUIRE(t->strides[1] == 1 && t->strides[0] >= t->shape[1], "%s: row strides", who);
        GTN_REQUIRE(t->dtype != GTN_Q8 || t->strides[0] % GTN_QBLK == 0, "%s: Q8 row stride %d", who, t->strides[0]);
        GTN_REQUIRE((uintptr_t)t->data % (t->dtype == GTN_F32 ? 4 : 2) == 0, "%s: row alignment", who);
    }
    GTN_CHECK(paged_apart(q, q_out, who, "q_out"));
    // what is written lies apart from what is read: k and v too where q_out is q's own memory (as column ranges beside it)
    const PagedSpan qo = paged_span(q_out), kp = paged_pool_span(a.c, a.c.k), vp = paged_pool_span(a.c, a.c.v);
    GTN_REQUIRE(!paged_meet(paged_span(k), qo) && !paged_meet(paged_span(v), qo), "%s: q_out overlaps k or v", who);
    GTN_REQUIRE(!paged_meet(kp, vp), "%s: the pools of the cache overlap", who);
    GTN_REQUIRE(!paged_meet(qo, kp) && !paged_meet(qo, vp), "%s: q_out overlaps the cache", who);
    const gtn_tensor* in[] = {q, k, v, pos, slots};
    for (const gtn_tensor* t : in)
        GTN_REQUIRE(!paged_meet(paged_span(t), kp) && !paged_meet(paged_span(t), vp), "%s: the cache overlaps an input", who);
    GTN_REQUIRE(!paged_meet(paged_span(pos), qo) && !paged_meet(paged_span(slots), qo), "%s: q_out overlaps pos or slots", who);
    GTN_REQUIRE(rope_pct >= 0.0f && rope_pct <= 1.0f, "%s: rope_pct", who);
    GTN_REQUIRE(rope_base > 0.0f && std::isfinite(rope_base), "%s: rope_base", who);
    const void* ptrs[] = {q->data, k->data, v->data, q_out->data, pos->data, slots->data, a.c.k, a.c.v};
    GTN_CHECK(paged_error_word(&a.err, who));
    GTN_CHECK(paged_on_device(ptrs, 8, who));
    a.q = (const uint8_t*)q->data;
    a.k = (const uint8_t*)k->data;
    a.v = (const uint8_t*)v->data;
    a.out = (uint8_t*)q_out->data;
    a.qs = bstride(q, 0);
    a.ks = bstride(k, 0);
    a.vs = bstride(v, 0);
    a.os = bstride(q_out, 0);
    a.pos = (const int32_t*)pos->data;
    a.slots = (const int32_t*)slots->data;
    a.heads = q->shape[1] / d;
    a.sdt = q->dtype;
    a.odt = q_out->dtype;
    const int rd = (int)((float)d * rope_pct);
    a.half = rd / 2;
    RopeFreq fr;
    for (int j = 0; j < 64; ++j) fr.f[j] = j < a.half ? std::pow((double)rope_base, -2.0 * j / rd) : 0.0;  // (rd may be odd)
    bool aligned = a.half % 8 == 0;
    for (const gtn_tensor* t : rt)
        aligned = aligned && (t->dtype == GTN_Q8 || ((uintptr_t)t->data % 16 == 0 && bstride(t, 0) % 16 == 0));
#define GTN_APP(DV, SDT) launch_pdl(k_paged_append<DV, SDT>, dim3(rows), dim3(APP_THREADS), 0, S(stream), a, fr)
#define GTN_APP_D(DV)                                                                              \
    (!aligned ? launch_pdl(k_paged_append_any<DV>, dim3(rows), dim3(APP_THREADS), 0, S(stream), a, fr) \
     : a.sdt == GTN_F16 ? GTN_APP(DV, GTN_F16) : a.sdt == GTN_F32 ? GTN_APP(DV, GTN_F32) : GTN_APP(DV, GTN_Q8))
    const cudaError_t e = d == 64 ? GTN_APP_D(64) : GTN_APP_D(128);
#undef GTN_APP_D
#undef GTN_APP
    return cuda_status(e, who);
}

}  // extern "C"
