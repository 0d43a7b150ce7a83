// Work distribution of the paged attention kernels.
//
// An item is one tile of ROWS query rows (token-major, the `group` query heads of one kv head per token)
// of one request and kv head; a unit is KEYS consecutive keys of an item. The units of all items form one
// line, ordered by request, kv head, row tile and key, and worker c (a warp or a CTA) takes units
// [c * share, (c + 1) * share) of it, share = ceil(units / workers): every worker does the same work whatever
// the lengths are, and a single long request spreads over the whole GPU. An item that lies in one worker's
// range is finished there; of an item that crosses a border, each worker leaves its unnormalised sums in
// its own scratch slots (slot 0: the item began before the range; slot 1: it begins in it), and
// k_paged_join adds them up in the order of the workers. Everything is computed from the lengths on the
// device, the same for every worker of a call.
#pragma once
#include "paged.cuh"

namespace gtn {

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// What a worker says of the item that begins in its range and goes on behind it.
struct PagedJoin {
    int last;                   // the last worker of the item; -1: there is no such item
    int first, h, tile, nrow;   // the item: first row of its request, kv head, row tile, query rows
};

struct PagedAttnArgs {
    const uint8_t* q;
    uint8_t* out;
    long qs, os;  // row strides, bytes
    int io;       // dtype of q and out
    PagedCache c;
    const int32_t *table, *q_start, *kv_lens;
    long table_stride;
    int n_req, rows, heads, group, window, n_sink;
    unsigned group_mul;  // floor(x / group) = umulhi(x, group_mul) for x < 2^32 / group (0: group is 1)
    long cap;          // keys that a row of the table can hold
    unsigned most;     // units that a kernel can have for lengths that agree with the tensors
    unsigned workers_mul;  // floor(2^32 / workers) + 1
    float scale_log2;  // scale * log2(e): the softmax runs in base 2
    float* part;       // scratch slots: [worker][2] of ROWS * (D + 2) floats
    PagedJoin* join;   // [worker]
    unsigned int* err;
};

// A request's rows as the kernels take them: row i of [0, n) sits at position base + i; lengths that the
// table cannot hold are flagged and cut; rows behind the tensor's end (a plan's refused requests) are cut.
struct PagedReq {
    int first;  // row of token 0 in q and out
    int n;      // tokens
    int base;   // position of token 0 (negative: tokens before the first key see nothing)
};
__device__ __forceinline__ PagedReq paged_req(const PagedAttnArgs& a, int b, bool flag) {
    const int s = a.q_start[b], e = a.q_start[b + 1];
    int kv = a.kv_lens[b];
    bool bad = kv < 0 || kv > a.cap || s < 0 || e < s;
    if (kv < 0 || kv > a.cap) kv = 0;
    PagedReq r;
    r.first = s;
    r.n = s < 0 || s >= a.rows || e <= s ? 0 : min(e, a.rows) - s;
    r.base = e > s ? kv - (e - s) : 0;
    if (bad && flag) atomicOr(a.err, GTN_DEVERR_PAGE);
    return r;
}

// The keys of one row tile: sink units [0, ns), then units w0, w0 + 1, ...
struct PagedTile {
    int plo, phi;  // positions of the tile's first and last token
    int ns, w0, units;
};
// A kernel spends some 20 cycles per instruction that it runs for the first time (the instruction cache is cold
// at its start), so what follows is short code rather than little work: 32-bit numbers (the host refuses calls of
// 2^31 units or more), a multiplication for the division by the group, loops that are not unrolled.
__device__ __forceinline__ int paged_group(const PagedAttnArgs& a, int m) {
    return a.group_mul ? (int)__umulhi((unsigned)m, a.group_mul) : m;
}
template <int ROWS, int KEYS>
__device__ __forceinline__ PagedTile paged_tile(const PagedAttnArgs& a, const PagedReq& r, int tile) {
    PagedTile t;
    t.plo = r.base + paged_group(a, tile * ROWS);
    t.phi = r.base + min(r.n - 1, paged_group(a, tile * ROWS + ROWS - 1));
    t.ns = t.w0 = 0;
    t.units = 1;  // a tile that sees nothing still writes its zeros
    if (t.phi >= 0) {
        if (a.window > 0) {
            t.w0 = (unsigned)max(0, t.plo - a.window + 1) / KEYS;
            t.ns = min((int)(((unsigned)min(a.n_sink, t.phi + 1) + KEYS - 1) / KEYS), t.w0);
        }
        t.units = t.ns + (int)((unsigned)t.phi / KEYS) - t.w0 + 1;
    }
    return t;
}
template <int KEYS>
__device__ __forceinline__ int paged_unit_key(const PagedTile& t, int u) {
    return (u < t.ns ? u : t.w0 + u - t.ns) * KEYS;
}

// Which requests a kernel takes: those of at most `cut` rows per kv head, or the others.
struct PagedPick {
    int cut;
    bool below;
    bool chained;  // the decode kernel behind the chunk kernel of the same call (see there)
};
template <int ROWS>
__device__ __forceinline__ int paged_tiles(const PagedAttnArgs& a, const PagedPick& p, const PagedReq& r) {
    const int m = r.n * a.group;
    return r.n > 0 && (m <= p.cut) == p.below ? (int)((unsigned)(m + ROWS - 1) / ROWS) : 0;
}

// A position on the line of units: item (b, h, tile), unit u of it, the item's first position.
struct PagedPos {
    int b, h, tile, u;
    PagedReq r;
    PagedTile t;
    unsigned start;
};

// Units of the tiles [0, nt) of a request (one kv head), by a whole warp.
template <int ROWS, int KEYS>
__device__ __forceinline__ unsigned paged_warp_units(const PagedAttnArgs& a, const PagedReq& r, int nt) {
    unsigned s = 0;
#pragma unroll 1
    for (int t = threadIdx.x & 31; t < nt; t += 32) s += paged_tile<ROWS, KEYS>(a, r, t).units;
    return __reduce_add_sync(0xffffffffu, s);
}

// pre[i]: units of the requests of threads 0 .. i of THREADS, thread i holding `per` requests from i * per on.
// By the whole CTA; ends with a barrier. BIG: requests of many tiles are common (each is summed by a warp).
// Returns the units of all, or 0 (and flags it) if they are more than valid lengths can give: row ranges that
// overlap must not become work without end. Sums stop at 2^31 - 1, which a single request's units do not reach
// (the host refuses such calls).
__device__ __forceinline__ unsigned paged_add(unsigned x, unsigned y) { return min(x + y, 0x7fffffffu); }
template <int ROWS, int KEYS, int THREADS, bool BIG>
__device__ __forceinline__ unsigned paged_sched(const PagedAttnArgs& a, const PagedPick& p, bool flag, unsigned* pre,
                                            unsigned* wsum) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (a.n_req + THREADS - 1) / THREADS;
    unsigned mine = 0, units;
#pragma unroll 1
    for (int i = 0; i < per; ++i) {
        const int b = tid * per + i;
        PagedReq r;
        r.first = r.n = r.base = 0;
        if (b < a.n_req) r = paged_req(a, b, flag);
        const int nt = paged_tiles<ROWS>(a, p, r);
        units = 0;
        if (BIG) {
            for (unsigned any = __ballot_sync(0xffffffffu, nt > 0); any; any &= any - 1) {
                const int src = __ffs(any) - 1;
                PagedReq q;
                q.first = 0;
                q.n = __shfl_sync(0xffffffffu, r.n, src);
                q.base = __shfl_sync(0xffffffffu, r.base, src);
                const unsigned one = paged_warp_units<ROWS, KEYS>(a, q, __shfl_sync(0xffffffffu, nt, src));
                if (lane == src) units = one;
            }
        } else {
#pragma unroll 1
            for (int t = 0; t < nt; ++t) units += paged_tile<ROWS, KEYS>(a, r, t).units;
        }
        mine = paged_add(mine, units * a.c.kv_heads);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, mine, o);
        if (lane >= o) mine = paged_add(mine, y);
    }
    if (lane == 31) wsum[warp] = mine;
    __syncthreads();
    for (int w = 0; w < warp; ++w) mine = paged_add(mine, wsum[w]);
    pre[tid] = mine;
    __syncthreads();
    const unsigned total = pre[THREADS - 1];
    if (total <= a.most) return total;
    if (flag && tid == 0) atomicOr(a.err, GTN_DEVERR_PAGE);
    return 0;
}
// Units per worker, a bit more than total / workers at most (the same for every worker).
__device__ __forceinline__ unsigned paged_share(unsigned total, unsigned workers_mul) {
    return total ? __umulhi(total - 1, workers_mul) + 1 : 1;
}

// The item at position `at` < total of the line, by a whole warp.
template <int ROWS, int KEYS, int THREADS, bool BIG>
__device__ __forceinline__ PagedPos paged_locate(const PagedAttnArgs& a, const PagedPick& p, unsigned at,
                                                 const unsigned* pre) {
    const int lane = threadIdx.x & 31, per = (a.n_req + THREADS - 1) / THREADS;
    int before = 0;  // threads whose requests end at or before the position
#pragma unroll 1
    for (int j = lane; j < THREADS; j += 32) before += pre[j] <= at;
    before = __reduce_add_sync(0xffffffffu, before);
    PagedPos x;
    x.b = before * per;
    x.start = before ? pre[before - 1] : 0;
    unsigned one;
    int nt;
#pragma unroll 1
    for (;; ++x.b) {
        x.r = paged_req(a, x.b, false);
        nt = paged_tiles<ROWS>(a, p, x.r);
        one = paged_warp_units<ROWS, KEYS>(a, x.r, nt);
        if (at - x.start < one * a.c.kv_heads || x.b + 1 >= a.n_req) break;
        x.start += one * a.c.kv_heads;
    }
    x.h = (int)((at - x.start) / one);
    x.start += x.h * one;
#pragma unroll 1
    for (int t0 = 0;; t0 += 32) {  // 32 tiles at a time: the first whose end lies behind the position
        const unsigned mu = t0 + lane < nt ? paged_tile<ROWS, KEYS>(a, x.r, t0 + lane).units : 0;
        unsigned e = mu;
        if (BIG) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned y = __shfl_up_sync(0xffffffffu, e, o);
                if (lane >= o) e += y;
            }
        } else if (nt > 1) {
#pragma unroll 1
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned y = __shfl_up_sync(0xffffffffu, e, o);
                if (lane >= o) e += y;
            }
        }
        const unsigned hit = __ballot_sync(0xffffffffu, e > at - x.start);
        const int l = hit ? __ffs(hit) - 1 : 31;
        if (hit || t0 + 32 >= nt) {
            x.start += __shfl_sync(0xffffffffu, e - mu, l);
            x.tile = t0 + l;
            break;
        }
        x.start += __shfl_sync(0xffffffffu, e, 31);
    }
    x.u = (int)(at - x.start);
    x.t = paged_tile<ROWS, KEYS>(a, x.r, x.tile);
    return x;
}

// The next item on the line (b >= n_req behind the last one).
template <int ROWS, int KEYS>
__device__ __forceinline__ void paged_next(const PagedAttnArgs& a, const PagedPick& p, PagedPos& x) {
    x.start += x.t.units;
    x.u = 0;
    if (++x.tile >= paged_tiles<ROWS>(a, p, x.r)) {
        x.tile = 0;
        if (++x.h == a.c.kv_heads) {
            x.h = 0;
            while (++x.b < a.n_req) {
                x.r = paged_req(a, x.b, false);
                if (paged_tiles<ROWS>(a, p, x.r) > 0) break;
            }
            if (x.b >= a.n_req) return;
        }
    }
    x.t = paged_tile<ROWS, KEYS>(a, x.r, x.tile);
}

// ---- scratch slots ------------------------------------------------------------------------------
// One slot: ROWS * D sums (row by row for warps as workers, column by column for CTAs, whose threads own a row
// each), ROWS running maxima, ROWS sums of weights.
template <int ROWS, int D>
__host__ __device__ constexpr long paged_slot() {
    return ((long)ROWS * (D + 2) + 3) / 4 * 4;  // (whole 16 bytes)
}

// Writes columns [c0, c0 + N) of one head's row in dtype io, 32 / N adjacent lanes per 32-element block;
// every lane of the warp takes part, those with `live` write.
template <int N>
__device__ __forceinline__ void paged_store(uint8_t* head, int io, int c0, const float (&y)[N], bool live) {
    constexpr int T = GTN_QBLK / N;
    static_assert(GTN_QBLK % N == 0 && N % 4 == 0, "whole blocks");
    if (io == GTN_F16) {
        if (!live) return;
        uint32_t w[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) w[i] = (uint32_t)f2h(y[2 * i]) | ((uint32_t)f2h(y[2 * i + 1]) << 16);
        if constexpr (N % 8 == 0) {
            uint4* dst = reinterpret_cast<uint4*>(head + 2 * c0);
#pragma unroll
            for (int i = 0; i < N / 8; ++i) dst[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        } else {
            uint2* dst = reinterpret_cast<uint2*>(head + 2 * c0);
#pragma unroll
            for (int i = 0; i < N / 4; ++i) dst[i] = make_uint2(w[2 * i], w[2 * i + 1]);
        }
        return;
    }
    // the activation quantizer (warp_quant_block): absmax without NaN, delta, 1 / delta unrounded, roundf
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, fabsf(y[i]));
#pragma unroll
    for (int o = 1; o < T; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (!live) return;
    const float delta = m / 127.0f, inv = delta != 0.0f ? 1.0f / delta : 0.0f;
    uint8_t* blk = head + c0 / GTN_QBLK * GTN_Q8_BYTES;
    if (c0 % GTN_QBLK == 0) *reinterpret_cast<uint16_t*>(blk) = f2h(delta);
    uint16_t* dst = reinterpret_cast<uint16_t*>(blk + 2 + c0 % GTN_QBLK);  // blocks start at even addresses
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const uint32_t lo = (uint8_t)(int8_t)roundf(y[2 * i] * inv), hi = (uint8_t)(int8_t)roundf(y[2 * i + 1] * inv);
        dst[i] = (uint16_t)(lo | (hi << 8));
    }
}

// Offset of an item's row in q or out: token, head.
__device__ __forceinline__ long paged_row_at(const PagedAttnArgs& a, int first, int h, int tile, int row, int rows_per_tile,
                                             long stride, long head_bytes) {
    const int m = tile * rows_per_tile + row, tok = paged_group(a, m);
    return (long)(first + tok) * stride + (long)(h * a.group + m - tok * a.group) * head_bytes;
}

// Joins the items that cross borders: the one that begins in worker w's range, rows row0, row0 + step, ..., by a
// warp.
template <int ROWS, int D>
__device__ __forceinline__ void paged_join_rows(const PagedAttnArgs& a, int w, int row0, int step) {
    const int lane = threadIdx.x & 31;
    const PagedJoin x = a.join[w];
    if (x.last < 0) return;
    constexpr int LANES = D / 4, WAYS = D == 64 ? 2 : 1;  // four columns per lane; parts taken side by side
    const long S = paged_slot<ROWS, D>();
    const float* part = a.part + 2L * w * S;
    const int n = x.last - w + 1;  // part 0: slot 1 of worker w; part i: slot 0 of worker w + i
    auto slot = [&](int i) { return part + (i == 0 ? S : 2L * i * S); };
    for (int row = row0; row < x.nrow; row += step) {
        float m = -INFINITY;
        for (int i = lane; i < n; i += 32) m = fmaxf(m, slot(i)[ROWS * D + row]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float mm = m == -INFINITY ? 0.0f : m;
        float l = 0.0f, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const int c0 = lane % LANES * 4, way = lane / LANES;
        for (int i0 = 0; i0 < n; i0 += 32) {  // lane i: the weight of part i0 + i
            float f = 0.0f;
            if (i0 + lane < n) {
                const float* ps = slot(i0 + lane) + ROWS * D + row;
                f = ex2(ps[0] - mm);
                l = fmaf(ps[ROWS], f, l);
            }
            const int k = min(32, n - i0);
#pragma unroll 8
            for (int i = 0; i < k; i += WAYS) {
                const float w = __shfl_sync(0xffffffffu, f, (i + way) & 31);
                if (WAYS == 1 || i + way < k) {
                    const float4 v = *reinterpret_cast<const float4*>(slot(i0 + i + way) + row * D + c0);
                    y[0] = fmaf(v.x, w, y[0]);
                    y[1] = fmaf(v.y, w, y[1]);
                    y[2] = fmaf(v.z, w, y[2]);
                    y[3] = fmaf(v.w, w, y[3]);
                }
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (WAYS == 2)
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] += __shfl_xor_sync(0xffffffffu, y[j], 16);
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = l != 0.0f ? y[j] * inv : 0.0f;
        paged_store<4>(a.out + paged_row_at(a, x.first, x.h, x.tile, row, ROWS, a.os, row_bytes(a.io, D)), a.io, c0, y,
                       lane < LANES);
    }
}

__host__ __device__ constexpr int join_threads(bool chunk) { return chunk ? 256 : 128; }

// The same for workers that are CTAs: rows row0 .. row0 + 31 of the item, by a CTA: lane = row, a warp D / 8 columns;
// through shared memory, so that rows leave whole.
template <int ROWS, int D>
__device__ __forceinline__ void paged_join_cols(const PagedAttnArgs& a, int w, int row0) {
    constexpr int N = D / 8, L = D / 4;  // columns per thread; lanes that write a row
    __shared__ float tile[32][D + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = row0 + lane;
    const PagedJoin x = a.join[w];
    if (x.last < 0 || row0 >= x.nrow) return;
    const long S = paged_slot<ROWS, D>();
    const float* part = a.part + 2L * w * S + row;
    const int n = x.last - w + 1;
    auto slot = [&](int i) { return part + (i == 0 ? S : 2L * i * S); };
    float m = -INFINITY;
#pragma unroll 1
    for (int i = 0; i < n; ++i) m = fmaxf(m, slot(i)[ROWS * D]);
    const float mm = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, y[N];
#pragma unroll
    for (int j = 0; j < N; ++j) y[j] = 0.0f;
#pragma unroll 2
    for (int i = 0; i < n; ++i) {
        const float* ps = slot(i);
        const float f = ex2(ps[ROWS * D] - mm);
        l = fmaf(ps[ROWS * (D + 1)], f, l);
#pragma unroll
        for (int j = 0; j < N; ++j) y[j] = fmaf(ps[(warp * N + j) * ROWS], f, y[j]);
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) tile[lane][warp * N + j] = l != 0.0f ? y[j] * inv : 0.0f;
    __syncthreads();
#pragma unroll 1
    for (int i = warp * 4; i < warp * 4 + 4; i += 32 / L) {
        const int r = i + lane / L, c0 = lane % L * 4;
        const bool live = row0 + r < x.nrow;
        float z[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) z[j] = tile[r][c0 + j];
        paged_store<4>(a.out + (live ? paged_row_at(a, x.first, x.h, x.tile, row0 + r, ROWS, a.os, row_bytes(a.io, D)) : 0), a.io,
                       c0, z, live);
    }
}

// What both kernels of a call have left: the first `chunk_ctas` CTAs join the chunk kernel's items, 32 rows each, the
// others the decode kernel's: a warp takes one row (of row_step) of one worker (of `workers`), so that an item's rows,
// which read the most where a sequence is spread over the whole GPU, fall to different SMs. CROWS = 0: there is no
// chunk kernel; without its part the code has the registers to keep eight parts in flight (TinyLlama at 1,990 keys:
// 12.3 us against 13.0).
template <int ROWS, int CROWS, int D>
__global__ void __launch_bounds__(join_threads(CROWS > 0), CROWS > 0 ? 4 : 1) k_paged_join(PagedAttnArgs dec, PagedAttnArgs chunk, int chunk_ctas,
                                                                int workers, int row_step) {
    pdl_wait();
    constexpr int WARPS = join_threads(CROWS > 0) / 32;
    const int i = blockIdx.x;
    if constexpr (CROWS > 0)
        if (i < chunk_ctas) {
            paged_join_cols<CROWS, D>(chunk, i / (CROWS / 32), i % (CROWS / 32) * 32);
            return;
        }
    const int w = (i - chunk_ctas) / row_step * WARPS + (threadIdx.x >> 5);
    if (w < workers) paged_join_rows<ROWS, D>(dec, w, (i - chunk_ctas) % row_step, row_step);
}

}  // namespace gtn
