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
    long cap;          // keys that a row of the table can hold
    float scale_log2;  // scale * log2(e): the softmax runs in base 2
    float* part;       // scratch slots: [worker][2] of ROWS * (D + 2) floats
    PagedJoin* join;   // [worker]
    unsigned int* err;
};

// A request's rows as the kernels take them: row i of [0, n) sits at position base + i; lengths that the
// table or the row tensor cannot hold are flagged and cut.
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
template <int ROWS, int KEYS>
__device__ __forceinline__ PagedTile paged_tile(const PagedAttnArgs& a, const PagedReq& r, int tile) {
    PagedTile t;
    t.plo = r.base + tile * ROWS / a.group;
    t.phi = r.base + min(r.n - 1, (tile * ROWS + ROWS - 1) / a.group);
    t.ns = t.w0 = 0;
    t.units = 1;  // a tile that sees nothing still writes its zeros
    if (t.phi >= 0) {
        const int lo = a.window > 0 ? max(0, t.plo - a.window + 1) : 0;
        t.w0 = lo / KEYS;
        t.ns = min((min(a.n_sink, t.phi + 1) + KEYS - 1) / KEYS, t.w0);
        t.units = t.ns + t.phi / KEYS - t.w0 + 1;
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
};
template <int ROWS>
__device__ __forceinline__ int paged_tiles(const PagedAttnArgs& a, const PagedPick& p, const PagedReq& r) {
    const int m = r.n * a.group;
    return r.n > 0 && (m <= p.cut) == p.below ? (m + ROWS - 1) / ROWS : 0;
}
// The units of each lane's request (nt row tiles; one kv head), by a whole warp: a request of more than two
// tiles is summed by all lanes.
template <int ROWS, int KEYS>
__device__ __forceinline__ long long paged_req_units(const PagedAttnArgs& a, const PagedReq& r, int nt) {
    const int lane = threadIdx.x & 31;
    long long s = 0;
    if (nt <= 2)
        for (int t = 0; t < nt; ++t) s += paged_tile<ROWS, KEYS>(a, r, t).units;
    for (unsigned big = __ballot_sync(0xffffffffu, nt > 2); big; big &= big - 1) {
        const int src = __ffs(big) - 1, n = __shfl_sync(0xffffffffu, nt, src);
        PagedReq q;
        q.first = 0;
        q.n = __shfl_sync(0xffffffffu, r.n, src);
        q.base = __shfl_sync(0xffffffffu, r.base, src);
        long long one = 0;
        for (int t = lane; t < n; t += 32) one += paged_tile<ROWS, KEYS>(a, q, t).units;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) one += __shfl_xor_sync(0xffffffffu, one, o);
        if (lane == src) s = one;
    }
    return s;
}

// a / b for a >= 0, b > 0; in 32 bits where they do.
__device__ __forceinline__ long long paged_div(long long a, long long b) {
    if (((a | b) >> 31) == 0) return (long long)((unsigned)a / (unsigned)b);
    return a / b;
}

// A position on the line of units: item (b, h, tile), unit u of it, the item's first position.
struct PagedPos {
    int b, h, tile, u;
    PagedReq r;
    PagedTile t;
    long long start;
};
template <int W>
struct PagedSchedSmem {
    long long warp[33];
    PagedPos pos[W];
};

// Total units (returned), and in sm.pos[i] the item at position (first + i) * share of workers first ..
// first + W - 1 of `workers` (its b is -1 at or past the end). Called by all THREADS threads of the CTA; ends
// with a barrier.
template <int ROWS, int KEYS, int THREADS, int W>
__device__ __forceinline__ long long paged_sched(const PagedAttnArgs& a, const PagedPick& p, int workers, int first,
                                                 bool flag, PagedSchedSmem<W>& sm) {
    constexpr int NW = THREADS / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // thread tid holds requests [b0, b0 + per); every warp runs all `per` steps
    const int per = (a.n_req + THREADS - 1) / THREADS, b0 = tid * per;
    auto request = [&](int i, PagedReq& r, bool fl) {
        r.first = r.n = r.base = 0;
        if (b0 + i >= a.n_req) return 0;
        r = paged_req(a, b0 + i, fl);
        return paged_tiles<ROWS>(a, p, r);
    };
    long long mine = 0;
    for (int i = 0; i < per; ++i) {
        PagedReq r;
        const int nt = request(i, r, flag);
        mine += paged_req_units<ROWS, KEYS>(a, r, nt);
    }
    mine *= a.c.kv_heads;
    long long s = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += y;
    }
    if (lane == 31) sm.warp[warp] = s;
    if (tid < W) sm.pos[tid].b = -1;
    __syncthreads();
    long long before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        before += w < warp ? sm.warp[w] : 0;
        total += sm.warp[w];
    }
    before += s - mine;
    const long long share = paged_div(total + workers - 1, workers);
    for (int i = 0; i < W; ++i) {
        const long long at = share * (first + i);
        const unsigned own = __ballot_sync(0xffffffffu, at < total && at >= before && at < before + mine);
        if (!own) continue;
        // the warp of the thread whose requests hold the position finds the request, head and tile together
        const int src = __ffs(own) - 1;
        long long start = __shfl_sync(0xffffffffu, before, src), left = at - start;
        bool found = false;
        for (int j = 0; j < per && !found; ++j) {
            PagedReq r;
            const int nt = request(j, r, false);
            const long long mine_one = paged_req_units<ROWS, KEYS>(a, r, nt);
            const long long one = __shfl_sync(0xffffffffu, mine_one, src), all = one * a.c.kv_heads;
            if (left >= all) {
                left -= all;
                start += all;
                continue;
            }
            found = true;
            PagedPos x;
            x.b = __shfl_sync(0xffffffffu, b0 + j, src);
            x.r.first = __shfl_sync(0xffffffffu, r.first, src);
            x.r.n = __shfl_sync(0xffffffffu, r.n, src);
            x.r.base = __shfl_sync(0xffffffffu, r.base, src);
            const int tiles = __shfl_sync(0xffffffffu, nt, src);
            x.h = (int)paged_div(left, one);
            left -= x.h * one;
            start += x.h * one;
            for (int t0 = 0;; t0 += 32) {  // 32 tiles at a time: the first whose end lies behind the position
                const int t = t0 + lane;
                const long long mu = t < tiles ? paged_tile<ROWS, KEYS>(a, x.r, t).units : 0;
                long long e = mu;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const long long y = __shfl_up_sync(0xffffffffu, e, o);
                    if (lane >= o) e += y;
                }
                const unsigned hit = __ballot_sync(0xffffffffu, e > left);
                if (hit || t0 + 32 >= tiles) {
                    const int l = hit ? __ffs(hit) - 1 : 31;
                    const long long st = __shfl_sync(0xffffffffu, e - mu, l);
                    x.tile = t0 + l;
                    x.u = (int)(left - st);
                    x.start = start + st;
                    break;
                }
                const long long e31 = __shfl_sync(0xffffffffu, e, 31);
                left -= e31;
                start += e31;
            }
            x.t = paged_tile<ROWS, KEYS>(a, x.r, x.tile);
            if (lane == 0) sm.pos[i] = x;
        }
    }
    __syncthreads();
    return total;
}

// The next item on the line (b >= n_req behind the last one).
template <int ROWS, int KEYS>
__device__ __forceinline__ void paged_next(const PagedAttnArgs& a, const PagedPick& p, PagedPos& x) {
    x.start += x.t.units;
    x.u = 0;
    if (++x.tile < paged_tiles<ROWS>(a, p, x.r)) {
        x.t = paged_tile<ROWS, KEYS>(a, x.r, x.tile);
        return;
    }
    x.tile = 0;
    if (++x.h == a.c.kv_heads) {
        x.h = 0;
        while (++x.b < a.n_req) {
            x.r = paged_req(a, x.b, false);
            if (paged_tiles<ROWS>(a, p, x.r) > 0) break;
        }
        if (x.b >= a.n_req) return;
    }
    x.t = paged_tile<ROWS, KEYS>(a, x.r, 0);
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
    const int m = tile * rows_per_tile + row, tok = m / a.group;
    return (long)(first + tok) * stride + (long)(h * a.group + m - tok * a.group) * head_bytes;
}

// Joins the items that cross borders: warp (worker w, row y, y + gridDim.y, ...) the one that begins in w's range.
template <int ROWS, int D>
__global__ void __launch_bounds__(128) k_paged_join(PagedAttnArgs a, int workers) {
    pdl_wait();
    const int lane = threadIdx.x & 31, w = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (w >= workers) return;
    const PagedJoin x = a.join[w];
    if (x.last < 0) return;
    constexpr int LANES = D / 4, WAYS = D == 64 ? 2 : 1;  // four columns per lane; parts taken side by side
    const long S = paged_slot<ROWS, D>();
    const float* part = a.part + 2L * w * S;
    const int n = x.last - w + 1;  // part 0: slot 1 of worker w; part i: slot 0 of worker w + i
    auto slot = [&](int i) { return part + (i == 0 ? S : 2L * i * S); };
    for (int row = blockIdx.y; row < x.nrow; row += gridDim.y) {
        float m = -INFINITY;
        for (int i = lane; i < n; i += 32) m = fmaxf(m, slot(i)[ROWS * D + row]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float mm = m == -INFINITY ? 0.0f : m;
        float l = 0.0f, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const int c0 = lane % LANES * 4;
#pragma unroll 4
        for (int i = lane / LANES; i < n; i += WAYS) {
            const float* ps = slot(i);
            const float f = exp2f(ps[ROWS * D + row] - mm);
            const float4 v = *reinterpret_cast<const float4*>(ps + row * D + c0);
            l = fmaf(ps[ROWS * (D + 1) + row], f, l);
            y[0] = fmaf(v.x, f, y[0]);
            y[1] = fmaf(v.y, f, y[1]);
            y[2] = fmaf(v.z, f, y[2]);
            y[3] = fmaf(v.w, f, y[3]);
        }
        if (WAYS == 2) {
            l += __shfl_xor_sync(0xffffffffu, l, 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] += __shfl_xor_sync(0xffffffffu, y[j], 16);
        }
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = l != 0.0f ? y[j] * inv : 0.0f;
        paged_store<4>(a.out + paged_row_at(a, x.first, x.h, x.tile, row, ROWS, a.os, row_bytes(a.io, D)), a.io, c0, y,
                       lane < LANES);
    }
}

// The same for workers that are CTAs: CTA (worker, 128-row tile, 32 columns), a thread per row.
template <int ROWS, int D>
__global__ void __launch_bounds__(128) k_paged_join_cols(PagedAttnArgs a) {
    pdl_wait();
    const int w = blockIdx.x, row = blockIdx.y * 128 + threadIdx.x, c0 = blockIdx.z * 32;
    const PagedJoin x = a.join[w];
    if (x.last < 0 || blockIdx.y * 128 >= x.nrow) return;
    const long S = paged_slot<ROWS, D>();
    const float* part = a.part + 2L * w * S;
    const int n = x.last - w + 1;
    auto slot = [&](int i) { return part + (i == 0 ? S : 2L * i * S); };
    float m = -INFINITY;
    for (int i = 0; i < n; ++i) m = fmaxf(m, slot(i)[ROWS * D + row]);
    const float mm = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, y[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) y[j] = 0.0f;
    for (int i = 0; i < n; ++i) {
        const float* ps = slot(i);
        const float f = exp2f(ps[ROWS * D + row] - mm);
        l = fmaf(ps[ROWS * (D + 1) + row], f, l);
#pragma unroll
        for (int j = 0; j < 32; ++j) y[j] = fmaf(ps[(c0 + j) * ROWS + row], f, y[j]);
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int j = 0; j < 32; ++j) y[j] = l != 0.0f ? y[j] * inv : 0.0f;
    const bool live = row < x.nrow;
    paged_store<32>(a.out + (live ? paged_row_at(a, x.first, x.h, x.tile, row, ROWS, a.os, row_bytes(a.io, D)) : 0), a.io,
                    c0, y, live);
}

}  // namespace gtn
