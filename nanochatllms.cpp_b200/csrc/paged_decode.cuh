// Paged attention for few query rows per kv head (single tokens, short drafts): bound by reading K and V
// once. The keys of all requests are spread evenly over the GPU's warps (paged_sched.cuh: a worker is a warp);
// each warp streams its keys through a ring of its own in shared memory (16-byte asynchronous copies, some
// 8 KB a stage, the next stages in flight while one is computed, across items too) and meets no other
// warp: there is no barrier behind the first lines.
//
// S = Q K^T and O = P V run on m16n8k16 instructions (fp16 in, fp32 sums) with up to 16 query rows as M; at one
// token the products are small next to the loads. Fragments come from shared memory without transposition:
//   * contraction over d: any one-to-one assignment of d to (k step, lane) works if Q uses the same; lane
//     (g, t) = (lane / 4, lane % 4) holds its key's elements 32 c + 8 t .. + 7 of each 32-element chunk c;
//   * contraction over keys: column n of a score tile is key perm(n); the weight fragment's keys are then
//     perm(2t), perm(2t + 1), and lane (g, t) reads those rows of V; a byte permute pairs two keys, and the
//     order of the columns in the result is the reads'.
// Rows lie with their 16-byte chunks exchanged by row (dst below); perm is chosen per row width so that every
// read of K and V meets all banks once.
// Q8 caches keep their 8-bit values exact in fp16; the deltas are applied in fp32, to the scores per
// 32-element block of K and to the weights per 32-column block of V before these round to fp16.
//
// One query row per kv head over a Q8 cache (no grouping, single tokens) wastes instructions on that way: 7
// of 8 rows of every fragment are empty. There (ROWS = 1) a lane owns whole keys: scores are 8-bit dot products
// (dp4a) of the key with the query, itself split into two bytes per element (q = scale (256 hi + lo), 2^-16 of
// the block's largest; Q8 queries are their own byte, exactly), softmax runs on one or two scores per lane, and
// only P V goes through the matrix instructions, the weights turned into its fragment in shared memory.
// (MiniCPM's batch of 64, Q8: 61.5 us against 76.1 through fragments.)
//
// Measured (graph replay, B200): 16 sequences of 32/8 heads of 128 behind a window of 4,096 keys, fp16: 59 us, 4.56 TB/s,
// 69% of a copy's rate; the kernel alone reads 269 MB (what it must) in 53 us. MiniCPM's batch of 64, Q8: 63 us, 3.8
// TB/s: 910 instructions per 64 keys take half the issue slots, with three warps per scheduler: what bounds it is the
// latency between dependent instructions rather than their number. One TinyLlama sequence of 1,990 keys: 12.3 us, all
// latency: the schedule and its first run of code 3 us, two steps of keys, and the join behind a second launch.
// Fewer stages with more CTAs per SM (F16: 2 stages, 3 CTAs), and more CTAs than are resident, measured the same or
// slower.
#pragma once
#include "paged_sched.cuh"

namespace gtn {

constexpr int PD_WARPS = 4;  // per CTA
// A worker takes two steps at least: a single sequence would else end in twice as many parts to join (TinyLlama
// at 1,990 keys: 16.9 us with one step, 14.3 with two, 14.7 with four).
constexpr unsigned PD_SHARE = 2;
// The weights are 2^(s - max + PD_BIAS) instead of 2^(s - max), which cancels in the division: small weights
// (and weights times small deltas) stay that much longer above fp16's subnormal range.
constexpr float PD_BIAS = 6.0f;

template <int DT, int D, int ROWS>
struct DecodeCfg {
    static constexpr bool Q = DT == GTN_Q8;
    static constexpr int RB = Q ? D : 2 * D;                // bytes of a row in the cache
    static constexpr int KEYS = 4096 / RB;                  // keys of a step (one unit): 4 KB of K and of V
    static constexpr int DELTA = Q ? KEYS * (D / 32) * 2 : 0;
    static constexpr int STAGE = 2 * (KEYS * RB + DELTA);
    static constexpr int STAGES = Q ? 2 : 3;
    // CTAs per SM, by shared memory; two of the kernel that 168 registers do not hold
    static constexpr int OCC = Q && !(D == 128 && ROWS == 16) ? 3 : 2;
    static constexpr int SMEM = PD_WARPS * STAGES * STAGE;
    // perm(0) in the lowest digit
    static constexpr uint32_t PERM = !Q ? 0x73625140u : D == 64 ? 0x67235410u : 0x57136420u;
    static constexpr uint32_t inverse() {
        uint32_t v = 0;
        for (int i = 0; i < 8; ++i) v |= (uint32_t)i << (4 * ((PERM >> (4 * i)) & 7));
        return v;
    }
    static constexpr uint32_t INVERSE = inverse();
};

__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const uint8_t* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// 16 bytes from global to shared memory, or 16 zero bytes (src is then not read).
__device__ __forceinline__ void cp_async16(uint32_t dst, const uint8_t* src, bool take) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t p) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t p) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(p) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds4(uint32_t p) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(p) : "memory");
    return v;
}

// Eight fp16 elements e0 .. e0 + 7 of a row in dtype io (Q8: rounded to fp16, 2^-11 relative, far below the step of Q8 queries).
__device__ __forceinline__ uint4 paged_q8x(const uint8_t* head, int io, int e0) {
    if (io == GTN_F16) return *reinterpret_cast<const uint4*>(head + 2 * e0);
    const uint8_t* blk = head + e0 / GTN_QBLK * GTN_Q8_BYTES;
    const float dl = h2f(ld_u16(blk));
    const uint8_t* p = blk + 2 + e0 % GTN_QBLK;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t two = ld_u16(p + 2 * i);
        w[i] = pack_f16((float)(int8_t)(two & 0xff) * dl, (float)(int8_t)(two >> 8) * dl);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Bytes b0, b1 of two words (one of each key) as fp16 pairs (exact integers): columns j and j + 1.
__device__ __forceinline__ uint2 pair_bytes(uint32_t k0, uint32_t k1, bool high) {
    return tc_bytes_to_f16x4(__byte_perm(k0, k1, high ? 0x7362 : 0x5140) ^ 0x80808080u, 0x64806480u);
}

template <int DT, int D, int ROWS>
__global__ void __launch_bounds__(32 * PD_WARPS, DecodeCfg<DT, D, ROWS>::OCC) k_paged_decode(PagedAttnArgs a, PagedPick p) {
    using C = DecodeCfg<DT, D, ROWS>;
    constexpr bool Q = C::Q;
    constexpr int KEYS = C::KEYS, RB = C::RB, NC = D / 32, NT = KEYS / 8, NH = KEYS / 16;
    constexpr int NO = D / 8;        // 8-column tiles of the output
    constexpr bool R16 = ROWS == 16, ONE = ROWS == 1;
    static_assert(!ONE || Q, "single rows of fp16 caches run as eight");
    constexpr int NR = R16 ? 2 : 1;  // rows per lane: g, and g + 8
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ unsigned s_pre[32 * PD_WARPS], s_wsum[PD_WARPS];
    // Behind the chunk kernel of the same call there is nothing to wait for: that one let this one start when all
    // before it was done, and the two share nothing. It then waits at its end instead, so that what follows finds
    // both done.
    if (!p.chained) pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const unsigned me = blockIdx.x * PD_WARPS + warp;
    if (lane == 0) a.join[me].last = -1;
    const unsigned total = paged_sched<ROWS, KEYS, 32 * PD_WARPS, false>(a, p, blockIdx.x == 0, s_pre, s_wsum);
    const unsigned share = max(PD_SHARE, paged_share(total, a.workers_mul));
    if (share * me >= total) {
        if (p.chained) pdl_wait();
        return;
    }
    PagedPos x = paged_locate<ROWS, KEYS, 32 * PD_WARPS, false>(a, p, share * me, s_pre);
    int left = (int)min(total - share * me, share);
    const long hb = row_bytes(a.io, D);
    const uint32_t ring = smem_u32(smem) + warp * (C::STAGES * C::STAGE);
    auto perm = [](int i) { return (int)(C::PERM >> (4 * i)) & 7; };

    // ---- copies: the warp's position `y` on the line runs STAGES - 1 steps ahead of the computed one
    PagedPos y = x;
    int ahead = left, slot_in = 0, page = 0, ykb = 0, ylo = 0;  // ykb: first key of the step at y
    const long vk = a.c.v - a.c.k;                              // from a byte of the K pool to V's
    const int hrow = a.c.ps * RB;                               // bytes of a head in a page
    // lane i < NH: the page of the step's 16-key piece i; -1: no key of it is seen
    auto find_page = [&]() {
        ykb = paged_unit_key<KEYS>(y.t, y.u);
        if (lane < NH) {
            const int k0 = ykb + 16 * lane;
            const bool need = k0 <= y.t.phi && (k0 + 15 >= ylo || k0 < a.n_sink);
            page = need ? a.table[y.b * a.table_stride + (k0 >> a.c.ps_shift)] : -1;
            if (need && (unsigned)page >= (unsigned)a.c.n_pages) {
                page = -1;
                atomicOr(a.err, GTN_DEVERR_PAGE);
            }
        }
    };
    ylo = a.window > 0 ? max(0, y.t.plo - a.window + 1) : 0;
    find_page();
    // where this lane's 16 bytes of copy i go in a stage: rows lie 128 (64) bytes apart with their chunks exchanged
    constexpr int CPR = RB / 16, RPI = 32 / CPR;  // chunks per row, rows per copy instruction
    const int cr = lane / CPR, cc = lane % CPR;
    const uint32_t d0 = RB == 256 ? (cc >> 3) * (KEYS * 128) + cr * 128 + (((cc & 7) ^ cr) << 4)
                      : RB == 128 ? cr * 128 + ((cc ^ cr) << 4)
                                  : cr * 64 + ((cc ^ ((cr >> 1) & 3)) << 4);
    auto dst_of = [&](int i) {  // copy i: rows i * RPI + cr
        if (RB == 256) return (d0 ^ ((uint32_t)(i & 3) << 5)) + i * 256;
        if (RB == 128) return (d0 ^ ((uint32_t)(i & 1) << 6)) + i * 512;
        return d0 + i * 512;
    };
    auto fetch = [&]() {
        if (ahead > 0) {
            const uint32_t st = ring + slot_in * C::STAGE;
            // every key of the step is seen by some row and every page is there
            const bool whole = ykb + KEYS - 1 <= y.t.phi && (ykb >= ylo || ykb + KEYS <= a.n_sink) &&
                               !__any_sync(0xffffffffu, lane < NH && page < 0);
            const uint8_t* head = a.c.k + (long)y.h * hrow + lane * 16;
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                const int pg = __shfl_sync(0xffffffffu, page, h);
                const int row0 = (ykb + 16 * h) & (a.c.ps - 1);
                const uint8_t* src = head + (unsigned long)(unsigned)max(pg, 0) * (unsigned)a.c.page_stride + row0 * RB;
                const uint8_t* vsrc = src + vk;
                if (whole) {
#pragma unroll
                    for (int i = 0; i < 16 / RPI; ++i) {
                        const uint32_t d = st + dst_of(h * (16 / RPI) + i);
                        cp_async16(d, src + i * 512);
                        cp_async16(d + KEYS * RB, vsrc + i * 512);
                    }
                } else {
#pragma unroll 1
                    for (int i = 0; i < 16 / RPI; ++i) {
                        const int key = ykb + 16 * h + i * RPI + cr;
                        const bool take = pg >= 0 && key <= y.t.phi && (key >= ylo || key < a.n_sink);
                        const uint32_t d = st + dst_of(h * (16 / RPI) + i);
                        cp_async16(d, src + i * 512, take);
                        cp_async16(d + KEYS * RB, vsrc + i * 512, take);
                    }
                }
            }
            if (Q) {  // the deltas: lanes 0-15 K's, 16-31 V's
                constexpr int LPP = 2 * NC;  // lanes per 16-key piece (16 keys of NC fp16 deltas)
                static_assert(!Q || LPP * NH == 16, "half a warp each");
                const int h = (lane & 15) / LPP, pg = __shfl_sync(0xffffffffu, page, h);
                const uint8_t* src = (lane < 16 ? a.c.k : a.c.v) +
                                     (unsigned long)(unsigned)max(pg, 0) * (unsigned)a.c.page_stride +
                                     (long)a.c.kv_heads * hrow +
                                     (y.h * a.c.ps + ((ykb + 16 * h) & (a.c.ps - 1))) * (NC * 2) + lane % LPP * 16;
                cp_async16(st + 2 * KEYS * RB + lane * 16, src, pg >= 0);
            }
            slot_in = slot_in + 1 == C::STAGES ? 0 : slot_in + 1;
            if (--ahead > 0) {
                if (++y.u == y.t.units) {
                    paged_next<ROWS, KEYS>(a, p, y);
                    ylo = a.window > 0 ? max(0, y.t.plo - a.window + 1) : 0;
                }
                find_page();
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int i = 0; i < C::STAGES - 1; ++i) fetch();

    // ---- reads of the fragments, relative to a stage
    const int pk = perm(g), p0 = perm(2 * t), p1 = perm(2 * t + 1);
    uint32_t koff, voff0, voff1;  // K: key pk, chunk 0; V: keys p0 and p1
    if (!Q) {
        const int ch = (g >> 1) + 4 * (g & 1);  // the 16-byte chunk of V (8 columns) of this lane
        koff = pk * 128 + ((t ^ pk) << 4);
        voff0 = p0 * 128 + ((ch ^ p0) << 4);
        voff1 = p1 * 128 + ((ch ^ p1) << 4);
    } else if (D == 64) {
        koff = pk * 64 + ((((t >> 1) ^ (pk >> 1)) & 3) << 4) + (t & 1) * 8;
        voff0 = p0 * 64 + ((((g >> 2) ^ (p0 >> 1)) & 3) << 4) + (g & 3) * 4;
        voff1 = p1 * 64 + ((((g >> 2) ^ (p1 >> 1)) & 3) << 4) + (g & 3) * 4;
    } else {
        koff = pk * 128 + (((t >> 1) ^ pk) << 4) + (t & 1) * 8;
        voff0 = p0 * 128 + (((g >> 2) ^ p0) << 4) + (g & 3) * 4;
        voff1 = p1 * 128 + (((g >> 2) ^ p1) << 4) + (g & 3) * 4;
    }
    // chunk c of a row: fp16 rows hold two chunks of 32 elements per 128 bytes, Q8 rows one per 32 bytes
    auto chunk = [](uint32_t off, int c) { return Q ? off ^ (c << 5) : (off ^ ((c & 1) << 6)) + (c >> 1) * (KEYS * 128); };

    int slot = 0;
    while (left > 0) {
        const int u0 = x.u, u1 = min(x.t.units, u0 + left);
        const int nrow = min(ROWS, x.r.n * a.group - x.tile * ROWS);  // query rows of this item
        uint32_t qa[ONE ? 1 : 2 * NC][4];                       // query fragments
        uint32_t qhi[ONE ? D / 4 : 1], qlo[ONE ? D / 4 : 1];    // or the query's bytes
        float qsc[ONE ? NC : 1];                                // and what they are worth, per 32 elements
        bool has_lo = false;
        int pos[NR];
        if constexpr (ONE) {
            pos[0] = x.r.base + paged_group(a, x.tile);
            const uint8_t* qh = a.q + paged_row_at(a, x.r.first, x.h, x.tile, 0, ROWS, a.qs, hb);
            has_lo = a.io == GTN_F16;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                uint32_t hi, lo = 0;
                if (a.io == GTN_F16) {
                    const float v = h2f(reinterpret_cast<const uint16_t*>(qh)[32 * c + lane]);
                    const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(v))));
                    const int q16 = top > 0.0f ? __float2int_rn(v * (32512.0f / top)) : 0;
                    hi = (uint32_t)((q16 + 128) >> 8);
                    lo = (uint32_t)(q16 - (int)(hi << 8));
                    qsc[c] = top * (1.0f / 32512.0f);  // (infinite or NaN with any element of the block)
                } else {
                    const uint8_t* blk = qh + c * GTN_Q8_BYTES;
                    hi = blk[2 + lane];
                    qsc[c] = h2f(ld_u16(blk));
                }
                // four lanes' bytes to a word, and the words to every lane
                hi &= 0xffu;
                lo &= 0xffu;
                hi |= __shfl_down_sync(0xffffffffu, hi, 1) << 8;
                lo |= __shfl_down_sync(0xffffffffu, lo, 1) << 8;
                hi |= __shfl_down_sync(0xffffffffu, hi, 2) << 16;
                lo |= __shfl_down_sync(0xffffffffu, lo, 2) << 16;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    qhi[8 * c + i] = __shfl_sync(0xffffffffu, hi, 4 * i);
                    qlo[8 * c + i] = __shfl_sync(0xffffffffu, lo, 4 * i);
                }
            }
        } else {
            // query fragments: k step i covers elements 4 (i % 2) .. + 3 of every lane's eight of chunk i / 2
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const int row = g + 8 * r;
                const bool in = row < nrow;
                pos[r] = in ? x.r.base + paged_group(a, x.tile * ROWS + row) : -1;
                const uint8_t* qh = a.q + (in ? paged_row_at(a, x.r.first, x.h, x.tile, row, ROWS, a.qs, hb) : 0);
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    uint4 v = make_uint4(0u, 0u, 0u, 0u);
                    if (in) v = paged_q8x(qh, a.io, 32 * c + 8 * t);
                    qa[2 * c][r] = v.x;
                    qa[2 * c][2 + r] = v.y;
                    qa[2 * c + 1][r] = v.z;
                    qa[2 * c + 1][2 + r] = v.w;
                }
            }
            if (!R16) {
#pragma unroll
                for (int i = 0; i < 2 * NC; ++i) qa[i][1] = qa[i][3] = 0u;
            }
        }
        float o[NO][4], m[NR], l[NR];
#pragma unroll
        for (int j = 0; j < NO; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[j][i] = 0.0f;
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.0f;
        }
        // keys [0, full_hi] from full_lo on (or below n_sink) are seen by every row of the tile
        const int full_lo = a.window > 0 ? max(0, x.t.phi - a.window + 1) : 0, full_hi = x.t.plo;

        for (int u = u0; u < u1; ++u) {
            fetch();
            asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 1) : "memory");
            __syncwarp();
            const uint32_t sk = ring + slot * C::STAGE, sv = sk + KEYS * RB, sd = sk + 2 * KEYS * RB;
            slot = slot + 1 == C::STAGES ? 0 : slot + 1;
            const int kb = paged_unit_key<KEYS>(x.t, u);
            const bool full = kb + KEYS - 1 <= full_hi && (kb >= full_lo || kb + KEYS <= a.n_sink);

            uint32_t pa[NH][Q ? NC : 1][4];  // weight fragments of 16 keys (Q8: times the deltas of V's block c)
            bool mixed = false;              // some row sees a key of this step that another does not
            if constexpr (ONE) {
                constexpr int KPL = KEYS / 32;  // keys per lane
                float sc[KPL];
                float mx = -INFINITY;
#pragma unroll
                for (int k = 0; k < KPL; ++k) {
                    const int kr = lane + 32 * k, key = kb + kr;
                    const uint2 dw = D == 64 ? make_uint2(lds4(sd + kr * 4), 0u) : lds8(sd + kr * 8);
                    float v = 0.0f;
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        int hi = 0, lo = 0;
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const int ch = 2 * c + j;
                            const uint4 f = lds16(sk + kr * RB + ((ch ^ (D == 64 ? (kr >> 1) & 3 : kr & 7)) << 4));
                            const uint32_t w[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                hi = dp4a((int)w[i], (int)qhi[4 * ch + i], hi);
                                if (has_lo) lo = dp4a((int)w[i], (int)qlo[4 * ch + i], lo);
                            }
                        }
                        const float d = h2f((uint16_t)((c < 2 ? dw.x : dw.y) >> (16 * (c & 1))));
                        v = fmaf((float)(has_lo ? (hi << 8) + lo : hi) * qsc[c], d, v);
                    }
                    const bool see = full || (key <= pos[0] && (a.window == 0 || key > pos[0] - a.window || key < a.n_sink));
                    sc[k] = see ? v * a.scale_log2 : -INFINITY;
                    mx = fmaxf(mx, sc[k]);
                }
                // the maximum as an order-preserving integer
                const uint32_t ub = __float_as_uint(mx);
                const uint32_t mk = __reduce_max_sync(0xffffffffu, (ub & 0x80000000u) ? ~ub : (ub | 0x80000000u));
                mx = __uint_as_float((mk & 0x80000000u) ? (mk ^ 0x80000000u) : ~mk);
                const float mn = fmaxf(m[0], mx), ms = mn == -INFINITY ? 0.0f : mn;
                if (mn > m[0]) {
                    const float f = ex2(m[0] - ms);
                    l[0] *= f;
#pragma unroll
                    for (int j = 0; j < NO; ++j) {
                        o[j][0] *= f;
                        o[j][1] *= f;
                    }
                    m[0] = mn;
                }
                __syncwarp();  // K is read: its place takes the weights, as the fragments want them
#pragma unroll
                for (int k = 0; k < KPL; ++k) {
                    const int kr = lane + 32 * k;
                    const float e = ex2(sc[k] + (PD_BIAS - ms));
                    l[0] += e;
                    const uint2 dw = D == 64 ? make_uint2(lds4(sd + C::DELTA + kr * 4), 0u) : lds8(sd + C::DELTA + kr * 8);
                    const int te = (int)(C::INVERSE >> (4 * (kr & 7))) & 7;  // 2 t + e of this key among its 8
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        // a hidden key's delta may hold anything: its weight is zero whatever it is
                        const float y = sc[k] == -INFINITY ? 0.0f : e * h2f((uint16_t)((c < 2 ? dw.x : dw.y) >> (16 * (c & 1))));
                        const uint32_t at = sk + ((((c * 4 + (te >> 1)) * NH + (kr >> 4)) * 2 + ((kr >> 3) & 1)) * 2 + (te & 1)) * 2;
                        asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(f2h(y)) : "memory");
                    }
                }
                __syncwarp();
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int i = 0; i < NH / 2; ++i) {
                        const uint4 v = lds16(sk + (c * 4 + t) * NH * 8 + 16 * i);
                        pa[2 * i][c][0] = g == 0 ? v.x : 0u;
                        pa[2 * i][c][2] = g == 0 ? v.y : 0u;
                        pa[2 * i + 1][c][0] = g == 0 ? v.z : 0u;
                        pa[2 * i + 1][c][2] = g == 0 ? v.w : 0u;
                    }
            } else {
                // ---- scores
                float sc[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc[n][i] = 0.0f;
                    const uint32_t row = sk + n * 8 * (Q ? RB : 128);
                    if (!Q) {
#pragma unroll
                        for (int c = 0; c < NC; ++c) {
                            const uint4 f = lds16(row + chunk(koff, c));
                            mma_16816(sc[n], qa[2 * c], f.x, f.y);
                            mma_16816(sc[n], qa[2 * c + 1], f.z, f.w);
                        }
                    } else {
                        // deltas of keys p0 and p1: NC halves each
                        uint2 w0, w1;
                        if (D == 64) {
                            w0.x = lds4(sd + (8 * n + p0) * 4);
                            w1.x = lds4(sd + (8 * n + p1) * 4);
                        } else {
                            w0 = lds8(sd + (8 * n + p0) * 8);
                            w1 = lds8(sd + (8 * n + p1) * 8);
                        }
#pragma unroll
                        for (int c = 0; c < NC; ++c) {
                            float blk[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            const uint2 f = lds8(row + chunk(koff, c));
                            const uint2 lo = tc_bytes_to_f16x4(f.x ^ 0x80808080u, 0x64806480u);
                            const uint2 hi = tc_bytes_to_f16x4(f.y ^ 0x80808080u, 0x64806480u);
                            mma_16816(blk, qa[2 * c], lo.x, lo.y);
                            mma_16816(blk, qa[2 * c + 1], hi.x, hi.y);
                            const float d0 = h2f((uint16_t)((c < 2 ? w0.x : w0.y) >> (16 * (c & 1))));
                            const float d1 = h2f((uint16_t)((c < 2 ? w1.x : w1.y) >> (16 * (c & 1))));
#pragma unroll
                            for (int r = 0; r < NR; ++r) {
                                sc[n][2 * r] = fmaf(blk[2 * r], d0, sc[n][2 * r]);
                                sc[n][2 * r + 1] = fmaf(blk[2 * r + 1], d1, sc[n][2 * r + 1]);
                            }
                        }
                    }
                }
                if (!full) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int key = kb + 8 * n + (e ? p1 : p0);
#pragma unroll
                            for (int r = 0; r < NR; ++r) {
                                const bool see = key <= pos[r] && (a.window == 0 || key > pos[r] - a.window || key < a.n_sink);
                                if (!see) sc[n][2 * r + e] = -INFINITY;
                            }
                        }
                    mixed = x.t.plo != x.t.phi;
                }

                // ---- softmax: running maximum and sum per row, in base 2
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    float mx = sc[0][2 * r];
#pragma unroll
                    for (int n = 0; n < NT; ++n) mx = fmaxf(mx, fmaxf(sc[n][2 * r], sc[n][2 * r + 1]));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    const float mn = fmaxf(m[r], mx * a.scale_log2), ms = mn == -INFINITY ? 0.0f : mn;
                    if (__any_sync(0xffffffffu, mn > m[r])) {
                        const float f = ex2(m[r] - ms);
                        l[r] *= f;
#pragma unroll
                        for (int j = 0; j < NO; ++j) {
                            o[j][2 * r] *= f;
                            o[j][2 * r + 1] *= f;
                        }
                        m[r] = mn;
                    }
                    float sum = 0.0f;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float e0 = ex2(fmaf(sc[n][2 * r], a.scale_log2, PD_BIAS - ms));
                        const float e1 = ex2(fmaf(sc[n][2 * r + 1], a.scale_log2, PD_BIAS - ms));
                        sum += e0 + e1;
                        const int s = n >> 1, at = r + 2 * (n & 1);
                        if (!Q) {
                            pa[s][0][at] = pack_f16(e0, e1);
                        } else {
                            uint2 w0, w1;
                            if (D == 64) {
                                w0.x = lds4(sd + C::DELTA + (8 * n + p0) * 4);
                                w1.x = lds4(sd + C::DELTA + (8 * n + p1) * 4);
                            } else {
                                w0 = lds8(sd + C::DELTA + (8 * n + p0) * 8);
                                w1 = lds8(sd + C::DELTA + (8 * n + p1) * 8);
                            }
#pragma unroll
                            for (int c = 0; c < NC; ++c) {
                                float y0 = e0 * h2f((uint16_t)((c < 2 ? w0.x : w0.y) >> (16 * (c & 1))));
                                float y1 = e1 * h2f((uint16_t)((c < 2 ? w1.x : w1.y) >> (16 * (c & 1))));
                                // a hidden key's delta may hold anything: its weight is zero whatever it is
                                if (!full) {
                                    y0 = sc[n][2 * r] == -INFINITY ? 0.0f : y0;
                                    y1 = sc[n][2 * r + 1] == -INFINITY ? 0.0f : y1;
                                }
                                pa[s][c][at] = pack_f16(y0, y1);
                            }
                        }
                    }
                    l[r] += sum;
                }
            }
            if (!R16) {
#pragma unroll
                for (int s = 0; s < NH; ++s)
#pragma unroll
                    for (int c = 0; c < (Q ? NC : 1); ++c) pa[s][c][1] = pa[s][c][3] = 0u;
            }

            // ---- O += P V; with `tok` >= 0 only the keys that this token sees
            auto pv = [&](float (&acc)[NO][4], int tok) {
#pragma unroll
                for (int s = 0; s < NH; ++s) {
                    if (!Q) {
                        bool h[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int key = kb + 16 * s + 8 * (i >> 1) + ((i & 1) ? p1 : p0);
                            h[i] = tok >= 0 && (key > tok || (a.window > 0 && key <= tok - a.window && key >= a.n_sink));
                        }
#pragma unroll
                        for (int c = 0; c < NC / 2; ++c) {
                            const uint32_t at = sv + c * (KEYS * 128) + s * 2048;
                            const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
                            const uint4 v0 = h[0] ? zero : lds16(at + voff0), v1 = h[1] ? zero : lds16(at + voff1);
                            const uint4 v2 = h[2] ? zero : lds16(at + 1024 + voff0), v3 = h[3] ? zero : lds16(at + 1024 + voff1);
                            const uint32_t w0[4] = {v0.x, v0.y, v0.z, v0.w}, w1[4] = {v1.x, v1.y, v1.z, v1.w};
                            const uint32_t w2[4] = {v2.x, v2.y, v2.z, v2.w}, w3[4] = {v3.x, v3.y, v3.z, v3.w};
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                mma_16816(acc[8 * c + 2 * j], pa[s][0], __byte_perm(w0[j], w1[j], 0x5410),
                                          __byte_perm(w2[j], w3[j], 0x5410));
                                mma_16816(acc[8 * c + 2 * j + 1], pa[s][0], __byte_perm(w0[j], w1[j], 0x7632),
                                          __byte_perm(w2[j], w3[j], 0x7632));
                            }
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < NC; ++c) {
                            const uint32_t at = sv + s * 16 * RB;
                            const uint32_t w0 = lds4(at + chunk(voff0, c)), w1 = lds4(at + chunk(voff1, c));
                            const uint32_t w2 = lds4(at + 8 * RB + chunk(voff0, c)), w3 = lds4(at + 8 * RB + chunk(voff1, c));
#pragma unroll
                            for (int hi = 0; hi < 2; ++hi) {
                                const uint2 b0 = pair_bytes(w0, w1, hi), b1 = pair_bytes(w2, w3, hi);
                                mma_16816(acc[4 * c + 2 * hi], pa[s][c], b0.x, b1.x);
                                mma_16816(acc[4 * c + 2 * hi + 1], pa[s][c], b0.y, b1.y);
                            }
                        }
                    }
                }
            };
            bool odd = false;  // fp16 values that are not finite where rows differ in what they see
            if (!Q && mixed) {
                for (int i = lane; i < KEYS * RB / 16; i += 32) {
                    const uint4 f = lds16(sv + i * 16);
                    const uint32_t w[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) odd |= (w[j] & 0x7c00u) == 0x7c00u || (w[j] & 0x7c000000u) == 0x7c000000u;
                }
                odd = __any_sync(0xffffffffu, odd);
            }
            if (!odd) {
                pv(o, -1);
            } else {
                // weight 0 times NaN or infinity must not reach the rows that do not see the key: once per
                // token, with only that token's keys of V, kept for that token's rows
                for (int tok = max(0, x.t.plo); tok <= x.t.phi; ++tok) {
                    float tmp[NO][4];
#pragma unroll
                    for (int j = 0; j < NO; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) tmp[j][i] = o[j][i];
                    pv(tmp, tok);
#pragma unroll
                    for (int j = 0; j < NO; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (pos[R16 ? i >> 1 : 0] == tok) o[j][i] = tmp[j][i];
                }
            }
            __syncwarp();  // the stage is read: the next fetch may fill it
        }

        // ---- the item, or its part: lane (g, t) holds columns 32 b + 8 t .. + 7 of its rows
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            float ll = l[r];
#pragma unroll
            for (int i = 1; i < (ONE ? 32 : 4); i <<= 1) ll += __shfl_xor_sync(0xffffffffu, ll, i);
            const int row = g + 8 * r;
            const bool live = row < nrow, done = u0 == 0 && u1 == x.t.units;
            float* ps = a.part + (2L * (int)me + (u0 == 0)) * paged_slot<ROWS, D>();
            uint8_t* dst = a.out + (live ? paged_row_at(a, x.r.first, x.h, x.tile, row, ROWS, a.os, hb) : 0);
            const float inv = ll != 0.0f ? 1.0f / ll : 0.0f;
#pragma unroll
            for (int b = 0; b < NC; ++b) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[e] = Q ? o[4 * b + (e & 3)][2 * r + (e >> 2)] : o[8 * (b >> 1) + e][2 * r + (b & 1)];
                if (done) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = ll != 0.0f ? v[e] * inv : 0.0f;
                    paged_store<8>(dst, a.io, 32 * b + 8 * t, v, live);
                } else if (live) {
                    float4* q4 = reinterpret_cast<float4*>(ps + row * D + 32 * b + 8 * t);
                    q4[0] = make_float4(v[0], v[1], v[2], v[3]);
                    q4[1] = make_float4(v[4], v[5], v[6], v[7]);
                }
            }
            if (!done && live && t == 0) {
                ps[ROWS * D + row] = m[r];
                ps[ROWS * (D + 1) + row] = ll;
            }
        }
        if (u0 == 0 && u1 < x.t.units && lane == 0)
            a.join[me] = PagedJoin{(int)((x.start + (unsigned)x.t.units - 1) / share), x.r.first, x.h, x.tile, nrow};
        left -= u1 - u0;
        if (left > 0) paged_next<ROWS, KEYS>(a, p, x);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (p.chained) pdl_wait();
}

}  // namespace gtn
