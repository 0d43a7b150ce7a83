// Paged attention for chunks of new tokens: bound by the matrix products and the exponentials.
//
// A worker (paged_sched.cuh) is a CTA, one per SM; an item is 256 query rows (two tiles of 128, the rows of
// one kv head's query heads packed token by token, so that K and V are read once for all of them), a unit 128
// keys, taken in halves of 64. S = Q K^T and O += P V run on tcgen05 with S (128 fp32 columns per tile), P (fp16, in
// S's place) and O in TMEM; one thread owns a query row, so that the softmax needs no exchange between threads. Four
// softmaxes are on their way (two tiles, two halves): while one half's scores are turned into weights, the tensor
// cores work for the others.
//
// Roles, which meet only at mbarriers:
//   warps 0-3, 4-7  softmax of tile 0, 1: read S, running maximum and sum, write P; rescale O when the maximum
//                   has grown by more than 2^CH_GROW (until then the old one serves, the weights stay below
//                   2^(CH_BIAS + CH_GROW) < 65504); load Q before an item and write O behind it. Weights round to fp16
//                   once (2^-11 relative), their sum is taken before that, in fp32;
//   warp 8          issues the MMAs: P V of unit u half by half, behind each the next scores that may go in its place;
//   warps 9-11      K and V. fp16 cache: warp 9 fetches pages with TMA (128-byte swizzle), warps 10 and 11
//                   look at the V tiles that not every row sees whole (below). Q8 cache: warp 9 copies the pages'
//                   bytes into shared memory, two groups ahead, and all three write the tiles as fp16: an element
//                   value * delta has up to 18 bits, so it is two fp16 values, the rounded product and the rest, each
//                   in a tile of its own, and every product runs over both. (Rounded once instead, K and V each add as
//                   much error as the output's own rounding: 5.2e-4 in all against 2.8e-4, for 106 us against 117.)
// Keys that a row does not see get weight 0, but 0 times NaN or infinity would reach the row all the same. So
// in the tiles that not every row sees whole, values that no row sees are zeroed in shared memory, and
// non-finite ones that some row sees are too, with a note of the item on which its epilogue adds them, read from the
// pages again, to the rows that see them (some milliseconds at most, far below the waits' bound).
// Every wait is bounded as in gemm_tc.cuh.
//
// Measured (graph replay, B200): 2,048 tokens over 29,999 keys, 32/8 heads of 128, fp16: 1,100 us, 945 TFLOP/s, 57% of
// the library product's rate: tensor cores and exponentials are both active 56% of the time, in turns, so that neither is
// the bound by itself. Window chunks (D = 64): 126 us, 330 TFLOP/s; the visible pairs' exponentials are some 36 us of it (16 per
// cycle and SM), keys that units hold and rows do not see come on top (halves end at the causal limit, but begin at
// the unit in which the window does, and a few first tokens cost a unit); what the rest waits for is not separated yet. Q8
// prompts: 117 us; the conversion of the pages (some 350 cycles per 512 elements and warp: 3,700 a unit, against 2,048 of
// exponentials) is less than half of it, and the rest is not separated either. A call of a few units per CTA is bound by
// the code's first run: 7,500 cycles to the first product, 5,500 behind an item.
// One query row per thread and 384 threads leave 168 registers each; four softmax warpgroups (two threads a row) spilled
// and were slower, as were more CTAs with smaller tiles.
#pragma once
#include "paged_decode.cuh"

namespace gtn {

constexpr int CH_THREADS = 384;
constexpr int CH_ROWS = 256;
constexpr int CH_KEYS = 128;
constexpr float CH_BIAS = 7.0f;
// Rescaling only when the maximum has grown past a threshold, instead of at every new one, is a published method of
// fused attention for this GPU generation; the threshold is set by the weights' type: 2^(CH_BIAS + CH_GROW) < 65504.
constexpr float CH_GROW = 8.0f;

template <int DT, int D>
struct ChunkCfg {
    static constexpr int TILE = 128 * D * 2;  // bytes of a Q, K or V tile
    static constexpr bool Q8 = DT == GTN_Q8;
    // Stages of K and V in flight. A Q8 element is two fp16 values (rounded product, rest) in two tiles of a stage.
    static constexpr int KS = D == 64 ? (Q8 ? 2 : 3) : Q8 ? 1 : 2, VS = KS;
    static constexpr int PARTS = Q8 ? 2 : 1, STG = PARTS * TILE;
    // Q8 pages' bytes on their way: groups of GH 64-key halves of a unit's four (K, K, V, V), two groups; a half is
    // 64 rows of 8-bit values, then their deltas
    static constexpr int GH = D == 64 ? 4 : 1;
    static constexpr int RAW = 64 * (D + D / 16), RAWS = Q8 ? 2 * GH * RAW : 0;
    static constexpr int STAGE = 32 * 32;  // bytes per softmax warp: 32 rows x 16 fp16 outputs on their way out
    static constexpr int OUT = 2 * TILE + (KS + VS) * STG, RAW0 = OUT + 8 * STAGE;  // offsets
    static constexpr int SMEM = 1024 + RAW0 + RAWS;
    static constexpr int COL_O = 256;  // TMEM columns: S0, S1 at 0 and 128; O0, O1 at 256 and 256 + D
    // Keys per score product. 64: the next unit's scores of a half start as soon as the half's weights are
    // used, so the softmax does not wait for them. But at N = 64 the operands (Q again for every half) come out
    // of shared memory slower than the product runs, which costs where the products or the shared memory are the
    // bound: one product over both halves at D = 128 (30,000-key chunk: 1144 us against 1284 with halves) and for
    // Q8 pages (prompts 117 us against 119); halves for fp16 at D = 64 (window chunks 164 us against 181).
    static constexpr int SN = D == 64 && !Q8 ? 64 : 128;
    // kind::f16, A = B = fp16, D = fp32; scores: both K-major, N = SN; output: B (V) MN-major, N = D
    static constexpr uint32_t IDESC_S = (1u << 4) | (((uint32_t)SN >> 3) << 17) | ((128u >> 4) << 24);
    static constexpr uint32_t IDESC_O = (1u << 4) | (1u << 16) | (((uint32_t)D >> 3) << 17) | ((128u >> 4) << 24);
};

// Matrix descriptors of tiles of 128-byte rows in the 128-byte swizzle (8-row groups of 1024 bytes). K-major
// (Q, K: a row holds 64 elements of d): stride between row groups. MN-major (V: a row holds 64 columns of one
// key): stride between groups of 8 keys, and between 64-column halves.
__device__ __forceinline__ uint64_t ch_desc(uint32_t saddr, uint32_t lbo) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) | ((uint64_t)(1024u >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// Called by a whole converged warp, done by its `leader` lane: so all operands are warp-uniform and stay in
// uniform registers (issued from a divergent lane, each MMA cost some 85 cycles of register moves, more than it
// runs).
__device__ __forceinline__ void ch_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate,
                                          uint32_t leader) {
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
}
// A in TMEM.
__device__ __forceinline__ void ch_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate,
                                          uint32_t leader) {
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void ch_commit(uint64_t* bar, uint32_t leader) {
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
        " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar)),
        "r"(leader)
        : "memory");
}
__device__ __forceinline__ uint32_t ch_elect() {
    uint32_t r;
    asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n selp.u32 %0, 1, 0, e;\n}\n" : "=r"(r));
    return r;
}
#define CH_R8(a, i) "=r"(a[i]), "=r"(a[i + 1]), "=r"(a[i + 2]), "=r"(a[i + 3]), "=r"(a[i + 4]), "=r"(a[i + 5]), "=r"(a[i + 6]), "=r"(a[i + 7])
#define CH_U8(a, i) "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3]), "r"(a[i + 4]), "r"(a[i + 5]), "r"(a[i + 6]), "r"(a[i + 7])
#define CH_W8(a, i) "+r"(a[i]), "+r"(a[i + 1]), "+r"(a[i + 2]), "+r"(a[i + 3]), "+r"(a[i + 4]), "+r"(a[i + 5]), "+r"(a[i + 6]), "+r"(a[i + 7])
// 32 consecutive TMEM columns of the thread's lane; valid after ch_wait_ld, which names the registers.
__device__ __forceinline__ void ch_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
        : CH_R8(r, 0), CH_R8(r, 8), CH_R8(r, 16), CH_R8(r, 24)
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void ch_wait_ld(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n" : CH_W8(r, 0), CH_W8(r, 8), CH_W8(r, 16), CH_W8(r, 24) : : "memory");
}
__device__ __forceinline__ void ch_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};\n" ::"r"(taddr),
        CH_U8(r, 0), CH_U8(r, 8), CH_U8(r, 16), CH_U8(r, 24)
        : "memory");
}
__device__ __forceinline__ void ch_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16};\n" ::"r"(taddr),
        CH_U8(r, 0), CH_U8(r, 8)
        : "memory");
}
__device__ __forceinline__ void ch_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 3-D TMA tile load (no multicast): box (x, y, z) of a pool of pages; boxes outside it read as zeros.
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

// Pairs of fp32 in one 64-bit register (packed multiply-add and add).
__device__ __forceinline__ uint64_t f2_pack(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 f2_get(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {  // NaN if any is
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// Untiled bulk copy (16-byte aligned, a multiple of 16 bytes), counted on `bar`.
__device__ __forceinline__ void ch_bulk(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
        "r"(bytes), "r"(smem_u32(bar))
        : "memory");
}

struct ChunkSmem {
    uint64_t k_full[3], k_empty[3], v_load[3], v_full[3], v_empty[3];
    uint64_t raw_full[2], raw_empty[2];  // Q8: per group of halves
    uint64_t q_full[2], s_full[2][2], p_full[2][2], pv_done[2], o_full[2], drain;  // s, p: per tile and 64-key half
    uint32_t tmem;
    volatile int abort;
    unsigned odd;  // 1 + the start (on the line) of the last item of which a non-finite value was set aside; 0: none
    unsigned pre[CH_THREADS], wsum[CH_THREADS / 32];
};

// Keys [kb, kb + nk) that every row of the positions plo .. phi sees.
__device__ __forceinline__ bool ch_whole(const PagedAttnArgs& a, int kb, int nk, int plo, int phi) {
    const int lo = a.window > 0 ? max(0, phi - a.window + 1) : 0;
    return kb + nk - 1 <= plo && (kb >= lo || kb + nk <= a.n_sink);
}

// Adds the values that were set aside (non-finite) to a row's columns c0 .. c0 + 15, as far as it sees them: those of
// the units that not every row sees whole, at most some 256 + 2 * 128 keys at each end of the window and the first
// tokens' last unit, however long the item is.
static __device__ __noinline__ void ch_add_odd(const PagedAttnArgs& a, const PagedPos& x, int u0, int u1, int pos, int wlo,
                                               int c0, float (&v)[16]) {
    for (int u = u0; u < u1; ++u) {
        const int kb = paged_unit_key<CH_KEYS>(x.t, u);
        if (ch_whole(a, kb, CH_KEYS, x.t.plo, x.t.phi)) continue;  // (nothing of it was set aside)
        for (int key = kb; key < kb + CH_KEYS && key <= pos; ++key) {
            if (key < wlo && key >= a.n_sink) continue;
            const int page = a.table[x.b * a.table_stride + (key >> a.c.ps_shift)];
            if ((unsigned)page >= (unsigned)a.c.n_pages) continue;
            const uint8_t* pg = a.c.v + (long)page * a.c.page_stride;
            for (int j = 0; j < 16; ++j) {
                const float y = paged_elem(a.c, pg, x.h, key & (a.c.ps - 1), c0 + j);
                if (!(fabsf(y) < INFINITY)) v[j] += y;
            }
        }
    }
}

// Q8 queries and outputs, out of line: seldom code beside the loops costs instruction cache.
static __device__ __noinline__ uint4 ch_q8_query(const PagedAttnArgs& a, const PagedPos& x, int row, int e0, int d) {
    return paged_q8x(a.q + paged_row_at(a, x.r.first, x.h, x.tile, row, CH_ROWS, a.qs, row_bytes(GTN_Q8, d)), GTN_Q8, e0);
}
template <int D>
static __device__ __noinline__ void ch_q8_rows(const PagedAttnArgs& a, const PagedPos& x, int row, bool live, bool any,
                                               bool odd, uint32_t to, float inv, int u0, int u1, int pos, int wlo) {
    uint8_t* blk = a.out + (live ? paged_row_at(a, x.r.first, x.h, x.tile, row, CH_ROWS, a.os, row_bytes(GTN_Q8, D)) : 0);
#pragma unroll 1
    for (int c = 0; c < D; c += 32, blk += GTN_Q8_BYTES) {
        float v[32];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t o[16];
            float y[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = 0u;
            if (any) {
                tc_ld16(to + c + 16 * h, o);
                tc_wait_ld(o);
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) y[j] = __uint_as_float(o[j]);
            if (odd) ch_add_odd(a, x, u0, u1, pos, wlo, c + 16 * h, y);
#pragma unroll
            for (int j = 0; j < 16; ++j) v[16 * h + j] = y[j] * inv;
        }
        // the activation quantizer (warp_quant_block)
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; ++i) m = fmaxf(m, fabsf(v[i]));
        const float delta = m / 127.0f, iv = delta != 0.0f ? 1.0f / delta : 0.0f;
        if (!live) continue;
        *reinterpret_cast<uint16_t*>(blk) = f2h(delta);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t lo = (uint8_t)(int8_t)roundf(v[2 * i] * iv), hi = (uint8_t)(int8_t)roundf(v[2 * i + 1] * iv);
            reinterpret_cast<uint16_t*>(blk + 2)[i] = (uint16_t)(lo | (hi << 8));
        }
    }
}

template <int DT, int D>
__global__ void __launch_bounds__(CH_THREADS, 1)
    k_paged_chunk(const __grid_constant__ PagedAttnArgs a, const __grid_constant__ PagedPick p, const __grid_constant__ CUtensorMap kmap,
                  const __grid_constant__ CUtensorMap vmap, int box) {
    using C = ChunkCfg<DT, D>;
    constexpr bool Q8 = DT == GTN_Q8;
    constexpr int HALVES = D / 64, HALF = 128 * 128;  // 64-column halves of a tile, bytes of one
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ ChunkSmem sm;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t sq = base, sk = sq + 2 * C::TILE, sv = sk + C::KS * C::STG;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)),
                     "r"(TC_TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (int s = 0; s < 3; ++s) {
            mbar_init(&sm.k_full[s], Q8 ? 3 : 1);
            mbar_init(&sm.k_empty[s], 1);
            mbar_init(&sm.v_load[s], 1);
            mbar_init(&sm.v_full[s], Q8 ? 3 : 2);
            mbar_init(&sm.v_empty[s], 1);
        }
        for (int r = 0; r < 2; ++r) {
            mbar_init(&sm.q_full[r], 128);
            for (int b = 0; b < 2; ++b) {
                mbar_init(&sm.s_full[r][b], 1);
                mbar_init(&sm.p_full[r][b], 128);
            }
            mbar_init(&sm.pv_done[r], 1);
            mbar_init(&sm.o_full[r], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.raw_full[i], C::GH);
            mbar_init(&sm.raw_empty[i], 3);
        }
        mbar_init(&sm.drain, 1);
        sm.abort = 0;
        sm.odd = 0;
        fence_mbar_init();
    }
    pdl_wait();
    pdl_trigger();
    const int me = blockIdx.x;
    if (tid == 0) a.join[me].last = -1;
    tc_fence_before();
    const unsigned total = paged_sched<CH_ROWS, CH_KEYS, CH_THREADS, true>(a, p, me == 0, sm.pre, sm.wsum);
    tc_fence_after();
    const uint32_t tmem = sm.tmem;
    const unsigned share = paged_share(total, a.workers_mul);
    PagedPos x{};
    int left = 0;
    if (share * (unsigned)me < total) {
        x = paged_locate<CH_ROWS, CH_KEYS, CH_THREADS, true>(a, p, share * (unsigned)me, sm.pre);
        left = (int)min(total - share * (unsigned)me, share);
    }

    // 64-key halves of units [u0, u1) that some row of row tile r sees to the causal limit: the first so many
    auto tile_halves = [&](int r, int u0, int u1) {
        const int m1 = min(x.r.n * a.group, x.tile * CH_ROWS + (r + 1) * 128) - 1;  // the tile's last row
        if (m1 < x.tile * CH_ROWS + r * 128) return 0;
        const int phi = x.r.base + paged_group(a, m1);
        if (phi < 0) return 0;
        // keys ascend: sink halves q < 2 ns hold keys 64 q, the others 64 (2 w0 + q - 2 ns)
        int n = min(2 * x.t.ns, phi / 64 + 1);
        if (n == 2 * x.t.ns) n += max(0, phi / 64 - 2 * x.t.w0 + 1);
        return max(0, min(2 * u1, n) - 2 * u0);
    };
    // by a whole warp; false once a wait of the CTA has run out
    auto wait = [&](uint64_t* bar, uint32_t ph) {
        bool got = mbar_try_wait(bar, ph);
        if (!__all_sync(0xffffffffu, got)) {
            got = got || (sm.abort == 0 && tc_wait(bar, ph, a.err));
            if (!__all_sync(0xffffffffu, got)) {
                sm.abort = 1;
                return false;
            }
        }
        return true;
    };
    auto seen_whole = [&](int kb) { return ch_whole(a, kb, CH_KEYS, x.t.plo, x.t.phi); };
    auto next_item = [&](int done) {
        left -= done;
        if (left > 0) paged_next<CH_ROWS, CH_KEYS>(a, p, x);
    };

    if (warp < 8) {
        // ---- softmax of tile r
        const int r = warp >> 2, row = tid & 127;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t ts = lanes + r * 128, to = lanes + C::COL_O + r * D;
        const uint32_t qs = sq + r * C::TILE;
        const long hb = row_bytes(a.io, D);
        uint32_t s_ph = 0, o_ph = 0, pvn = 0;  // phases (s_full: a bit per half); halves handed to P V so far
        bool ok = true;
        // The row's query into the swizzled tile. Not for a tile without units: its softmax waits for nothing
        // and could pass q_full twice before the MMA warp looks.
        auto load_q = [&]() {
            if (tile_halves(r, x.u, min(x.t.units, x.u + left)) == 0) return;
            // D / 8 adjacent lanes per row
            constexpr int CPR = D / 8;
            const int c = lane % CPR;
            const int m0 = x.tile * CH_ROWS + r * 128 + (warp & 3) * 32 + lane / CPR, m1 = x.r.n * a.group;
            const int l0 = (warp & 3) * 32 + lane / CPR;  // the lane's first row of the tile
            if (a.io == GTN_F16) {
#pragma unroll 1
                for (int i = 0; i < 32; i += 4 * (32 / CPR)) {
                    uint4 v[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int m = m0 + i + k * (32 / CPR), tok = paged_group(a, m);
                        v[k] = make_uint4(0u, 0u, 0u, 0u);
                        if (m < m1)
                            v[k] = *reinterpret_cast<const uint4*>(a.q + (long)(x.r.first + tok) * a.qs +
                                                                   (x.h * a.group + m - tok * a.group) * (D * 2) + 16 * c);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int rw = l0 + i + k * (32 / CPR);
                        const uint32_t dst = qs + (c >> 3) * HALF + rw * 128 + (((c & 7) ^ (rw & 7)) << 4);
                        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v[k].x), "r"(v[k].y),
                                     "r"(v[k].z), "r"(v[k].w)
                                     : "memory");
                    }
                }
            } else {
#pragma unroll 1
                for (int i = 0; i < 32; i += 32 / CPR) {
                    const int rw = l0 + i;
                    const uint4 v = m0 + i < m1 ? ch_q8_query(a, x, r * 128 + rw, 8 * c, D) : make_uint4(0u, 0u, 0u, 0u);
                    const uint32_t dst = qs + (c >> 3) * HALF + rw * 128 + (((c & 7) ^ (rw & 7)) << 4);
                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                                 : "memory");
                }
            }
            fence_async_smem();
            mbar_arrive(&sm.q_full[r]);
        };
        if (left > 0) load_q();
        while (left > 0 && ok) {
            const int u0 = x.u, u1 = min(x.t.units, u0 + left), n = tile_halves(r, u0, u1);
            const int m_row = x.tile * CH_ROWS + r * 128 + row;
            const bool live = m_row < x.r.n * a.group;
            const int pos = live ? x.r.base + paged_group(a, m_row) : -1;
            const int wlo = a.window > 0 ? pos - a.window + 1 : 0;
            // positions of this tile's first and last row
            const int t0 = x.tile * CH_ROWS + r * 128;
            const int tlo = x.r.base + paged_group(a, t0), thi = x.r.base + min(x.r.n - 1, paged_group(a, t0 + 127));
            // the maximum in use (base 2; a row behind the item's last needs none), the sum of weights
            float mu = live ? -INFINITY : 0.0f, l = 0.0f;
            for (int q = 0; q < n; ++q) {
                const int b = q & 1;
                if (!(ok = wait(&sm.s_full[r][b], (s_ph >> b) & 1u))) break;
                s_ph ^= 1u << b;
                tc_fence_after();
                const int kb = paged_unit_key<CH_KEYS>(x.t, u0 + (q >> 1)) + 64 * b;
                const uint32_t tb = ts + 64 * b;
                uint32_t v[2][32];
                ch_ld32(tb, v[0]);
                ch_ld32(tb + 32, v[1]);
                const bool whole = ch_whole(a, kb, 64, tlo, thi);
                // the keys of chunk i (32) that this row sees, as bits
                auto seen_bits = [&](int i) -> uint32_t {
                    const int k0 = kb + 32 * i;
                    auto below = [](int n) -> uint32_t { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; };
                    uint32_t v = below(pos - k0 + 1);
                    if (a.window > 0) v &= ~below(wlo - k0) | below(a.n_sink - k0);
                    return v;
                };
                auto hide = [](uint32_t (&v)[32], uint32_t bits) {
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (!((bits >> j) & 1u)) v[j] = 0xff800000u;
                };
                ch_wait_ld(v[0]);
                ch_wait_ld(v[1]);
                if (!whole) {
                    const uint32_t b0 = seen_bits(0), b1 = seen_bits(1);
                    if (__any_sync(0xffffffffu, b0 != ~0u)) hide(v[0], b0);
                    if (__any_sync(0xffffffffu, b1 != ~0u)) hide(v[1], b1);
                }
                float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    mx0 = max3_nan(mx0, __uint_as_float(v[0][j]), __uint_as_float(v[0][j + 1]));
                    mx1 = max3_nan(mx1, __uint_as_float(v[1][j]), __uint_as_float(v[1][j + 1]));
                }
                const float mx = max3_nan(mx0, mx1, mx1) * a.scale_log2;
                if (!(mx < INFINITY)) l = __int_as_float(0x7fffffff);  // NaN or +infinity: the row has no softmax
                // the maximum in use moves when the new one lies too far above it; the sums so far follow
                const bool grow = mx > mu + CH_GROW || (mu == -INFINITY && mx > mu);
                if (__any_sync(0xffffffffu, grow)) {
                    const float f = grow ? ex2(mu - mx) : 1.0f;  // 0 when nothing was seen yet
                    if (grow) mu = mx;
                    l *= f;
                    if (q > 0) {
                        // O as of the half before (P V of the one before that is done: these scores came behind it, so
                        // the barrier is at most one phase back)
                        if (!(ok = wait(&sm.pv_done[r], (pvn - 1) & 1u))) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t o[32];
                            ch_ld32(to + 32 * c, o);
                            ch_wait_ld(o);
#pragma unroll
                            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                            ch_st32(to + 32 * c, o);
                        }
                    }
                }
                const float sub = CH_BIAS - (mu == -INFINITY ? 0.0f : mu);
                const uint64_t sc2 = f2_pack(a.scale_log2, a.scale_log2), sub2 = f2_pack(sub, sub);
                uint64_t acc0 = 0, acc1 = 0;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t w[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const uint64_t t =
                            f2_fma(f2_pack(__uint_as_float(v[h][2 * j]), __uint_as_float(v[h][2 * j + 1])), sc2, sub2);
                        float2 e = f2_get(t);
                        e = make_float2(ex2(e.x), ex2(e.y));
                        if (j & 1) acc1 = f2_add(acc1, f2_pack(e.x, e.y));
                        else acc0 = f2_add(acc0, f2_pack(e.x, e.y));
                        w[j] = pack_f16(e.x, e.y);
                    }
                    ch_st16(tb + 16 * h, w);  // over scores that are read
                }
                ch_wait_st();
                tc_fence_before();
                mbar_arrive(&sm.p_full[r][b]);
                ++pvn;
                const float2 h = f2_get(f2_add(acc0, acc1));
                l += h.x + h.y;
            }
            // the next item's queries go in before this item's output comes out: all products with this item's
            // are done (its last scores were seen)
            const PagedPos was = x;
            next_item(u1 - u0);
            if (ok && left > 0) load_q();
            if (ok && n > 0) {
                ok = wait(&sm.o_full[r], o_ph);
                o_ph ^= 1u;
                tc_fence_after();
            }
            if (ok && was.r.n * a.group > was.tile * CH_ROWS + r * 128) {
                const bool done = u0 == 0 && u1 == was.t.units;
                const float inv = l != 0.0f ? 1.0f / l : 0.0f;
                const int prow = r * 128 + row;
                float* ps = a.part + (2L * me + (u0 == 0)) * paged_slot<CH_ROWS, D>();
                const uint32_t stage = sq + C::OUT + warp * C::STAGE;
                const bool odd = n > 0 && sm.odd > was.start;  // of this item, or of one that the copies are ahead at
                if (done && a.io != GTN_F16) {
                    ch_q8_rows<D>(a, was, prow, live, n > 0, odd, to, inv, u0, u1, pos, wlo);
                } else {
                    uint8_t* orow[2];  // the rows whose 16 bytes this lane writes
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int rw = r * 128 + (warp & 3) * 32 + 16 * i + (lane >> 1);
                        orow[i] = done && was.tile * CH_ROWS + rw < was.r.n * a.group
                                      ? a.out + paged_row_at(a, was.r.first, was.h, was.tile, rw, CH_ROWS, a.os, hb) + 16 * (lane & 1)
                                      : nullptr;
                    }
#pragma unroll 1
                    for (int c = 0; c < D; c += 16) {
                        uint32_t o[16];
                        float v[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[j] = 0u;
                        if (n > 0) {
                            tc_ld16(to + c, o);
                            tc_wait_ld(o);
                        }
#pragma unroll
                        for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(o[j]);
                        if (odd) ch_add_odd(a, was, u0, u1, pos, wlo, c, v);
                        if (!done) {
#pragma unroll
                            for (int j = 0; j < 16; ++j) ps[(long)(c + j) * CH_ROWS + prow] = v[j];
                            continue;
                        }
                        // through shared memory, so that two adjacent lanes write 16 columns of a row
                        __syncwarp();
#pragma unroll
                        for (int j = 0; j < 2; ++j)
                            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(
                                             stage + lane * 32 + ((j ^ ((lane >> 2) & 1)) << 4)),
                                         "r"(pack_f16(v[8 * j] * inv, v[8 * j + 1] * inv)),
                                         "r"(pack_f16(v[8 * j + 2] * inv, v[8 * j + 3] * inv)),
                                         "r"(pack_f16(v[8 * j + 4] * inv, v[8 * j + 5] * inv)),
                                         "r"(pack_f16(v[8 * j + 6] * inv, v[8 * j + 7] * inv))
                                         : "memory");
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int lr = 16 * i + (lane >> 1);
                            const uint4 y = lds16(stage + lr * 32 + (((lane & 1) ^ ((lr >> 2) & 1)) << 4));
                            if (orow[i]) *reinterpret_cast<uint4*>(orow[i] + 2 * c) = y;
                        }
                    }
                }
                if (!done && live) {
                    ps[CH_ROWS * D + prow] = mu;
                    ps[CH_ROWS * (D + 1) + prow] = l;
                }
                if (tid == 0 && u0 == 0 && u1 < was.t.units)
                    a.join[me] = PagedJoin{(int)((was.start + (unsigned)was.t.units - 1) / share), was.r.first, was.h, was.tile,
                                           min(CH_ROWS, was.r.n * a.group - was.tile * CH_ROWS)};
            }
        }
    } else {
        if (warp == 8) {
            // ---- MMA issue
            const uint32_t leader = ch_elect(), tm = __shfl_sync(0xffffffffu, tmem, 0);
            const uint32_t q0 = __shfl_sync(0xffffffffu, sq, 0);
            const uint32_t k0 = q0 + 2 * C::TILE, v0 = k0 + C::KS * C::STG;
            int ks = 0, vs = 0;
            uint32_t k_ph = 0, v_ph = 0, q_ph = 0, p_ph = 0;
            bool ok = true;
            // scores of half b of the unit in stage ks, or (b = 0) of both halves; `two`: the second is wanted
            auto qk = [&](int r, int b, bool two) {
                const uint64_t qd = ch_desc(q0 + r * C::TILE, 16), kd = ch_desc(k0 + ks * C::STG + b * 8192, 16);
#pragma unroll
                for (int i = 0; i < C::PARTS * (D / 16); ++i) {
                    const int e = i % (D / 16);
                    const uint32_t off = ((e >> 2) * HALF + (e & 3) * 32) >> 4;
                    ch_mma_ss(tm + r * 128 + b * 64, qd + off, kd + off + (i >= D / 16 ? C::TILE >> 4 : 0), C::IDESC_S, i > 0,
                              leader);
                }
                ch_commit(&sm.s_full[r][b], leader);
                if (C::SN == 128 && two) ch_commit(&sm.s_full[r][1], leader);
            };
            while (left > 0 && ok) {
                const int u0 = x.u, u1 = min(x.t.units, u0 + left), n = u1 - u0;
                const int n0 = tile_halves(0, u0, u1), n1 = tile_halves(1, u0, u1);
                ok = wait(&sm.k_full[ks], k_ph);
                for (int i = 0; i < (C::SN == 64 ? 4 : 2) && ok; ++i) {
                    const int b = i >> 1, r = i & 1, nr = r ? n1 : n0;
                    if (b >= nr) continue;
                    if (b == 0) {
                        ok = wait(&sm.q_full[r], (q_ph >> r) & 1u);
                        q_ph ^= 1u << r;
                        tc_fence_after();
                    }
                    if (ok) qk(r, b, nr > 1);
                }
                for (int u = 0; u < n && ok; ++u) {
                    ch_commit(&sm.k_empty[ks], leader);  // the scores of unit u are issued
                    if (++ks == C::KS) {
                        ks = 0;
                        k_ph ^= 1u;
                    }
                    if (u + 1 < n) ok = wait(&sm.k_full[ks], k_ph);
                    if (ok) ok = wait(&sm.v_full[vs], v_ph);
                    for (int i = 0; i < 4 && ok; ++i) {
                        const int b = i >> 1, r = i & 1, nr = r ? n1 : n0, q = 2 * u + b;
                        if (q >= nr) continue;
                        if (!(ok = wait(&sm.p_full[r][b], (p_ph >> i) & 1u))) break;
                        p_ph ^= 1u << i;
                        tc_fence_after();
                        const uint64_t vd = ch_desc(v0 + vs * C::STG + b * 8192, HALF);
#pragma unroll
                        for (int j = 0; j < 4 * C::PARTS; ++j)
                            ch_mma_ts(tm + C::COL_O + r * D, tm + r * 128 + b * 64 + (j & 3) * 8,
                                      vd + (((j & 3) * 2048 + (j >> 2) * C::TILE) >> 4), C::IDESC_O, q > 0 || j > 0, leader);
                        ch_commit(&sm.pv_done[r], leader);
                        if (C::SN == 64 ? q + 2 < nr : b == 1 && q + 1 < nr) qk(r, C::SN == 64 ? b : 0, q + 2 < nr);
                        if (q + 1 == nr) ch_commit(&sm.o_full[r], leader);
                    }
                    if (!ok) break;
                    ch_commit(&sm.v_empty[vs], leader);
                    if (++vs == C::VS) {
                        vs = 0;
                        v_ph ^= 1u;
                    }
                }
                next_item(n);
            }
            ch_commit(&sm.drain, leader);  // nothing of this CTA is in flight behind this
            tc_wait(&sm.drain, 0, a.err);
        } else if (!Q8 && warp == 9) {
            // ---- fetch of fp16 pages: lane i issues the boxes of piece i (`box` rows) of a unit
            int ks = 0, vs = 0, k_issued = 0, v_issued = 0;
            uint32_t k_ph = 1, v_ph = 1;  // the first use of a stage waits for nothing
            bool ok = true;
            const int pieces = CH_KEYS / box;
            while (left > 0 && ok) {
                const int u0 = x.u, u1 = min(x.t.units, u0 + left);
                for (int u = u0; u < u1; ++u) {
                    const int kb = paged_unit_key<CH_KEYS>(x.t, u), k0 = kb + lane * box;
                    const int lo = a.window > 0 ? max(0, x.t.plo - a.window + 1) : 0;
                    int page = a.c.n_pages;  // outside the pool: zeros
                    if (lane < pieces && k0 <= x.t.phi && (k0 + box - 1 >= lo || k0 < a.n_sink)) {
                        page = a.table[x.b * a.table_stride + (k0 >> a.c.ps_shift)];
                        if ((unsigned)page >= (unsigned)a.c.n_pages) {
                            page = a.c.n_pages;
                            atomicOr(a.err, GTN_DEVERR_PAGE);
                        }
                    }
                    const int yrow = x.h * a.c.ps + (k0 & (a.c.ps - 1));
                    if (!(ok = wait(&sm.k_empty[ks], k_ph))) break;
                    if (lane == 0) mbar_arrive_expect_tx(&sm.k_full[ks], C::TILE);
                    __syncwarp();
                    if (lane < pieces)
                        for (int h = 0; h < HALVES; ++h)
                            tma_load_3d(sk + ks * C::STG + h * HALF + lane * box * 128, &kmap, 64 * h, yrow, page,
                                        &sm.k_full[ks]);
                    ++k_issued;
                    if (++ks == C::KS) {
                        ks = 0;
                        k_ph ^= 1u;
                    }
                    if (!(ok = wait(&sm.v_empty[vs], v_ph))) break;
                    if (lane == 0) mbar_arrive_expect_tx(&sm.v_load[vs], C::TILE);
                    __syncwarp();
                    if (lane < pieces)
                        for (int h = 0; h < HALVES; ++h)
                            tma_load_3d(sv + vs * C::STG + h * HALF + lane * box * 128, &vmap, 64 * h, yrow, page,
                                        &sm.v_load[vs]);
                    ++v_issued;
                    if (++vs == C::VS) {
                        vs = 0;
                        v_ph ^= 1u;
                    }
                }
                next_item(u1 - u0);
            }
            // a wait has run out somewhere: the copies in flight end before the shared memory goes
            if (sm.abort != 0 && lane == 0) {
                for (int i = max(0, k_issued - C::KS); i < k_issued; ++i)
                    tc_wait(&sm.k_full[i % C::KS], (uint32_t)(i / C::KS) & 1u, a.err);
                for (int i = max(0, v_issued - C::VS); i < v_issued; ++i)
                    tc_wait(&sm.v_load[i % C::VS], (uint32_t)(i / C::VS) & 1u, a.err);
            }
            __syncwarp();
        } else if (!Q8) {
            // ---- V tiles that not every row sees whole
            int vs = 0;
            uint32_t v_ph = 0;
            bool ok = true;
            const int ct = tid - 320;
            while (left > 0 && ok) {
                const int u0 = x.u, u1 = min(x.t.units, u0 + left);
                for (int u = u0; u < u1; ++u) {
                    if (!(ok = wait(&sm.v_load[vs], v_ph))) break;
                    const int kb = paged_unit_key<CH_KEYS>(x.t, u);
                    if (!seen_whole(kb)) {
                        const int lo = a.window > 0 ? max(0, x.t.plo - a.window + 1) : 0;
                        for (int i = ct; i < HALVES * 1024; i += 64) {
                            const int key = kb + ((i >> 3) & 127);
                            const uint32_t at = sv + vs * C::STG + i * 16;
                            const bool seen = key <= x.t.phi && (key >= lo || key < a.n_sink);
                            uint4 v = lds16(at);
                            uint32_t w[4] = {v.x, v.y, v.z, v.w};
                            bool change = !seen, bad = false;
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                if (!seen) w[j] = 0u;
                                if ((w[j] & 0x7c00u) == 0x7c00u) { w[j] &= 0xffff0000u; bad = true; }
                                if ((w[j] & 0x7c000000u) == 0x7c000000u) { w[j] &= 0x0000ffffu; bad = true; }
                            }
                            if (change || bad)
                                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]),
                                             "r"(w[2]), "r"(w[3])
                                             : "memory");
                            if (bad) atomicMax(&sm.odd, x.start + 1);
                        }
                        fence_async_smem();
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sm.v_full[vs]);
                    if (++vs == C::VS) {
                        vs = 0;
                        v_ph ^= 1u;
                    }
                }
                next_item(u1 - u0);
            }
        } else {
            // ---- Q8 pages to fp16 tiles. Warp 9 brings the pages' bytes into shared memory, two groups ahead (bulk
            // copies of 16 rows and of their deltas, a lane each); all three convert: a warp takes groups of RPG
            // rows, lane = 16 elements of a row.
            int ks = 0, vs = 0, rs = 0;
            uint32_t k_ph = 1, v_ph = 1, r_ph = 0;
            bool ok = true;
            constexpr int CPR = D / 16, RPG = 32 / CPR, PASS = C::GH == 4 ? 128 : 64;  // PASS: rows converted in a go
            const int lrow = lane / CPR, c16 = lane % CPR, g0 = warp == 9 ? 12 : (warp - 10) * 6, g1 = warp == 9 ? 16 : g0 + 6;
            PagedPos y = x;  // warp 9: the unit whose bytes are asked for next
            int ahead = left, asked = 0, page = -1, cell = 0;
            // lane: half lane / 8 of a group; of its 8, lanes 0-3 copy a 16-key piece's values, 4-7 its deltas
            const bool mine = lane < 8 * C::GH, dl = lane & 4;
            auto half_of = [&]() { return C::GH == 4 ? (lane >> 3) & 3 : asked & 3; };
            auto find_page = [&]() {  // of the next group; looked up a group ahead of its use
                const int lo = a.window > 0 ? max(0, y.t.plo - a.window + 1) : 0;
                const int k0 = paged_unit_key<CH_KEYS>(y.t, y.u) + 64 * (half_of() & 1) + 16 * (lane & 3);
                page = -1;
                cell = y.h * a.c.ps + (k0 & (a.c.ps - 1));  // row among the page's
                if (mine && k0 <= y.t.phi && (k0 + 15 >= lo || k0 < a.n_sink))
                    page = (int)min((unsigned)a.table[y.b * a.table_stride + (k0 >> a.c.ps_shift)], 0x7fffffffu);  // negative: too large
            };
            auto fetch = [&]() {  // the next group
                const int slot = asked & 1, half = half_of();
                if (asked >= 2 && !(ok = wait(&sm.raw_empty[slot], (uint32_t)((asked >> 1) - 1) & 1u))) return;
                if (page >= a.c.n_pages) {
                    page = -1;
                    atomicOr(a.err, GTN_DEVERR_PAGE);
                }
                const uint32_t here = __ballot_sync(0xffffffffu, page >= 0) >> (lane & 24) & 0xfu;
                if (mine && (lane & 7) == 0) mbar_arrive_expect_tx(&sm.raw_full[slot], __popc(here) * 16 * (D + D / 16));
                __syncwarp();
                if (page >= 0) {
                    const long off = (long)page * a.c.page_stride +
                                     (dl ? (long)a.c.kv_heads * a.c.ps * D + cell * (D / 16) : (long)cell * D);
                    ch_bulk(sq + C::RAW0 + (slot * C::GH + (C::GH == 4 ? half : 0)) * C::RAW +
                                (dl ? 64 * D + (lane & 3) * D : (lane & 3) * 16 * D),
                            (half & 2 ? a.c.v : a.c.k) + off, dl ? D : 16 * D, &sm.raw_full[slot]);
                }
                ++asked;
                if (C::GH == 4 || (asked & 3) == 0)
                    if (--ahead > 0 && ++y.u == y.t.units) paged_next<CH_ROWS, CH_KEYS>(a, p, y);
                if (ahead > 0) find_page();
            };
            if (warp == 9 && ahead > 0) find_page();
            if (warp == 9)
                for (int i = 0; i < 2 && ahead > 0 && ok; ++i) fetch();
            while (left > 0 && ok) {
                const int kb = paged_unit_key<CH_KEYS>(x.t, x.u);
                const bool scan = !seen_whole(kb);
                const int lo = a.window > 0 ? max(0, x.t.plo - a.window + 1) : 0;
                const bool all = kb + CH_KEYS - 1 <= x.t.phi && (kb >= lo || kb + CH_KEYS <= a.n_sink);
#pragma unroll 1
                for (int q = 0; q < 2 * (128 / PASS) && ok; ++q) {
                    const int kv = q / (128 / PASS), r0 = PASS == 64 ? 64 * (q & 1) : 0;
                    const bool first = PASS == 128 || !(q & 1), last = PASS == 128 || (q & 1);
                    if (C::GH == 1 || q == 0) ok = wait(&sm.raw_full[rs], r_ph);
                    if (ok && first) ok = kv ? wait(&sm.v_empty[vs], v_ph) : wait(&sm.k_empty[ks], k_ph);
                    if (!ok) break;
                    const uint32_t raw = sq + C::RAW0 + (rs * C::GH + (C::GH == 4 ? 2 * kv : 0)) * C::RAW;
                    const uint32_t tile = kv ? sv + vs * C::STG : sk + ks * C::STG;
                    bool bad = false;
#pragma unroll 1
                    for (int grp = g0; grp < g1; ++grp) {
                        const int hrow = (grp * RPG) % 64 + lrow, row = r0 + grp * RPG + lrow, key = kb + row;
                        const uint32_t src = raw + grp * RPG / 64 * C::RAW;
                        uint4 f = lds16(src + hrow * D + c16 * 16);
                        uint16_t d1;
                        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(d1) : "r"(src + 64 * D + (hrow * (D / 32) + (c16 >> 1)) * 2) : "memory");
                        if (!all && (key > x.t.phi || (key < lo && key >= a.n_sink))) {  // nobody sees it: zeros
                            f = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
                            d1 = 0;
                        }
                        const __half2 d2 = __half2half2(__ushort_as_half(d1));
                        const uint32_t in[4] = {f.x, f.y, f.z, f.w};
                        uint32_t w[8], rest[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const uint2 two = tc_bytes_to_f16x4(in[j >> 1] ^ 0x80808080u, 0x64806480u);
                            const uint32_t one = j & 1 ? two.y : two.x;
                            const __half2 z = *reinterpret_cast<const __half2*>(&one), h = __hmul2(z, d2), e = __hfma2(z, d2, __hneg2(h));
                            w[j] = *reinterpret_cast<const uint32_t*>(&h);
                            rest[j] = *reinterpret_cast<const uint32_t*>(&e);
                        }
                        if ((d1 & 0x7c00u) == 0x7c00u)  // infinity and NaN have no rest
#pragma unroll
                            for (int j = 0; j < 8; ++j) rest[j] = 0u;
                        if (kv && scan) {
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const uint32_t keep = ((w[j] & 0x7c00u) == 0x7c00u ? 0u : 0xffffu) |
                                                      ((w[j] & 0x7c000000u) == 0x7c000000u ? 0u : 0xffff0000u);
                                bad |= keep != 0xffffffffu;
                                w[j] &= keep;
                                rest[j] &= keep;
                            }
                        }
                        const uint32_t at = tile + (c16 >> 2) * HALF + row * 128;
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const uint32_t to = at + ((((2 * c16 + j) & 7) ^ (row & 7)) << 4);
                            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(w[4 * j]), "r"(w[4 * j + 1]),
                                         "r"(w[4 * j + 2]), "r"(w[4 * j + 3])
                                         : "memory");
                            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to + C::TILE), "r"(rest[4 * j]),
                                         "r"(rest[4 * j + 1]), "r"(rest[4 * j + 2]), "r"(rest[4 * j + 3])
                                         : "memory");
                        }
                    }
                    if (bad) atomicMax(&sm.odd, x.start + 1);
                    if (last) fence_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        if (last) mbar_arrive(kv ? &sm.v_full[vs] : &sm.k_full[ks]);
                        if (C::GH == 1 || kv) mbar_arrive(&sm.raw_empty[rs]);
                    }
                    if (C::GH == 1 || kv) {
                        rs ^= 1;
                        r_ph ^= rs == 0;
                        if (warp == 9 && ahead > 0) fetch();
                    }
                }
                if (!ok) break;
                if (++ks == C::KS) {
                    ks = 0;
                    k_ph ^= 1u;
                }
                if (++vs == C::VS) {
                    vs = 0;
                    v_ph ^= 1u;
                }
                if (--left > 0 && ++x.u == x.t.units) paged_next<CH_ROWS, CH_KEYS>(a, p, x);
            }
            // a wait has run out somewhere: the copies in flight end before the shared memory goes
            if (warp == 9 && sm.abort != 0)
                for (int i = max(0, asked - 2); i < asked; ++i) tc_wait(&sm.raw_full[i & 1], (uint32_t)(i >> 1) & 1u, a.err);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TC_TMEM_COLS) : "memory");
    }
}

}  // namespace gtn
