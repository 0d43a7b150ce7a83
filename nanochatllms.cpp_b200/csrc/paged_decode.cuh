// Paged attention for few query rows per kv head (single tokens, short drafts): bound by reading K and V
// once, so the keys are split over the whole GPU (paged_sched.cuh) and streamed from global memory
// straight into matrix-instruction fragments; no shared memory on the way and no barrier inside an item.
//
// A warp owns every fourth 32-key step. S = Q K^T and O = P V run on m16n8k16 instructions (fp16 in, fp32
// sums) with up to 16 query rows as M: at one token the products are small next to the loads, and the
// fragment layouts are what lets one 16-byte load feed them without a transposition:
//   * contraction over d: any one-to-one assignment of d to (k step, lane) works if Q uses the same; lane
//     (g, t) = (lane / 4, lane % 4) holds key g's elements 32 c + 8 t .. + 7, one 16-byte load per chunk c;
//   * contraction over keys: the score fragment's keys (2t, 2t + 1, 2t + 8, 2t + 9 of 16) are the weight
//     fragment's, and lane (g, t) loads those keys' columns 8 g .. 8 g + 7 of V; a byte permute pairs two
//     keys, and the column order of the result is the loads'.
// Q8 caches keep their 8-bit values exact in fp16; the deltas are applied in fp32, to the scores per
// 32-element block of K and to the weights per 32-column block of V before these round to fp16.
#pragma once
#include "paged_sched.cuh"

namespace gtn {

constexpr int PD_THREADS = 128;
constexpr int PD_KEYS = 128;  // keys of a unit: one 32-key step per warp
// The weights are 2^(s - max + PD_BIAS) instead of 2^(s - max), which cancels in the division: small weights
// (and weights times small deltas) stay that much longer above fp16's subnormal range.
constexpr float PD_BIAS = 6.0f;

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
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Read-once data: past L1.
__device__ __forceinline__ uint4 ld_stream16(const uint8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 ld_stream8(const uint8_t* p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t ld_stream4(const uint8_t* p) {
    uint32_t v;
    asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}

// Eight fp16 elements e0 .. e0 + 7 of a row in dtype io (Q8: rounded to fp16, as the header says).
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
__global__ void __launch_bounds__(PD_THREADS, D == 64 ? 3 : 2) k_paged_decode(PagedAttnArgs a, PagedPick p) {
    constexpr int NC = D / 32;       // 32-element chunks of a head row
    constexpr int NO = D / 8;        // 8-column tiles of the output
    constexpr bool R16 = ROWS == 16;
    constexpr int NR = R16 ? 2 : 1;  // rows per lane: g, and g + 8
    constexpr bool Q = DT == GTN_Q8;
    __shared__ PagedSchedSmem sm;
    __shared__ float s_ml[4][2][ROWS];
    extern __shared__ __align__(16) float s_o[];  // [4 warps][ROWS][D + 4]
    constexpr int OS = D + 4;
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const PagedSched sch = paged_sched<ROWS, PD_KEYS, PD_THREADS>(a, p, gridDim.x, blockIdx.x, blockIdx.x == 0, sm);
    PagedPos x = sch.pos;
    if (x.b < 0) return;
    const long long begin = sch.share * blockIdx.x;
    long long left = min(sch.total - begin, sch.share);
    const long hb = row_bytes(a.io, D);
    const int psm = a.c.ps - 1;
    while (left > 0) {
        const int u0 = x.u, u1 = (int)min((long long)x.t.units, u0 + left);
        const int nrow = min(ROWS, x.r.n * a.group - x.tile * ROWS);  // query rows of this item
        // query fragments: k step i covers elements 4 (i % 2) .. + 3 of every lane's eight of chunk i / 2
        uint32_t qa[2 * NC][4];
        int pos[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const int row = g + 8 * r;
            const bool in = row < nrow;
            pos[r] = in ? x.r.base + (x.tile * ROWS + row) / a.group : -1;
            const uint8_t* qh = a.q + (in ? paged_row_at(a, x, row, ROWS, a.qs, hb) : 0);
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
        const int32_t* table = a.table + x.b * a.table_stride;
        const int wlo = a.window > 0 ? max(0, x.t.plo - a.window + 1) : 0;  // first window key of the tile
        // keys [0, full_hi] and from full_lo on (or below n_sink) are seen by every row
        const int full_lo = a.window > 0 ? max(0, x.t.phi - a.window + 1) : 0, full_hi = x.t.plo;

        for (int u = u0; u < u1; ++u) {
            const int kb = paged_unit_key<PD_KEYS>(x.t, u) + warp * 32;
            if (kb > x.t.phi || (kb + 31 < wlo && kb >= a.n_sink)) continue;  // nothing of this step is seen
            // the step's two 16-key halves: their pages, and whether any key of them is seen
            const uint8_t *kp[2], *vp[2];
            bool need[2];
            int kr[2];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int k0 = kb + 16 * s;
                need[s] = k0 <= x.t.phi && (k0 + 15 >= wlo || k0 < a.n_sink);
                int page = need[s] ? table[k0 >> a.c.ps_shift] : 0;
                if (need[s] && (unsigned)page >= (unsigned)a.c.n_pages) {
                    need[s] = false;
                    if (lane == 0) atomicOr(a.err, GTN_DEVERR_PAGE);
                }
                if (!need[s]) page = 0;
                kr[s] = k0 & psm;
                kp[s] = a.c.k + (long)page * a.c.page_stride;
                vp[s] = a.c.v + (long)page * a.c.page_stride;
            }
            const bool full = need[0] && need[1] && kb + 31 <= full_hi && (kb >= full_lo || kb + 32 <= a.n_sink);
            auto seen_any = [&](int key) { return key <= x.t.phi && (key >= wlo || key < a.n_sink); };

            // ---- loads
            uint4 kf[4][Q ? 1 : NC];      // fp16: chunk c of key 8 n + g
            uint2 kq[4][Q ? NC : 1];      // Q8: eight int8 of chunk c
            uint2 kd[4][Q ? NC / 2 : 1];  // Q8: the deltas of keys 8 n + 2t, + 1 (D = 64: both keys' two)
            uint4 vf[8][Q ? 1 : NC / 2];  // fp16: columns 64 c + 8 g .. + 7 of the lane's key i of 8
            uint32_t vq[8][Q ? NC : 1];   // Q8: columns 32 c + 4 g .. + 3
            uint2 vd[4][Q ? NC / 2 : 1];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int s = n >> 1, r0 = kr[s] + 8 * (n & 1);
                const bool ld = need[s] && (full || seen_any(kb + 8 * n + g));
                const uint8_t* row = kp[s] + paged_row(a.c, x.h, r0 + g);
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    if (Q) kq[n][c] = ld ? ld_stream8(row + 32 * c + 8 * t) : make_uint2(0u, 0u);
                    else kf[n][c] = ld ? ld_stream16(row + 64 * c + 16 * t) : make_uint4(0u, 0u, 0u, 0u);
                }
                if (Q) {
                    const uint8_t* dl = kp[s] + paged_delta(a.c, x.h, r0 + 2 * t);
#pragma unroll
                    for (int c = 0; c < NC / 2; ++c) kd[n][c] = need[s] ? ld_stream8(dl + 8 * c) : make_uint2(0u, 0u);
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {  // keys 16 s + 8 h + 2t + e, i = 4 s + 2 h + e
                const int s = i >> 2, kk = 8 * ((i >> 1) & 1) + 2 * t + (i & 1);
                const bool ld = need[s] && (full || seen_any(kb + 16 * s + kk));
                const uint8_t* row = vp[s] + paged_row(a.c, x.h, kr[s] + kk);
                if (Q) {
#pragma unroll
                    for (int c = 0; c < NC; ++c) vq[i][c] = ld ? ld_stream4(row + 32 * c + 4 * g) : 0u;
                    if ((i & 1) == 0) {
                        const uint8_t* dl = vp[s] + paged_delta(a.c, x.h, kr[s] + kk);
#pragma unroll
                        for (int c = 0; c < NC / 2; ++c) vd[i >> 1][c] = need[s] ? ld_stream8(dl + 8 * c) : make_uint2(0u, 0u);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < NC / 2; ++c)
                        vf[i][c] = ld ? ld_stream16(row + 128 * c + 16 * g) : make_uint4(0u, 0u, 0u, 0u);
                }
            }

            // ---- scores
            float sc[4][4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[n][i] = 0.0f;
                if (!Q) {
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        mma_16816(sc[n], qa[2 * c], kf[n][c].x, kf[n][c].y);
                        mma_16816(sc[n], qa[2 * c + 1], kf[n][c].z, kf[n][c].w);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        float blk[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        const uint2 lo = tc_bytes_to_f16x4(kq[n][c].x ^ 0x80808080u, 0x64806480u);
                        const uint2 hi = tc_bytes_to_f16x4(kq[n][c].y ^ 0x80808080u, 0x64806480u);
                        mma_16816(blk, qa[2 * c], lo.x, lo.y);
                        mma_16816(blk, qa[2 * c + 1], hi.x, hi.y);
                        // deltas of keys 2t and 2t + 1: NC halves per key, keys adjacent
                        const uint32_t w0 = D == 64 ? kd[n][0].x : (c < 2 ? kd[n][0].x : kd[n][0].y);
                        const uint32_t w1 = D == 64 ? kd[n][0].y : (c < 2 ? kd[n][NC / 2 - 1].x : kd[n][NC / 2 - 1].y);
                        const float d0 = h2f((uint16_t)(w0 >> (16 * (c & 1)))), d1 = h2f((uint16_t)(w1 >> (16 * (c & 1))));
                        sc[n][0] = fmaf(blk[0], d0, sc[n][0]);
                        sc[n][1] = fmaf(blk[1], d1, sc[n][1]);
                        if (R16) {
                            sc[n][2] = fmaf(blk[2], d0, sc[n][2]);
                            sc[n][3] = fmaf(blk[3], d1, sc[n][3]);
                        }
                    }
                }
            }
            bool mixed = false;  // some row sees a key of this step that another does not
            if (!full) {
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int key = kb + 8 * n + 2 * t + e;
                        const bool any = need[n >> 1] && seen_any(key);
#pragma unroll
                        for (int r = 0; r < NR; ++r) {
                            const bool see = any && key <= pos[r] &&
                                             (a.window == 0 || key > pos[r] - a.window || key < a.n_sink);
                            if (!see) sc[n][2 * r + e] = -INFINITY;
                            mixed |= any && !see;
                        }
                    }
                mixed = x.t.plo != x.t.phi && __any_sync(0xffffffffu, mixed);
            }

            // ---- softmax: running maximum and sum per row, in base 2
            uint32_t pa[2][Q ? NC : 1][4];  // weight fragments of 16 keys (Q8: times the deltas of V's block c)
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                float mx = sc[0][2 * r];
#pragma unroll
                for (int n = 0; n < 4; ++n) mx = fmaxf(mx, fmaxf(sc[n][2 * r], sc[n][2 * r + 1]));
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
                for (int n = 0; n < 4; ++n) {
                    const float e0 = ex2(fmaf(sc[n][2 * r], a.scale_log2, PD_BIAS - ms));
                    const float e1 = ex2(fmaf(sc[n][2 * r + 1], a.scale_log2, PD_BIAS - ms));
                    sum += e0 + e1;
                    const int s = n >> 1, slot = r + 2 * (n & 1);
                    if (!Q) {
                        pa[s][0][slot] = pack_f16(e0, e1);
                    } else {
#pragma unroll
                        for (int c = 0; c < NC; ++c) {
                            const uint32_t w0 = D == 64 ? vd[n][0].x : (c < 2 ? vd[n][0].x : vd[n][0].y);
                            const uint32_t w1 = D == 64 ? vd[n][0].y : (c < 2 ? vd[n][NC / 2 - 1].x : vd[n][NC / 2 - 1].y);
                            float y0 = e0 * h2f((uint16_t)(w0 >> (16 * (c & 1))));
                            float y1 = e1 * h2f((uint16_t)(w1 >> (16 * (c & 1))));
                            // a hidden key's delta may hold anything: its weight is zero whatever it is
                            if (!full) {
                                y0 = sc[n][2 * r] == -INFINITY ? 0.0f : y0;
                                y1 = sc[n][2 * r + 1] == -INFINITY ? 0.0f : y1;
                            }
                            pa[s][c][slot] = pack_f16(y0, y1);
                        }
                    }
                }
                l[r] += sum;
            }
            if (!R16) {
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int c = 0; c < (Q ? NC : 1); ++c) pa[s][c][1] = pa[s][c][3] = 0u;
            }

            // ---- O += P V
            auto pv = [&](float (&acc)[NO][4]) {
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    if (!Q) {
#pragma unroll
                        for (int c = 0; c < NC / 2; ++c) {
                            const uint4 v0 = vf[4 * s][c], v1 = vf[4 * s + 1][c], v2 = vf[4 * s + 2][c], v3 = vf[4 * s + 3][c];
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
                        for (int c = 0; c < NC; ++c)
#pragma unroll
                            for (int hi = 0; hi < 2; ++hi) {
                                const uint2 b0 = pair_bytes(vq[4 * s][c], vq[4 * s + 1][c], hi);
                                const uint2 b1 = pair_bytes(vq[4 * s + 2][c], vq[4 * s + 3][c], hi);
                                mma_16816(acc[4 * c + 2 * hi], pa[s][c], b0.x, b1.x);
                                mma_16816(acc[4 * c + 2 * hi + 1], pa[s][c], b0.y, b1.y);
                            }
                    }
                }
            };
            bool odd = false;  // a non-finite value where rows differ in what they see
            if (!Q && mixed) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int c = 0; c < NC / 2; ++c) {
                        const uint32_t w[4] = {vf[i][c].x, vf[i][c].y, vf[i][c].z, vf[i][c].w};
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            odd |= (w[j] & 0x7c00u) == 0x7c00u || (w[j] & 0x7c000000u) == 0x7c000000u;
                    }
                odd = __any_sync(0xffffffffu, odd);
            }
            if (!odd) {
                pv(o);
            } else {
                // weight 0 times NaN or infinity must not reach the rows that do not see the key: once per
                // token, with only that token's keys of V, kept for that token's rows
                for (int tok = x.t.plo; tok <= x.t.phi; ++tok) {
                    uint4 keep[8][Q ? 1 : NC / 2];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int key = kb + 16 * (i >> 2) + 8 * ((i >> 1) & 1) + 2 * t + (i & 1);
                        const bool see = key <= tok && (a.window == 0 || key > tok - a.window || key < a.n_sink);
#pragma unroll
                        for (int c = 0; c < (Q ? 1 : NC / 2); ++c) {
                            keep[i][c] = vf[i][c];
                            if (!see) vf[i][c] = make_uint4(0u, 0u, 0u, 0u);
                        }
                    }
                    float tmp[NO][4];
#pragma unroll
                    for (int j = 0; j < NO; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) tmp[j][i] = o[j][i];
                    pv(tmp);
#pragma unroll
                    for (int j = 0; j < NO; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (pos[R16 ? i >> 1 : 0] == tok) o[j][i] = tmp[j][i];
#pragma unroll
                    for (int i = 0; i < 8; ++i)
#pragma unroll
                        for (int c = 0; c < (Q ? 1 : NC / 2); ++c) vf[i][c] = keep[i][c];
                }
            }
        }

        // ---- join the warps and write the item, or its part
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if (t == 0) {
                s_ml[warp][0][g + 8 * r] = m[r];
                s_ml[warp][1][g + 8 * r] = l[r];
            }
            // fp16: tile 8 c + j holds columns 64 c + 8 (2t) + j and 64 c + 8 (2t + 1) + j; Q8: tile 4 c + j
            // columns 32 c + 4 (2t) + j and 32 c + 4 (2t + 1) + j
            float* dst = s_o + (long)(warp * ROWS + g + 8 * r) * OS;
#pragma unroll
            for (int j = 0; j < NO; ++j) {
                const int c0 = Q ? 32 * (j >> 2) + 8 * t + (j & 3) : 64 * (j >> 3) + 16 * t + (j & 7);
                dst[c0] = o[j][2 * r];
                dst[c0 + (Q ? 4 : 8)] = o[j][2 * r + 1];
            }
        }
        __syncthreads();
        constexpr int TPR = PD_THREADS / ROWS, N = D / TPR;  // threads per row, columns per thread
        {
            const int row = tid / TPR, c0 = tid % TPR * N;
            float mm = -INFINITY, ll = 0.0f, y[N];
#pragma unroll
            for (int w = 0; w < 4; ++w) mm = fmaxf(mm, s_ml[w][0][row]);
            const float ms = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
            for (int j = 0; j < N; ++j) y[j] = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = ex2(s_ml[w][0][row] - ms);
                ll = fmaf(s_ml[w][1][row], f, ll);
#pragma unroll
                for (int j = 0; j < N; j += 4) {
                    const float4 v = *reinterpret_cast<const float4*>(s_o + (long)(w * ROWS + row) * OS + c0 + j);
                    y[j] = fmaf(v.x, f, y[j]);
                    y[j + 1] = fmaf(v.y, f, y[j + 1]);
                    y[j + 2] = fmaf(v.z, f, y[j + 2]);
                    y[j + 3] = fmaf(v.w, f, y[j + 3]);
                }
            }
            if (u0 == 0 && u1 == x.t.units) {
                const float inv = ll != 0.0f ? 1.0f / ll : 0.0f;
#pragma unroll
                for (int j = 0; j < N; ++j) y[j] = ll != 0.0f ? y[j] * inv : 0.0f;
                const bool live = row < nrow;
                paged_store<N>(a.out + (live ? paged_row_at(a, x, row, ROWS, a.os, hb) : 0), a.io, c0, y, live);
            } else {
                float* ps = a.part + (2L * blockIdx.x + (u0 == 0)) * paged_slot<ROWS, D>();
#pragma unroll
                for (int j = 0; j < N; j += 4)
                    *reinterpret_cast<float4*>(ps + row * D + c0 + j) = make_float4(y[j], y[j + 1], y[j + 2], y[j + 3]);
                if (c0 == 0) {
                    ps[ROWS * D + row] = mm;
                    ps[ROWS * (D + 1) + row] = ll;
                }
            }
        }
        __syncthreads();
        left -= u1 - u0;
        if (left > 0) paged_next<ROWS, PD_KEYS>(a, p, x);
    }
}

template <int D, int ROWS>
constexpr size_t paged_decode_smem() {
    return (size_t)4 * ROWS * (D + 4) * sizeof(float);
}

}  // namespace gtn
