// vb_tree.cu -- attention of drafted tokens over a paged cache.
//
// For token j of sequence i and query head h of K/V head g:
//   o = sum_r p_r v_r / sum_r p_r,  p_r = exp(scale * q.k_r - max)
// over the rows before the draft and the draft rows that j's mask names
// (without a mask: rows up to its own).  A row that sees nothing gives 0.
//
// The rows of the score matrix are the (token, query head) pairs of one K/V
// head: T * group rows share every K/V row that is read.  One pass over the
// cache with the running maximum and sum of the softmax; its tiles go
// through a TMA ring in shared memory, the products through the tensor
// cores.
//
// Work split: an item is (sequence, K/V head, block of rows), a unit one
// 64-row tile of an item's cache.  All units of a call form one line that is
// cut evenly over the CTAs (one per SM), whatever the sequences' lengths, by
// arithmetic that every CTA repeats from the device's own lengths.  A CTA's
// first and last item may be shared with its neighbours: it leaves their
// (max, sum, weighted sum) in its two slots of a workspace and a join kernel
// adds the slots of an item in CTA order, so results do not depend on timing.
//
// This file's kernel multiplies with mma.sync and serves blocks of up to 16
// rows of any type, and what the tcgen05 kernel does not take (launch_rows).
// With few rows the cache's bytes bound it: 524,288 rows of 2 x 2 heads of
// 128 under one token of 16 heads take 95 us in bf16 and in fp32, the second
// 262,144 rows 39 us of it (6.9 TB/s); the constant 17 us are two launches,
// the cut, the first tiles' way and the join.
#include "vb_common.cuh"
#include "vb_kernels.cuh"
#include "vb_tree.cuh"

#include <algorithm>

namespace vb {

constexpr int TR_KT = 64;            // cache rows per tile
constexpr int TR_MAX_STAGES = 8;
// What an item's start and end cost, in tiles: with 2 | 4 | 6 the prompt of
// 4096 fp32 tokens takes 607 | 566 | 588 us, 64 decode steps 98 | 97 | 97.
constexpr int TR_OVER = 4;
constexpr int TR_THREADS = 384;      // warps 0..7 compute, 8..11 load
// Registers: the launch gives 168 a thread; the loading warpgroup goes down
// to 56 and the two computing ones up to 224 (2 * 224 + 56 = 3 * 168), which
// their sums need.
constexpr int TR_SMEM = 226 * 1024;  // dynamic shared memory

// ------------------------------------------------------------ mma helpers
template <int TYPE>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t *a, uint32_t b0, uint32_t b1) {
    if constexpr (TYPE == TR_F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// Room for the queries, and after them for the merge of an item's warps.
__host__ __device__ constexpr int tree_scratch(int hdp, int q_rows, int merge_rows) {
    const int q = q_rows * (hdp * 2 + 16), merge = merge_rows * (hdp + 4) * 4;
    return q > merge ? q : merge;
}

// TYPE: the types; HDP: head_dim rounded up to 64, 128 or 256; WM: groups of
// warps with 16 rows each.  8 / WM warps share a group's rows, split a tile's
// rows and merge at the item's end (with WM = 1 two sets of four warps take
// tiles in turn).  PK: rows of a block of 4 or 8.  A thread then keeps one row
// in place of two (the other eight of an instruction's 16 count for nothing):
// half the exponentials, merges and parts (bf16, 8 sequences of 4000 rows under
// one token took 20.4 us without and 18.7 with it; 17.5 since its loads changed).  The 16-bit terms of an fp32 value lie under one
// another in the 16 rows (row t * PK + m: term t of row m), which takes one
// product or two in place of three; a row's scores and sums are added over
// its terms.  (64 sequences of 8192 rows under one token of 16 heads over 2 took
// 125 us with three products and 111 us with two; 98 to 107 since the loads
// changed, of 82 us that reading the cache takes.)
template <int TYPE, int HDP, int WM, int PK>
__global__ void __launch_bounds__(TR_THREADS, 1)
    tree_attention_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                          const __grid_constant__ TreeArgs g) {
    constexpr bool PACKED = PK < 16;
    static_assert(!PACKED || (WM == 1 && (PK == 8 || TYPE == TR_F32)), "only terms need four");
    constexpr int MT = PACKED ? PK : 16 * WM;    // rows of a block
    constexpr int H = PACKED ? 1 : 2;                // rows that a thread keeps of 16
    constexpr int KW = 8 / WM;                       // warps of a row group
    constexpr int SETS = WM == 1 ? 2 : 1;
    constexpr int NS = WM == 1 ? 1 : 4 / KW;         // 16-row slices of a tile per warp
    constexpr int QT = TYPE == TR_F32 ? 3 : 1;       // 16-bit terms of a query value: 3 bf16 hold an fp32 exactly
    constexpr int NM = PK == 4 ? 1 : PK == 8 ? (QT + 1) / 2 : QT;                  // products that hold them
    constexpr int QROWS = PACKED ? 16 * NM : QT * MT;
    constexpr int CB = HDP / 64;                     // 128-byte column blocks
    constexpr int NT = HDP / 8;                      // output tiles of 8 columns
    constexpr uint32_t TILE = TR_KT * 128;           // bytes of a column block
    constexpr uint32_t STAGE = 2 * CB * TILE;
    constexpr int QPITCH = HDP * 2 + 16;             // bytes; rows 16 bytes apart modulo 128: no bank conflicts
    constexpr int MPITCH = HDP + 4;                  // floats

    extern __shared__ uint8_t raw[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    // the queries and the buffer of the merge share their room: an item's queries are done when its warps merge
    uint8_t *qs = ring + (size_t)g.stages * STAGE;                                  // [QROWS][QPITCH]: term t of row m at t * MT + m
    float *merge = reinterpret_cast<float *>(qs);                                   // [WM * KW / 2][8 * H][MPITCH]
    constexpr int QS = tree_scratch(HDP, QROWS, WM * (KW / 2) * 8 * H);
    float2 *ml = reinterpret_cast<float2 *>(qs + QS);                               // [8][16]
    __shared__ uint64_t full[TR_MAX_STAGES], empty[TR_MAX_STAGES];
    __shared__ TreeCut cut;
    __shared__ int abort_flag, not_finite;           // last item (by its number in this CTA) with a draft value that was not finite

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < TR_MAX_STAGES; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], WM == 1 ? 4 : 8);
        }
        mbar_fence_init();
        abort_flag = 0;
        not_finite = -1;
    }
    pdl_trigger();
    pdl_wait();

    TreeWalk w;
    TreeLine line;
    tree_cut<TR_THREADS>(g, cut, w, line);
    if (w.left <= 0) return;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        // ------------------------------------------------------------ loads
        // Four warps (two for one column block) issue a tile's copies: a box per
        // page, column block and K or V; with pages of 16 rows 16 of them, more
        // than one warp can issue in the time of a tile.  Every warp has a box in
        // every tile (a tile without rows takes the pool's first, which count for
        // nothing), so no fill is over before all have come by, and none can fall
        // behind, or run ahead, to where a parity names another phase than its own.
        // (With an arrival of every warp for that 64 sequences of 8192 rows take
        // 106 us, with a box of every warp 98.)
        constexpr int LW = CB == 1 ? 2 : 4;
        const int P = g.p.page_rows, box = min(P, TR_KT), me = warp - 8;
        if (me >= LW) return;
        int it = 0;
        while (w.left > 0) {
            const int n_tiles = tree_take(g, w);
            const int32_t *row = g.p.table + (int64_t)w.q.s * g.p.max_pages;
            // unit u of a tile: K or V, box u / 2 / CB, column block u / 2 % CB
            const int u = LW * lane + me, k = u / 2 / CB, c = u / 2 % CB;
            auto place = [&](int x) {                   // row of the pool that the lane's box starts at
                const int r = (w.tile + x) * TR_KT + k * box;
                if (r >= w.visible || k * box >= TR_KT) return 0;
                int page = row[r / P];
                if (page < 0 || page >= g.p.n_pages) {
                    atomicCAS(g.err, 0, VB_DEV_TREE_PAGE);
                    page = 0;
                }
                return (page * g.p.n_kv_heads + w.g) * P + r % P;
            };
            int y = n_tiles > 0 ? place(0) : 0;
            for (int x = 0; x < n_tiles; x++, it++) {
                const int y1 = x + 1 < n_tiles ? place(x + 1) : 0;
                const int have = min(TR_KT, w.visible - (w.tile + x) * TR_KT);        // rows of the tile that count
                const int nbox = max(1, (have + box - 1) / box);
                const int s = it % g.stages;
                tree_wait_warp(&empty[s], ((uint32_t)(it / g.stages) & 1u) ^ 1u, &abort_flag, g.err);
                // after a wait that ran out no barrier is touched any more
                const bool go = __shfl_sync(0xffffffffu, *(volatile int *)&abort_flag, 0) == 0;
                if (go && me == 0 && lane == 0) mbar_arrive_expect_tx(&full[s], (uint32_t)nbox * box * 128 * 2 * CB);
                if (go && k < nbox)
                    tma_load_2d(ring + (size_t)s * STAGE + ((u & 1) * CB + c) * TILE + k * box * 128, u & 1 ? &tv : &tk, 64 * c, y,
                                &full[s]);
                __syncwarp();
                y = y1;
            }
            if (w.left > 0) tree_next(g, w);
        }
        // every copy has landed before the CTA can end
        for (int s = 0; s < g.stages; s++) {
            const int fills = it / g.stages + (it % g.stages > s ? 1 : 0);
            if (fills) gm_wait(&full[s], (uint32_t)(fills - 1) & 1u);
        }
        return;
    }

    // ---------------------------------------------------------------- compute
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int wm = WM == 1 ? 0 : warp / KW, kw = warp % KW, set = SETS == 2 ? warp >> 2 : 0;
    const int slice = (WM == 1 ? warp & 3 : kw * NS) * 16;      // this warp's first row of a tile
    const int hd = g.p.head_dim;
    const int quad = lane >> 2, ql = lane & 3;
    int it = 0, item = 0;
    bool first_item = true;
    while (w.left > 0) {
        const int n_tiles = tree_take(g, w);
        if (n_tiles == 0) {
            if (w.left > 0) tree_next(g, w);
            continue;
        }
        const bool whole = n_tiles == w.units;
        const int rows = w.tokens * w.heads;                            // rows of the block that exist
        // queries of the block, in 16-bit terms
        constexpr int N_Q = (MT * (HDP / 4) + 255) / 256;          // four values each
#pragma unroll
        for (int i0 = 0; i0 < N_Q; i0 += 4) {
            float x[4][4];
            uint2 y[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int e = threadIdx.x + 256 * (i0 + i), m = e / (HDP / 4), d = e % (HDP / 4) * 4;
                x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.0f;
                y[i] = make_uint2(0, 0);
                if (i0 + i < N_Q && m < rows && d < hd) {
                    const int64_t at = tree_row(g, w.q.t0, w.tok, w.heads, w.head, 0, m, g.a.ldq) + d;
                    if constexpr (TYPE == TR_F32) {
                        const float *src = static_cast<const float *>(g.a.q) + at;
                        if (g.vec) *reinterpret_cast<float4 *>(x[i]) = *reinterpret_cast<const float4 *>(src);
                        else
#pragma unroll
                            for (int c = 0; c < 4; c++) x[i][c] = src[c];
                    } else {
                        const uint16_t *src = static_cast<const uint16_t *>(g.a.q) + at;
                        if (g.vec) y[i] = *reinterpret_cast<const uint2 *>(src);
                        else y[i] = make_uint2(src[0] | (uint32_t)src[1] << 16, src[2] | (uint32_t)src[3] << 16);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int e = threadIdx.x + 256 * (i0 + i), m = e / (HDP / 4), d = e % (HDP / 4) * 4;
                if (i0 + i >= N_Q || m >= MT) continue;
#pragma unroll
                for (int t = 0; t < (PK == 4 ? 4 : QT); t++) {      // four rows: the fourth term is 0 and fills the 16
                    if constexpr (TYPE == TR_F32) {
                        y[i] = make_uint2(pack2<TYPE>(x[i][0], x[i][1]), pack2<TYPE>(x[i][2], x[i][3]));
                        x[i][0] -= bf16_to_f((uint16_t)y[i].x);
                        x[i][1] -= bf16_to_f((uint16_t)(y[i].x >> 16));
                        x[i][2] -= bf16_to_f((uint16_t)y[i].y);
                        x[i][3] -= bf16_to_f((uint16_t)(y[i].y >> 16));
                    }
                    *reinterpret_cast<uint2 *>(qs + (t * MT + m) * QPITCH + d * 2) = y[i];
                }
            }
        }
        consumer_sync(256);

        float o[NT][4], m[H], l[H];
        int tok[H];                                  // token of the thread's rows, -1: no such row
#pragma unroll
        for (int h = 0; h < H; h++) {
            m[h] = -INFINITY;
            l[h] = 0.0f;
            const int mr = PACKED ? quad % PK : wm * 16 + quad + 8 * h;
            tok[h] = mr < rows ? w.tok + mr / w.heads : -1;
        }
#pragma unroll
        for (int t = 0; t < NT; t++) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.0f;
        const uint32_t q_at = smem_u32(qs) +
                              (uint32_t)((wm * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * QPITCH + (lane >> 4) * 16);
        for (int x = 0; x < n_tiles; x++, it++) {
            if (SETS == 2 && (it & 1) != set) continue;
            const int s = it % g.stages;
            tree_wait_warp(&full[s], (uint32_t)(it / g.stages) & 1u, &abort_flag, g.err);
            const uint32_t kt = smem_u32(ring + (size_t)s * STAGE), vt = kt + CB * TILE;
            // scores: 16 rows x 16 cache rows for each r and slice
            float c[2 * NS][4], lo[2 * NS][4];
#pragma unroll
            for (int t = 0; t < 2 * NS; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) c[t][e] = lo[t][e] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < HDP / 16; ks++) {
                // fp32: the leading term of each step starts from zero and joins
                // the sum in a rounded fp32 add, the small terms run along in `lo`
                uint32_t kb[NS][4];
#pragma unroll
                for (int n = 0; n < NS; n++)
                    ldsm4(kb[n], kt + (ks / 4) * TILE +
                                     sw128(slice + 16 * n + (lane & 7) + (lane >> 4) * 8, (ks % 4) * 2 + ((lane >> 3) & 1)));
                uint32_t qa[4];
#pragma unroll
                for (int t = NM - 1; t > 0; t--) {
                    ldsm4(qa, q_at + (uint32_t)(t * (PACKED ? 16 : MT) * QPITCH + ks * 32));
#pragma unroll
                    for (int n = 0; n < NS; n++) {
                        mma16816<TYPE>(lo[2 * n], qa, kb[n][0], kb[n][1]);
                        mma16816<TYPE>(lo[2 * n + 1], qa, kb[n][2], kb[n][3]);
                    }
                }
                ldsm4(qa, q_at + (uint32_t)(ks * 32));
#pragma unroll
                for (int n = 0; n < NS; n++) {
                    if constexpr (TYPE == TR_F32) {
                        float d0[4] = {}, d1[4] = {};
                        mma16816<TYPE>(d0, qa, kb[n][0], kb[n][1]);
                        mma16816<TYPE>(d1, qa, kb[n][2], kb[n][3]);
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            c[2 * n][e] += d0[e];
                            c[2 * n + 1][e] += d1[e];
                        }
                    } else {
                        mma16816<TYPE>(c[2 * n], qa, kb[n][0], kb[n][1]);
                        mma16816<TYPE>(c[2 * n + 1], qa, kb[n][2], kb[n][3]);
                    }
                }
            }
            if constexpr (TYPE == TR_F32) {
#pragma unroll
                for (int t = 0; t < 2 * NS; t++)
#pragma unroll
                    for (int e = 0; e < 2 * H; e++) {
                        if constexpr (PACKED) lo[t][e] += c[t][e + 2];
                        c[t][e] += lo[t][e];
                        if constexpr (PK == 4) c[t][e] += __shfl_xor_sync(0xffffffffu, c[t][e], 16);
                    }
            }
            const int r0 = (w.tile + x) * TR_KT + slice;       // cache row of the warp's first column
            const bool edge = r0 + 16 * NS > w.clear;          // not every row is seen by every token
#pragma unroll
            for (int t = 0; t < 2 * NS; t++)
#pragma unroll
                for (int e = 0; e < 2 * H; e++) c[t][e] *= g.scale_log2;
            if (edge) {
#pragma unroll
                for (int t = 0; t < 2 * NS; t++)
#pragma unroll
                    for (int e = 0; e < 2 * H; e++) {
                        const int j = tok[e >> 1], d = r0 + 8 * t + 2 * ql + (e & 1) - w.q.base;
                        if (j < 0 || d + w.q.base >= w.visible || (d >= 0 && !tree_sees(g, w.q, j, d)))
                            c[t][e] = -INFINITY;
                    }
                // rows past the end may hold anything: they become zeros, as
                // do draft values that are not finite
                uint8_t *vg = ring + (size_t)s * STAGE + CB * TILE;
                bool found = false;
                for (int e = lane; e < 16 * NS * CB * 8; e += 32) {
                    const int rr = e / (CB * 8), cc = e % (CB * 8);
                    uint4 *p = reinterpret_cast<uint4 *>(vg + (cc >> 3) * TILE + sw128(slice + rr, cc & 7));
                    if (r0 + rr >= w.visible) *p = make_uint4(0, 0, 0, 0);
                    else if (r0 + rr >= w.clear) {
                        bool here = false;
                        const uint4 v = tree_finite<TYPE>(*p, here);
                        if (here) *p = v;
                        found |= here;
                    }
                }
                if (found) not_finite = item;
                __syncwarp();
            }
            // running maximum and sum
            float al[H];
            bool moved = false;
#pragma unroll
            for (int h = 0; h < H; h++) {
                float v = fmaxf(c[0][2 * h], c[0][2 * h + 1]);
#pragma unroll
                for (int t = 1; t < 2 * NS; t++) v = fmaxf(v, fmaxf(c[t][2 * h], c[t][2 * h + 1]));
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
                const float mn = fmaxf(m[h], v), ms = mn == -INFINITY ? 0.0f : mn;
                al[h] = ex2(m[h] - ms);
                moved |= mn != m[h];
                m[h] = mn;
                float sum = 0.0f;
#pragma unroll
                for (int t = 0; t < 2 * NS; t++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float &p = c[t][2 * h + e];
                        p = ex2(p - ms);
                        sum += p;
                    }
                l[h] = fmaf(l[h], al[h], sum);
            }
            if constexpr (TYPE != TR_F32) {
                if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++) o[t][e] *= al[PACKED ? 0 : e >> 1];
                }
            }
            {
                uint32_t pa[4 * NS], pb[4 * NS], pc[4 * NS];      // fp32: a weight in three bf16 terms
#pragma unroll
                for (int k = 0; k < 4 * NS; k += PACKED ? 2 : 1) {
                    const float x0 = c[k >> 1][2 * (k & 1)], x1 = c[k >> 1][2 * (k & 1) + 1];
                    pa[k] = pack2<TYPE>(x0, x1);
                    if constexpr (TYPE == TR_F32) {
                        const float y0 = x0 - bf16_to_f((uint16_t)pa[k]), y1 = x1 - bf16_to_f((uint16_t)(pa[k] >> 16));
                        pb[k] = pack2<TYPE>(y0, y1);
                        pc[k] = pack2<TYPE>(y0 - bf16_to_f((uint16_t)pb[k]), y1 - bf16_to_f((uint16_t)(pb[k] >> 16)));
                    }
                    if constexpr (PK == 4) {            // rows 0..3 | 4..7, 8..11 | 12..15
                        pa[k + 1] = quad < 4 ? pc[k] : 0;
                        pa[k] = quad < 4 ? pa[k] : pb[k];
                    } else if constexpr (PK == 8 && TYPE != TR_F32) {
                        pa[k + 1] = 0;
                    } else if constexpr (PK == 8) {     // rows 0..7, 8..15 of two products
                        pa[k + 1] = pb[k];
                        pb[k] = pc[k];
                        pb[k + 1] = 0;
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; t += 4) {
                    // fp32: a tile's products start from zero and join the sum in
                    // one rounded fp32 step: the tensor cores' own long sums lose
                    // more.  Four sums at a time, so that none waits for its last.
                    float d[4][4] = {};
#pragma unroll
                    for (int n = 0; n < NS; n++) {
                        uint32_t vb[2][4];
#pragma unroll
                        for (int u = 0; u < 2; u++)
                            ldsm4_t(vb[u], vt + (t >> 3) * TILE + sw128(slice + 16 * n + (lane & 7) + ((lane >> 3) & 1) * 8,
                                                                        (t & 7) + 2 * u + (lane >> 4)));
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            if constexpr (NM > 2) mma16816<TYPE>(d[u], pc + 4 * n, vb[u >> 1][2 * (u & 1)], vb[u >> 1][2 * (u & 1) + 1]);
                        }
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            if constexpr (NM > 1) mma16816<TYPE>(d[u], pb + 4 * n, vb[u >> 1][2 * (u & 1)], vb[u >> 1][2 * (u & 1) + 1]);
                        }
#pragma unroll
                        for (int u = 0; u < 4; u++)
                            mma16816<TYPE>(TYPE == TR_F32 ? d[u] : o[t + u], pa + 4 * n, vb[u >> 1][2 * (u & 1)],
                                           vb[u >> 1][2 * (u & 1) + 1]);
                    }
                    if constexpr (TYPE == TR_F32) {
#pragma unroll
                        for (int u = 0; u < 4; u++)
#pragma unroll
                            for (int e = 0; e < 4; e++) o[t + u][e] = fmaf(o[t + u][e], al[PACKED ? 0 : e >> 1], d[u][e]);
                    }
                }
            }
            if (edge) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // zeros written before the next copy
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[s]);
        }

        if constexpr (PACKED && TYPE == TR_F32) {
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float &x = o[t][e];
                    x += o[t][e + 2];
                    if constexpr (PK == 4) x += __shfl_xor_sync(0xffffffffu, x, 16);
                }
        }
        // ---- merge the row group's warps
#pragma unroll
        for (int h = 0; h < H; h++) {
            float &x = l[h];
            x += __shfl_xor_sync(0xffffffffu, x, 1);
            x += __shfl_xor_sync(0xffffffffu, x, 2);
            if (ql == 0) ml[warp * 16 + quad + 8 * h] = make_float2(m[h], x);
        }
        consumer_sync(256);
        // (no warp marks the next item before the barrier behind its queries, which
        // every warp reaches after this)
        const bool mend = *(volatile int *)&not_finite == item;
#pragma unroll
        for (int h = 0; h < H; h++) {
            float2 other[KW];
            float top = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int k = 0; k < KW; k++) {
                other[k] = ml[(wm * KW + k) * 16 + quad + 8 * h];
                top = fmaxf(top, other[k].x);
            }
            const float ms = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int k = 0; k < KW; k++) sum = fmaf(other[k].y, ex2(other[k].x - ms), sum);
            const float f = ex2(m[h] - ms);
            m[h] = top;
            l[h] = sum;
#pragma unroll
            for (int t = 0; t < NT; t++) {
                o[t][2 * h] *= f;
                o[t][2 * h + 1] *= f;
            }
        }
#pragma unroll
        for (int half = KW / 2; half >= 1; half >>= 1) {
            float *slot = merge + (size_t)((wm * (KW / 2) + kw % half) * 8 * H) * MPITCH;
            if (kw >= half && kw < 2 * half) {
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int h = 0; h < H; h++)
                        *reinterpret_cast<float2 *>(slot + (quad + 8 * h) * MPITCH + 8 * t + 2 * ql) =
                            make_float2(o[t][2 * h], o[t][2 * h + 1]);
            }
            consumer_sync(256);
            if (kw < half) {
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int h = 0; h < H; h++) {
                        const float2 v = *reinterpret_cast<const float2 *>(slot + (quad + 8 * h) * MPITCH + 8 * t + 2 * ql);
                        o[t][2 * h] += v.x;
                        o[t][2 * h + 1] += v.y;
                    }
            }
            consumer_sync(256);
        }
        if (kw == 0) {
            float *part = g.part + (size_t)(2 * blockIdx.x + (first_item ? 0 : 1)) * MT * (hd + 2);
            const int lo = max(w.clear, w.tile * TR_KT), hi = min(w.visible, (w.tile + n_tiles) * TR_KT);
#pragma unroll
            for (int h = 0; h < H; h++) {
                const int mr = wm * 16 + quad + 8 * h;
                if (mr >= rows) continue;
                if (whole) {
                    const int64_t at = tree_row(g, w.q.t0, w.tok, w.heads, w.head, 0, mr, g.a.ldo);
                    const float inv = l[h] > 0.0f || l[h] != l[h] ? 1.0f / l[h] : 0.0f;
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        if (8 * t >= hd) break;
                        const float y0 = o[t][2 * h] * inv, y1 = o[t][2 * h + 1] * inv;
                        const int64_t e = at + 8 * t + 2 * ql;
                        if constexpr (TYPE == TR_F32) {
                            float *dst = static_cast<float *>(g.a.out) + e;
                            if (g.vec) *reinterpret_cast<float2 *>(dst) = make_float2(y0, y1);
                            else dst[0] = y0, dst[1] = y1;
                        } else {
                            uint16_t *dst = static_cast<uint16_t *>(g.a.out) + e;
                            const uint32_t y = pack2<TYPE>(y0, y1);
                            if (g.vec) *reinterpret_cast<uint32_t *>(dst) = y;
                            else dst[0] = (uint16_t)y, dst[1] = (uint16_t)(y >> 16);
                        }
                    }
                    __syncwarp(__activemask());
                    if (mend && ql == 0)
                        tree_not_finite<TYPE>(&g, w.q.t0, w.q.s, w.q.base, w.g, tok[h], lo, hi, 0, hd,
                                              static_cast<uint8_t *>(g.a.out) + at * (TYPE == TR_F32 ? 4 : 2), 1,
                                              TYPE == TR_F32);
                } else {
                    if (ql == 0) {
                        part[hd * MT + mr] = m[h];
                        part[(hd + 1) * MT + mr] = l[h];
                    }
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        if (8 * t >= hd) break;
                        part[(8 * t + 2 * ql) * MT + mr] = o[t][2 * h];
                        part[(8 * t + 2 * ql + 1) * MT + mr] = o[t][2 * h + 1];
                    }
                    __syncwarp(__activemask());
                    if (mend && ql == 0)
                        tree_not_finite<TYPE>(&g, w.q.t0, w.q.s, w.q.base, w.g, tok[h], lo, hi, 0, hd, part + mr, MT, 1);
                }
            }
        }
        if (threadIdx.x == 0) tree_describe(g, w, line, n_tiles, first_item);
        __syncwarp();
        first_item = false;
        item++;
        if (w.left > 0) tree_next(g, w);
    }
}

// Joins the parts of items that several CTAs shared:
//   o = sum_c o_c 2^(m_c - m) / sum_c l_c 2^(m_c - m), m the largest m_c.
// A task is 32 rows by 16 columns of an item; a lane holds a row of it and adds
// up parts, several of them on their way at once.  The parts come out of L2:
// bound by the launch and two or three trips there.
//
// Three forms, by the call's items (at most 148 CTAs, so few items have many
// parts); microseconds of a whole call with 16 warps a task | 4 | 1:
//   2 items (one token of 16 heads over 2, 4,000 rows)        14.5 | 22 | 53
//   16 items (8 sequences of up to 25 tokens, 2000 rows)      32.1 | 22.4 | 29.4
//   32 items (16 sequences of one token, 3000 rows)           23.6 | 21.2 | 23.4
//   128 items (64 sequences of one token, 8192 rows)         112.4 | 97.2 | 97.7
//   256 items (one prompt of 4096)                             -   | 138 | 98
// (Joining in the attention kernel, by the last CTA to leave a part, saves the
// launch but costs a fence, a ticket and one SM's reading: from 0.4 us less to
// 15 us more.)
constexpr int TC_COLS = 16;

struct TreeTask {
    int row, t, tr, col, cols;
    bool real;
};

__device__ __forceinline__ TreeTask tree_task(const TreeArgs &g, const TreeShare &d, int task) {
    const int lane = threadIdx.x & 31, row_tasks = (g.mt + 31) / 32;
    TreeTask k;
    const int r = task % row_tasks * 32 + lane;
    k.col = task / row_tasks * TC_COLS;
    k.cols = min(TC_COLS, g.p.head_dim - k.col);
    k.t = r / g.tile_rows;
    k.tr = r - k.t * g.tile_rows;
    k.real = r < g.mt && tree_token(g, d.tokens, d.heads, k.t, k.tr) >= 0;
    k.row = k.real ? r : 0;
    return k;
}

// Parts of CTAs first, first + step, ... of the item.
template <int AHEAD>
__device__ __forceinline__ void tree_join(const TreeArgs &g, const TreeShare &d, const TreeTask &k, int first, int step, float &m, float &l,
                                          float (&o)[TC_COLS]) {
    const int hd = g.p.head_dim;
    for (int c0 = first; c0 <= d.last; c0 += AHEAD * step) {
        float om[AHEAD], ol[AHEAD], v[AHEAD][TC_COLS];
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
            const int c = c0 + a * step;
            const float *part = g.part + (size_t)(c == d.first ? d.slot : 2 * c) * (hd + 2) * g.mt + k.row;
            const bool there = c <= d.last;
            om[a] = there ? part[(size_t)hd * g.mt] : -INFINITY;
            ol[a] = there ? part[(size_t)(hd + 1) * g.mt] : 0.0f;
#pragma unroll
            for (int i = 0; i < TC_COLS; i++) v[a][i] = there && i < k.cols ? part[(size_t)(k.col + i) * g.mt] : 0.0f;
        }
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
            const float mn = fmaxf(m, om[a]), ms = mn == -INFINITY ? 0.0f : mn;
            const float f = ex2(m - ms), e = ex2(om[a] - ms);
            m = mn;
            l = l * f + ol[a] * e;
#pragma unroll
            for (int i = 0; i < TC_COLS; i++) o[i] = o[i] * f + v[a][i] * e;
        }
    }
}

// Few items, each shared by many CTAs: grid (item, task), the warps take the
// parts in turn and are added in shared memory in their order.
template <int TYPE, int TC_MANY>
__global__ void __launch_bounds__(TC_MANY * 32) tree_join_many(const __grid_constant__ TreeArgs g) {
    __shared__ float so[TC_MANY][TC_COLS][32], sm[TC_MANY][32], sl[TC_MANY][32];
    pdl_trigger();
    pdl_wait();
    // the entry was written if the item exists
    const int b = blockIdx.x % g.item_blocks / g.chunks, i = blockIdx.x / g.item_blocks / g.p.n_kv_heads;
    const TreeShare d = g.share[blockIdx.x];
    if (b * g.tb >= tree_seq(g, i).T || d.last < 0) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const TreeTask k = tree_task(g, d, blockIdx.y);
    if (!__any_sync(0xffffffffu, k.real)) return;     // for the whole CTA alike: the rows are the same in every warp
    float m = -INFINITY, l = 0.0f, o[TC_COLS] = {};
    tree_join<3>(g, d, k, d.first + warp, TC_MANY, m, l, o);
#pragma unroll
    for (int c = 0; c < TC_COLS; c++) so[warp][c][lane] = o[c];
    sm[warp][lane] = m;
    sl[warp][lane] = l;
    __syncthreads();
    if (8 * warp >= k.cols) return;                   // two warps write eight columns each
    float top = -INFINITY, sum = 0.0f, f[TC_MANY], y[8] = {};
#pragma unroll
    for (int w = 0; w < TC_MANY; w++) top = fmaxf(top, sm[w][lane]);
    const float ms = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < TC_MANY; w++) {
        f[w] = ex2(sm[w][lane] - ms);
        sum = fmaf(sl[w][lane], f[w], sum);
#pragma unroll
        for (int c = 0; c < 8; c++) y[c] = fmaf(so[w][8 * warp + c][lane], f[w], y[c]);
    }
    const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int c = 0; c < 8; c++) y[c] *= inv;
    if (k.real) tree_store8<TYPE>(g, tree_row(g, d.t0, d.tok, d.heads, d.head, k.t, k.tr, g.a.ldo) + k.col + 8 * warp, y);
}

// More items, of two or three parts, seldom more:
// grid (CTA whose last item goes on, tasks / 4), a task for each warp.
constexpr int TC_FEW = 4;            // warps
template <int TYPE>
__global__ void __launch_bounds__(TC_FEW * 32) tree_join_few(const __grid_constant__ TreeArgs g) {
    pdl_trigger();
    pdl_wait();
    const TreeShare d = g.share[blockIdx.x];
    if (d.last < 0) return;
    const int task = blockIdx.y * TC_FEW + (threadIdx.x >> 5);
    const TreeTask k = tree_task(g, d, task);
    if (k.cols <= 0 || !k.real) return;
    float m = -INFINITY, l = 0.0f, o[TC_COLS] = {};
    tree_join<2>(g, d, k, d.first, 1, m, l, o);
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    const int64_t dst = tree_row(g, d.t0, d.tok, d.heads, d.head, k.t, k.tr, g.a.ldo) + k.col;
#pragma unroll
    for (int c = 0; c < TC_COLS; c += 8) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = o[c + i] * inv;
        if (c < k.cols) tree_store8<TYPE>(g, dst + c, y);
    }
}

// -------------------------------------------------------------------- host
int check_pages(vb_ctx *ctx, const vb_pages *p, const char *who);

typedef void (*TreeKernel)(CUtensorMap, CUtensorMap, TreeArgs);

template <int TYPE, int HDP, int WM, int PK>
static void tree_fit(TreeArgs &g, size_t &smem) {
    constexpr int QROWS = PK == 4 ? 16 : PK == 8 ? (TYPE == TR_F32 ? 32 : 16) : 16 * WM * (TYPE == TR_F32 ? 3 : 1), SLOTS = WM * (8 / WM / 2) * (PK < 16 ? 8 : 16);
    constexpr size_t stage = (size_t)2 * TR_KT * HDP * 2;
    constexpr size_t rest = tree_scratch(HDP, QROWS, SLOTS) + 8 * 16 * 8 + 1024;
    static_assert(rest + 2 * stage <= TR_SMEM, "two stages must fit");
    g.stages = (int)std::min<size_t>(TR_MAX_STAGES, (TR_SMEM - rest) / stage);
    // two sets of warps take tiles in turn: an even ring gives each its own
    // stages.  (A set that met a stage of the other's could wait for its
    // second fill while the first is still on its way, and a parity wait
    // takes that for the phase before, which is over.)
    if (WM == 1) g.stages &= ~1;
    smem = g.stages * stage + rest;
}

// How blocks of row tiles and tiles of kt cache rows cut a call, and its
// workspace: two parts for each CTA, and where the items' parts are.
int tree_prepare(vb_ctx *ctx, TreeArgs &g, int tile_rows, int tiles, int kt, int over) {
    g.tile_rows = tile_rows;
    g.tile_tokens = std::max(1, tile_rows / g.group);
    g.tb = tiles * g.tile_tokens;
    g.mt = tiles * tile_rows;
    g.chunks = (g.group + tile_rows - 1) / tile_rows;
    g.over = over;
    g.kt_log2 = 0;
    while ((1 << g.kt_log2) < kt) g.kt_log2++;
    const int64_t blocks = (int64_t)((g.a.max_tokens + g.tb - 1) / g.tb) * g.chunks, items = blocks * g.a.n * g.p.n_kv_heads;
    const int64_t most = ((int64_t)g.p.max_pages * g.p.page_rows + kt - 1) / kt + over;
    if ((double)items * (double)most >= 2147483647.0)
        return set_error(ctx, VB_ERR_INVALID_ARG, "vb_tree_attention: too many rows for one call");
    g.by_item = items * 4 <= ctx->sm_count;      // four parts each, or more: the join's warps share them
    g.item_blocks = (int)blocks;
    const size_t parts = (size_t)2 * ctx->sm_count * g.mt * (g.p.head_dim + 2) * sizeof(float);
    int rc = arena_reserve(ctx, ctx->tree_ws, parts + (size_t)ctx->sm_count * sizeof(TreeShare));
    if (rc) return rc;
    g.part = static_cast<float *>(ctx->tree_ws.ptr);
    g.share = reinterpret_cast<TreeShare *>(static_cast<char *>(ctx->tree_ws.ptr) + parts);
    return VB_OK;
}

template <int TYPE>
static cudaError_t launch_join(vb_ctx *ctx, const TreeArgs &g) {
    const int tasks = (g.mt + 31) / 32 * ((g.p.head_dim + TC_COLS - 1) / TC_COLS);
    if (g.by_item) {
        const int items = g.a.n * g.p.n_kv_heads * g.item_blocks;
        if (items * 16 <= ctx->sm_count)
            return pdl_launch(ctx, tree_join_many<TYPE, 16>, dim3(items, tasks), dim3(16 * 32), 0, g);
        return pdl_launch(ctx, tree_join_many<TYPE, 4>, dim3(items, tasks), dim3(4 * 32), 0, g);
    }
    return pdl_launch(ctx, tree_join_few<TYPE>, dim3(ctx->sm_count, (tasks + TC_FEW - 1) / TC_FEW), dim3(TC_FEW * 32), 0, g);
}

int launch_tree_combine(vb_ctx *ctx, const TreeArgs &g) {
    VB_CHECK(ctx, g.a.type == VB_TYPE_F32   ? launch_join<TR_F32>(ctx, g)
                  : g.a.type == VB_TYPE_F16 ? launch_join<TR_F16>(ctx, g)
                                            : launch_join<TR_BF16>(ctx, g));
    VB_LAUNCH_CHECK(ctx, "tree_join");
    return VB_OK;
}

template <int TYPE, int HDP, int WM, int PK = 16>
static int launch_tree(vb_ctx *ctx, TreeArgs &g) {
    size_t smem;
    tree_fit<TYPE, HDP, WM, PK>(g, smem);
    const vb_pages &p = g.p;
    int rc = tree_prepare(ctx, g, PK < 16 ? PK : 16 * WM, 1, TR_KT, TR_OVER);
    if (rc) return rc;
    CUtensorMap tk, tv;
    const int64_t rows = (int64_t)p.n_pages * p.n_kv_heads * p.page_rows, layer = (int64_t)g.a.layer * rows * p.head_dim * 2;
    const CUtensorMapDataType dt = p.type == VB_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const int box = std::min(p.page_rows, TR_KT);
    if (!make_map(&tk, static_cast<char *>(p.k) + layer, dt, 2, p.head_dim, rows, 64, box, true) ||
        !make_map(&tv, static_cast<char *>(p.v) + layer, dt, 2, p.head_dim, rows, 64, box, true))
        return set_error(ctx, VB_ERR_BACKEND, "vb_tree_attention: tensor map of the cache refused");
    rc = tree_allow(ctx, reinterpret_cast<const void *>(tree_attention_kernel<TYPE, HDP, WM, PK>), TR_SMEM);
    if (rc) return rc;
    VB_CHECK(ctx, pdl_launch(ctx, tree_attention_kernel<TYPE, HDP, WM, PK>, dim3(ctx->sm_count), dim3(TR_THREADS), smem, tk,
                             tv, g));
    VB_LAUNCH_CHECK(ctx, "tree_attention");
    return launch_tree_combine(ctx, g);
}

// Which kernel and how many rows per block.  16-bit queries of more than 16
// rows go to the tcgen05 kernel (vb_tree_tc.cu), whose tile of 128 rows costs
// the tensor cores less than reading the cache costs the memory, however few
// of its rows exist (8 sequences of 32,768 rows, 32 rows of queries: 64 us
// there, 67 us here; 64 rows 64 | 82; pages of 16 rows).  What is left: up to
// 16 rows, where padding to 128 only delays the first result; heads above 128 values, whose sums and scores do
// not fit its tensor memory; and fp32 queries, whose sums the tcgen05
// accumulators hold less exactly.
//
// There more rows per block mean fewer readings of a tile and more work for
// each; the warps then split rows rather than a tile, and each keeps its
// operands for more products.  Measured at one sequence of 32,768 rows with
// 2 heads (microseconds with blocks of 32 | 64 | 128 rows; "prompt": 4096
// tokens over themselves):
//   fp32, 128 values: 32 rows 27 | 33 | 48, 64 rows 36 | 34 | 49,
//                     128 rows 59 | 49 | 52, 384 rows 144 | 123 | 115, prompt 787 | 635 | 567
//   bf16, 256 values: 32 rows 34 | 38 | 51, 64 rows 46 | 44 | 55,
//                     128 rows 66 | 66 | 66, 384 rows 136 | 121 | 132, prompt 1153 | 863 | 730
// fp32 heads of 256 values leave room for blocks of 32 and two stages only.
template <int TYPE, int HDP>
static int launch_rows(vb_ctx *ctx, TreeArgs &g) {
    const int64_t rows = (int64_t)g.a.max_tokens * g.group;
    if constexpr (TYPE == TR_F32) {
        if (rows <= 4) return launch_tree<TYPE, HDP, 1, 4>(ctx, g);
    }
    if (rows <= 8) return launch_tree<TYPE, HDP, 1, 8>(ctx, g);
    if (rows <= 16) return launch_tree<TYPE, HDP, 1>(ctx, g);
    if constexpr (TYPE == TR_F32) {
        if constexpr (HDP == 256) return launch_tree<TYPE, HDP, 2>(ctx, g);      // more rows leave no room for two stages
        else if (rows <= 32) return launch_tree<TYPE, HDP, 2>(ctx, g);
        else if (rows <= 128) return launch_tree<TYPE, HDP, 4>(ctx, g);
        else return launch_tree<TYPE, HDP, 8>(ctx, g);
    } else {
        if constexpr (HDP == 256) return rows <= 64 ? launch_tree<TYPE, HDP, 2>(ctx, g) : rows <= 512 ? launch_tree<TYPE, HDP, 4>(ctx, g) : launch_tree<TYPE, HDP, 8>(ctx, g);
        else return launch_tree_tc(ctx, g);
    }
}

template <int TYPE>
static int launch_heads(vb_ctx *ctx, TreeArgs &g) {
    const int hd = g.p.head_dim;
    return hd <= 64 ? launch_rows<TYPE, 64>(ctx, g) : hd <= 128 ? launch_rows<TYPE, 128>(ctx, g) : launch_rows<TYPE, 256>(ctx, g);
}

// A kernel's leave to take so much dynamic shared memory, asked for once, when
// it first runs: asking loads it, which took a context's creation 18 ms for all
// of this operator's.
int tree_allow(vb_ctx *ctx, const void *kernel, int bytes) {
    for (const void *k : ctx->tree_kernels)
        if (k == kernel) return VB_OK;
    VB_CHECK(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    try {
        ctx->tree_kernels.push_back(kernel);
    } catch (...) {                                   // asked for again next time
    }
    return VB_OK;
}

}  // namespace vb

using namespace vb;

extern "C" int vb_tree_attention(vb_ctx *ctx, const vb_tree_args *in) {
    if (!ctx) return VB_ERR_INVALID_ARG;
    auto bad = [&](const char *why) { return set_error(ctx, VB_ERR_INVALID_ARG, "vb_tree_attention: %s", why); };
    if (!in) return bad("null arguments");
    TreeArgs g{};
    g.a = *in;
    vb_tree_args &a = g.a;
    int rc = check_pages(ctx, a.pages, "vb_tree_attention");
    if (rc) return rc;
    g.p = *a.pages;
    if (a.type != g.p.type && !(a.type == VB_TYPE_F32 && g.p.type == VB_TYPE_BF16))
        return bad("type must be the cache's, or F32 over a BF16 cache");
    if (a.layer < 0 || a.layer >= g.p.n_layers) return bad("layer out of range");
    if (a.n < 0 || a.n_tokens < 0 || a.max_tokens < 0 || a.n_heads <= 0) return bad("bad sizes");
    if (a.n_heads % g.p.n_kv_heads) return bad("n_heads must be a multiple of the cache's n_kv_heads");
    g.group = a.n_heads / g.p.n_kv_heads;
    const int64_t qd = (int64_t)a.n_heads * g.p.head_dim;
    if (!a.ldq) a.ldq = qd;
    if (!a.ldo) a.ldo = qd;
    if (a.ldq < qd || a.ldo < qd) return bad("row stride below the row");
    if (!(a.scale >= 0.0f)) return bad("negative scale");
    g.scale_log2 = (float)((a.scale == 0.0f ? 1.0 / sqrt((double)g.p.head_dim) : (double)a.scale) * 1.4426950408889634);
    if (a.mask && a.mask_words <= 0) return bad("mask without words");
    if ((int64_t)a.max_tokens * g.group > INT32_MAX / 2) return bad("too many rows");
    if (a.n == 0 || a.n_tokens == 0 || a.max_tokens == 0) return VB_OK;
    if (!a.q || !a.out || !a.seqs || !a.start) return bad("null pointer");
    const uintptr_t es = a.type == VB_TYPE_F32 ? 4 : 2;
    if (((uintptr_t)a.q | (uintptr_t)a.out) % es || ((uintptr_t)a.seqs | (uintptr_t)a.start | (uintptr_t)a.mask) % 4)
        return bad("misaligned pointer");
    g.vec = ((uintptr_t)a.q | (uintptr_t)a.out) % 16 == 0 && (a.ldq | a.ldo) % (16 / (int64_t)es) == 0;
    g.err = ctx->op_error;
    return a.type == VB_TYPE_F32   ? launch_heads<TR_F32>(ctx, g)
           : a.type == VB_TYPE_F16 ? launch_heads<TR_F16>(ctx, g)
                                   : launch_heads<TR_BF16>(ctx, g);
}
