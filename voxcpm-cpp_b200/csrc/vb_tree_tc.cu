// vb_tree_tc.cu -- drafted-token attention on the tcgen05 tensor cores, for
// 16-bit queries of more than 16 rows (tokens x query heads of a K/V head).
//
// Both products run as kind::f16 MMAs of 128 score rows: S = Q K^T from
// shared memory into tensor memory, where the softmax threads (one per row)
// read it and leave the weights P as 16-bit values in its place; O += P V
// takes P from tensor memory and V as it lies in the cache (rows along the
// contraction) from shared memory.
//
// Two streams of four softmax warps keep the tensor cores busy while the
// other stream takes its exponentials:
//   PAIR  (more than 128 rows): the streams are two row tiles that share
//         every K and V tile, 256 rows per block;
//   else: the streams take the cache tiles of one row tile in turn and are
//         added at the end.
// The sums follow a running maximum that moves only when a score exceeds it
// by 2^8 (the weights stay far inside the 16-bit formats), so O is rarely
// rescaled in tensor memory.
//
// Bound by the tensor cores with the exponentials beside them where rows are
// many (four prompts of 4096 tokens, 16 heads over 2 of 128 values: 282 to 289 us, 950
// to 975 TFLOP/s of the 1647 that a large matrix product reaches), by the cache's
// bytes and the first and last tiles below that (262,144 rows under 32 tokens
// 79 to 81 us, of which reading takes 41 and the products alone 42).  In a block
// of two row tiles whose second has no rows that one's products are issued too.
//
// Warps 0..7 softmax (warpgroup = stream), 9 issues the MMAs, 8, 10 and 11
// issue the copies (TMA, one box per page and column block).
#include "vb_kernels.cuh"
#include "vb_tree.cuh"

#include <algorithm>
#include <type_traits>

namespace vb {

constexpr int TT_KT = 128;
constexpr int TT_THREADS = 384;
constexpr int TT_SLOTS = 12;
// What an item's start and end cost, in tiles.  A prompt of 4096 tokens (89 to 97
// us over several GPUs) took on one of them with 3 | 4 89 | 89 us, four of them 282 | 287, 64 ragged drafts over 4000 rows
// 60 | 62; while an item's first and last tiles still took two passes, that
// prompt took 159 | 98 | 92 | 95 with 0 | 2 | 4 | 6.
constexpr int TT_OVER = 3;
constexpr int TT_SMEM = 225 * 1024;
// Of 16 pairs of weights, those that the multiply-add pipe takes: 0 | 5 | 10
// made that prompt 111 | 98 | 112 us (then with 2 tiles for an item's ends).
constexpr int TT_POLY = 5;
constexpr float TT_SLACK = 8.0f;     // log2 of how far a score may exceed the running maximum

// One lane of the (converged) warp.
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r;
}

// MMAs and commits issued where `one` is set, so that the code around them
// is the same for the whole warp.
__device__ __forceinline__ void umma_f16_ss(uint32_t one, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p, e;\n setp.ne.b32 e, %0, 0;\n setp.ne.b32 p, %5, 0;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%1], %2, %3, %4, p;\n}\n" ::"r"(one),
        "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}

__device__ __forceinline__ void umma_f16_ts(uint32_t one, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p, e;\n setp.ne.b32 e, %0, 0;\n setp.ne.b32 p, %5, 0;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], %3, %4, p;\n}\n" ::"r"(one),
        "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}

__device__ __forceinline__ void umma_commit_one(uint32_t one, uint64_t *bar) {
    asm volatile(
        "{\n .reg .pred e;\n setp.ne.b32 e, %0, 0;\n"
        " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n}\n" ::"r"(one),
        "r"(smem_u32(bar))
        : "memory");
}

// A tile of [rows][64 values] column blocks 16 KB apart whose rows run along
// the contraction: 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t sw128_desc_mn(uint32_t addr) {
    uint64_t d = (uint64_t)((addr >> 4) & 0x3FFFu);
    d |= (uint64_t)(16384 >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

// Load and wait in one statement (the registers are written asynchronously).
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A load whose wait comes later: until then nothing may touch the registers,
// so the wait takes them all as its operands.
__device__ __forceinline__ void tmem_ld32_start(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}

__device__ __forceinline__ void tmem_ld32_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                   "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                   "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// Pairs of fp32 values in one 64-bit register.
__device__ __forceinline__ uint64_t pack_b32x2(uint32_t a, uint32_t b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint64_t pack_f32x2(float a, float b) { return pack_b32x2(__float_as_uint(a), __float_as_uint(b)); }
__device__ __forceinline__ void unpack_f32x2(uint64_t d, float &a, float &b) {
    uint32_t x, y;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(x), "=r"(y) : "l"(d));
    a = __uint_as_float(x);
    b = __uint_as_float(y);
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// max(a, b, c), NaN where there is one.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// 2^x of two values on the multiply-add pipe instead of the special-function
// unit: x = i + f with i its nearest integer (adding 1.5 * 2^23 leaves i in
// the low bits), 2^f by the cubic of least relative error on [-1/2, 1/2]
// (7.5e-5, a sixth of fp16's rounding), i added to the exponent.  Values
// below -126 count as -126; NaN is not kept.
__device__ __forceinline__ void exp2_pair(uint64_t x2, float &p0, float &p1) {
    float x0, x1, i0, i1;
    unpack_f32x2(x2, x0, x1);
    x2 = pack_f32x2(fmaxf(x0, -126.0f), fmaxf(x1, -126.0f));
    const uint64_t magic = pack_f32x2(12582912.0f, 12582912.0f);
    const uint64_t t = add_f32x2(x2, magic);
    const uint64_t f = add_f32x2(x2, fma_f32x2(t, pack_f32x2(-1.0f, -1.0f), magic));
    uint64_t p = fma_f32x2(f, pack_f32x2(0.05517167f, 0.05517167f), pack_f32x2(0.24261113f, 0.24261113f));
    p = fma_f32x2(p, f, pack_f32x2(0.69326097f, 0.69326097f));
    p = fma_f32x2(p, f, pack_f32x2(0.99992806f, 0.99992806f));
    unpack_f32x2(p, p0, p1);
    unpack_f32x2(t, i0, i1);
    p0 = __uint_as_float(__float_as_uint(p0) + (__float_as_uint(i0) << 23));
    p1 = __uint_as_float(__float_as_uint(p1) + (__float_as_uint(i1) << 23));
}

// The ring holds K and V tiles in the order in which the MMAs use them:
// PAIR K0 V0 K1 V1 ..., else K0 K1 V0 K2 V1 ... V(n-1).
template <bool PAIR>
__device__ __forceinline__ void ring_entry(int e, int n, int &tile, bool &is_v) {
    if (PAIR) {
        tile = e >> 1;
        is_v = e & 1;
    } else if (e & 1) {
        is_v = (e + 1) / 2 >= n;
        tile = is_v ? n - 1 : (e + 1) / 2;
    } else {
        is_v = e > 0;
        tile = is_v ? e / 2 - 1 : 0;
    }
}
template <bool PAIR>
__device__ __forceinline__ int ring_k(int j) { return PAIR ? 2 * j : j == 0 ? 0 : 2 * j - 1; }
template <bool PAIR>
__device__ __forceinline__ int ring_v(int j, int n) { return PAIR ? 2 * j + 1 : min(2 * j + 2, 2 * n - 1); }

template <int TYPE, int HDP, bool PAIR>
__global__ void __launch_bounds__(TT_THREADS, 1)
    tree_tc_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                   const __grid_constant__ CUtensorMap tq, const __grid_constant__ TreeArgs g) {
    constexpr int CB = HDP / 64;
    constexpr uint32_t BLOCK = TT_KT * 128;          // bytes of a 64-value column block of 128 rows
    constexpr uint32_t SLOT = CB * BLOCK;
    constexpr int MT = PAIR ? 256 : 128;

    extern __shared__ uint8_t raw[];
    uint8_t *qs = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *ring = qs + (PAIR ? 2 : 1) * SLOT;
    float2 (*ml)[128] = reinterpret_cast<float2 (*)[128]>(ring + (size_t)g.stages * SLOT);   // !PAIR: (max, sum) of both streams
    __shared__ uint64_t full[TT_SLOTS], empty[TT_SLOTS], q_full, q_empty, s_full[2], p_full[2], pv_done[2];
    __shared__ TreeCut cut;
    __shared__ uint32_t s_tmem;
    __shared__ int abort_flag, not_finite[2];        // item number in which a draft value was not finite, by its parity

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < TT_SLOTS; s++) {
            mbar_init(&full[s], 3);
            mbar_init(&empty[s], 1);
        }
        mbar_init(&q_full, g.q_tma ? 1 : 8);
        mbar_init(&q_empty, 2);
        for (int t = 0; t < 2; t++) {
            mbar_init(&s_full[t], 1);
            mbar_init(&p_full[t], 4);
            mbar_init(&pv_done[t], 1);
            not_finite[t] = -1;
        }
        mbar_fence_init();
        abort_flag = 0;
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    pdl_trigger();
    pdl_wait();
    TreeWalk w;
    TreeLine line;
    tree_cut<TT_THREADS>(g, cut, w, line);
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    // tensor memory: scores (then weights) of stream t at column 128 t, sums at 256 + HDP t
    const int n_slots = g.stages;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 152;");
        if (warp != 9) {
            // -------------------------------------------------------- loads
            // Three warps issue a tile's copies (a box per page and column
            // block: 16 of them with pages of 16 rows, more than one warp can
            // issue in the time of a tile).  Every warp waits for every slot and
            // arrives at every fill, whether or not it has a box in it: a fill is
            // over only when all three have come by, so that none can fall behind, or
            // run ahead, to where a parity names another phase than its own.
            const int P = g.p.page_rows, box = min(P, TT_KT), me = warp == 8 ? 0 : warp - 9;
            const int u = 3 * lane + me, k = u / CB, c = u % CB;         // box and column block of the lane's copy
            int slot = 0, item = 0;
            uint32_t phase = 1;
            bool filled = false;                                         // the ring has gone round
            // after a wait that ran out no barrier is touched any more
            auto going = [&]() { return __shfl_sync(0xffffffffu, *(volatile int *)&abort_flag, 0) == 0; };
            while (w.left > 0) {
                const int n = tree_take(g, w);
                if (n == 0) {
                    if (w.left > 0) tree_next(g, w);
                    continue;
                }
                if (g.q_tma && me == 0) {
                    // the queries, once the scores of the item before are done
                    if (item) tree_wait_warp(&q_empty, (uint32_t)(item - 1) & 1u, &abort_flag, g.err);
                    const int tiles = PAIR && w.tokens > g.tile_tokens ? 2 : 1;
                    const bool go = going();
                    if (go && lane == 0) mbar_arrive_expect_tx(&q_full, (uint32_t)(tiles * CB * 128) * (uint32_t)(w.heads * g.tile_tokens));
                    __syncwarp();
                    if (go && lane < tiles * CB) {
                        const int t = lane / CB, cq = lane % CB;
                        tma_load_3d(qs + t * SLOT + cq * BLOCK, &tq, 64 * cq, w.head, w.q.t0 + w.tok + t * g.tile_tokens, &q_full);
                    }
                }
                item++;
                const int32_t *row = g.p.table + (int64_t)w.q.s * g.p.max_pages;
                auto place = [&](int e, int &nbox, bool &is_v) {         // row of the pool that the lane's box starts at
                    int tile;
                    ring_entry<PAIR>(e, n, tile, is_v);
                    const int r0 = (w.tile + tile) * TT_KT, have = min(TT_KT, w.visible - r0);
                    nbox = have <= 0 ? 0 : (have + box - 1) / box;
                    if (k >= nbox) return 0;
                    const int r = r0 + k * box;
                    int page = row[r / P];
                    if (page < 0 || page >= g.p.n_pages) {
                        atomicCAS(g.err, 0, VB_DEV_TREE_PAGE);
                        page = 0;
                    }
                    return (page * g.p.n_kv_heads + w.g) * P + r % P;
                };
                int nbox;
                bool is_v;
                int y = place(0, nbox, is_v);
                for (int e = 0; e < 2 * n; e++) {
                    int nbox1 = 0;
                    bool is_v1 = false;
                    const int y1 = e + 1 < 2 * n ? place(e + 1, nbox1, is_v1) : 0;
                    tree_wait_warp(&empty[slot], phase, &abort_flag, g.err);
                    const bool go = going();
                    if (go && lane == 0) {
                        if (me == 0 && nbox) mbar_arrive_expect_tx(&full[slot], (uint32_t)nbox * box * 128 * CB);
                        else mbar_arrive(&full[slot]);
                    }
                    if (go && k < nbox)
                        tma_load_2d(ring + (size_t)slot * SLOT + c * BLOCK + k * box * 128, is_v ? &tv : &tk, 64 * c, y, &full[slot]);
                    __syncwarp();
                    if (++slot == n_slots) {
                        slot = 0;
                        phase ^= 1u;
                        filled = true;
                    }
                    y = y1;
                    nbox = nbox1;
                    is_v = is_v1;
                }
                if (w.left > 0) tree_next(g, w);
            }
            // every copy has landed before the CTA can end: the last fill of each
            // slot, in this round of the ring (phase is the parity waited for in
            // it, the opposite of its fills') or the one before
            for (int s = 0; s < n_slots; s++)
                if (s < slot) gm_wait(&full[s], phase ^ 1u);
                else if (filled) gm_wait(&full[s], phase);
            if (g.q_tma && item) gm_wait(&q_full, (uint32_t)(item - 1) & 1u);
        } else if (warp == 9) {
            // --------------------------------------------------------- MMAs
            const uint32_t fmt = TYPE == TR_F16 ? 0u : 1u;
            constexpr uint32_t N_S = (uint32_t)(TT_KT >> 3) << 17, N_O = (uint32_t)(HDP >> 3) << 17;
            const uint32_t id_s = (1u << 4) | (fmt << 7) | (fmt << 10) | ((128u >> 4) << 24) | N_S;
            const uint32_t id_o = (1u << 4) | (fmt << 7) | (fmt << 10) | ((128u >> 4) << 24) | N_O | (1u << 16);   // V: rows along k
            const uint64_t d_q = sw128_desc(qs), d_k = sw128_desc(ring), d_v = sw128_desc_mn(smem_u32(ring));
            // The whole warp goes through the steps, one lane of it issues.
            const uint32_t one = elect_one();
            int item = 0, slot = 0;                   // slot: the ring's next tile, in the order of use
            uint32_t ring_phase = 0, phase = 0;       // phase: parity of p_full, a bit per stream
            auto take = [&]() {
                tree_wait_warp(&full[slot], ring_phase, &abort_flag, g.err);
                const int s = slot;
                if (++slot == n_slots) {
                    slot = 0;
                    ring_phase ^= 1u;
                }
                return (uint32_t)s * (SLOT >> 4);
            };
            while (w.left > 0) {
                const int n = __shfl_sync(0xffffffffu, tree_take(g, w), 0);
                if (n == 0) {
                    if (w.left > 0) tree_next(g, w);
                    continue;
                }
                tree_wait_warp(&q_full, (uint32_t)item & 1u, &abort_flag, g.err);
                // One place of the pipeline: the values of tile j, the scores of the
                // tile that stream t takes next, and one commit for both (a commit
                // holds up the MMAs behind it, and scores that have come say that the
                // values before them are done: no other commit is needed).
                uint32_t v_slot = 0, k_slot = 0;
#pragma unroll 1
                for (int x = -2; x < (PAIR ? 2 * n : n); x++) {
                    const int j = PAIR ? x >> 1 : x, t = x & 1, next = j + (PAIR ? 1 : 2);
                    const bool scores = next >= 0 && next < n;
                    if (!PAIR || t == 0) {
                        if (j >= 0) v_slot = take();
                        if (scores) k_slot = take();
                    }
                    if (j >= 0) {
                        tree_wait_warp(&p_full[t], phase >> t & 1u, &abort_flag, g.err);
                        phase ^= 1u << t;
                    }
                    tc_fence_after();
                    if (j >= 0) {
                        const uint64_t v = d_v + v_slot;
                        const uint32_t p = tmem + 128 * t, o = tmem + 256 + HDP * t;
                        const uint32_t more = PAIR ? j > 0 : j > 1;
#pragma unroll
                        for (int i = 0; i < TT_KT / 16; i++)
                            umma_f16_ts(one, o, p + 8 * i, v + (uint64_t)(i * (2048 >> 4)), id_o, i ? 1u : more);
                    }
                    if (scores) {
                        const uint64_t k = d_k + k_slot, q = d_q + (uint64_t)(PAIR ? t * (SLOT >> 4) : 0);
                        const uint32_t sc = tmem + 128 * t;
#pragma unroll
                        for (int i = 0; i < HDP / 16; i++) {
                            const uint64_t off = (i >> 2) * (BLOCK >> 4) + (i & 3) * 2;
                            umma_f16_ss(one, sc, q + off, k + off, id_s, i ? 1u : 0u);
                        }
                    }
                    if (scores || j >= 0) umma_commit_one(one, scores ? &s_full[t] : &pv_done[t]);
                }
                item++;
                if (w.left > 0) tree_next(g, w);
            }
        }
    } else {
        // -------------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");        // 2 * 176 + 152 = 3 * 168, the launch's share
        const int t = warp >> 2, tid = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;           // TMEM lane of the warp's first row
        const int hd = g.p.head_dim;
        const bool lead = (warp & 3) == 0 && lane == 0;
        int pos = 0, item = 0, seen = 0, ends = 0;                   // tiles and items of this stream so far
        bool first_item = true;
        while (w.left > 0) {
            const int n = tree_take(g, w);
            if (n == 0) {
                if (w.left > 0) tree_next(g, w);
                continue;
            }
            // where TMA cannot: the queries of this stream's row tile (of half of the one tile)
            if (!g.q_tma) {
                uint8_t *qt = qs + (PAIR ? t * SLOT : 0);
                // a thread takes a row (PAIR) or half a row, its loads in flight together
                constexpr int N_C = HDP / 8 / (PAIR ? 1 : 2);          // 16-byte chunks
                const int r = PAIR ? tid : (int)threadIdx.x >> 1, c0 = PAIR ? 0 : (threadIdx.x & 1) * N_C;
                const bool real = tree_token(g, w.tokens, w.heads, PAIR ? t : 0, r) >= 0;
                const uint16_t *src = static_cast<const uint16_t *>(g.a.q) +
                                      (real ? tree_row(g, w.q.t0, w.tok, w.heads, w.head, PAIR ? t : 0, r, g.a.ldq) : 0);
                const int n_c = real ? (hd - 8 * c0) / 8 : 0;              // chunks that exist
                uint4 x[N_C];
                if (g.vec) {
#pragma unroll
                    for (int i = 0; i < N_C; i++)
                        x[i] = i < n_c ? *reinterpret_cast<const uint4 *>(src + 8 * (c0 + i)) : make_uint4(0, 0, 0, 0);
                } else {
#pragma unroll
                    for (int i = 0; i < N_C; i++) {
                        uint32_t y[4] = {};
                        if (i < n_c)
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                y[k] = src[8 * (c0 + i) + 2 * k] | (uint32_t)src[8 * (c0 + i) + 2 * k + 1] << 16;
                        x[i] = make_uint4(y[0], y[1], y[2], y[3]);
                    }
                }
#pragma unroll
                for (int i = 0; i < N_C; i++)
                    *reinterpret_cast<uint4 *>(qt + ((c0 + i) >> 3) * BLOCK + sw128(r, (c0 + i) & 7)) = x[i];
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full);
            }
            const int mrow = 32 * (warp & 3) + lane;                             // this thread's row of the row tile
            const int in_block = tree_token(g, w.tokens, w.heads, PAIR ? t : 0, mrow);
            const bool alive = __any_sync(0xffffffffu, in_block >= 0);           // the warp has rows
            const int j = in_block >= 0 ? w.tok + in_block : -1;
            float m = -INFINITY, l = 0.0f;
            const int mine = PAIR ? n : (n + 1 - t) / 2;                         // tiles of this stream
            for (int x = 0; x < mine; x++, seen++) {
                const int jt = PAIR ? x : 2 * x + t;
                const int r0 = (w.tile + jt) * TT_KT;
                const bool edge = r0 + TT_KT > w.clear;          // not every row is seen by every token
                tree_wait_warp(&s_full[t], (uint32_t)seen & 1u, &abort_flag, g.err);
                tc_fence_after();
                // what the scores' MMAs and those before them read is free again
                if (lead) {
                    if (t == 1 || !PAIR) {
                        mbar_arrive(&empty[(pos + ring_k<PAIR>(jt)) % n_slots]);
                        if (x > 0) mbar_arrive(&empty[(pos + ring_v<PAIR>(jt - (PAIR ? 1 : 2), n)) % n_slots]);
                    }
                    if (g.q_tma && x == mine - 1) mbar_arrive(&q_empty);
                }
                if (edge && (t == 0 || !PAIR)) {
                    // (after the scores: the ring's tiles up to their K have landed, so
                    // this slot's fill before V is over and the parity names V's)
                    // V rows past the end may hold anything: they become zeros,
                    // as do draft values that are not finite
                    const int at = pos + ring_v<PAIR>(jt, n);
                    tree_wait_warp(&full[at % n_slots], (uint32_t)(at / n_slots) & 1u, &abort_flag, g.err);
                    uint8_t *v = ring + (size_t)(at % n_slots) * SLOT;
                    bool found = false;
                    const int from = max(0, w.clear - r0);
                    for (int e = from * CB * 8 + tid; e < TT_KT * CB * 8; e += 128) {
                        const int r = e / (CB * 8), c = e % (CB * 8);
                        uint4 *p = reinterpret_cast<uint4 *>(v + (c >> 3) * BLOCK + sw128(r, c & 7));
                        if (r0 + r >= w.visible) *p = make_uint4(0, 0, 0, 0);
                        else {
                            bool here = false;
                            const uint4 y = tree_finite<TYPE>(*p, here);
                            if (here) *p = y;
                            found |= here;
                        }
                    }
                    if (found) not_finite[item & 1] = item;
                    __syncwarp();
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                if (alive) {
                    const uint32_t sc = tmem + 128 * t + lanes;
                    // columns that this row does not see, 32 to a word
                    uint32_t gone[4] = {};
                    if (edge) {
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const int d = r0 + 32 * k - w.q.base;                // draft place of the first column
                            int lim = w.visible - (r0 + 32 * k);
                            uint32_t bits = 0xffffffffu;
                            if (!g.a.mask) lim = min(lim, j + 1 - d);
                            else if (d > -32 && j >= 0) {
                                const uint32_t *row = g.a.mask + (int64_t)(w.q.t0 + j) * g.a.mask_words;
                                if (d < 0) bits = (row[0] << -d) | ((1u << -d) - 1u);
                                else {
                                    const int k0 = d >> 5;
                                    const uint32_t lo = k0 < g.a.mask_words ? row[k0] : 0u;
                                    const uint32_t hi = k0 + 1 < g.a.mask_words ? row[k0 + 1] : 0u;
                                    bits = __funnelshift_r(lo, hi, d & 31);
                                }
                            }
                            if (j < 0 || lim <= 0) bits = 0u;
                            else if (lim < 32) bits &= (1u << lim) - 1u;
                            gone[k] = ~bits;
                        }
                    }
                    // One pass over the row in pieces of 32, the next on its way from
                    // tensor memory: the weights against the running maximum as it
                    // stands (in an item's first tile that of the first piece), and the
                    // row's own maximum beside them.  They count if that maximum is no
                    // further than 2^TT_SLACK above and there was no NaN and no infinite
                    // score (whose NaN exp2_pair would not keep); else two
                    // passes, the maximum first.  (The weights wait in registers: in
                    // tensor memory they would take the scores' place.)
                    uint32_t a[32], b[32];
                    bool done = false;
                    auto one_pass = [&](auto is_masked) {
                        constexpr bool masked = decltype(is_masked)::value;
                        auto drop = [&](uint32_t (&v)[32], uint32_t out) {
                            if constexpr (masked)
#pragma unroll
                                for (int c = 0; c < 32; c++)
                                    if (out >> c & 1u) v[c] = 0xff800000u;
                        };
                        tmem_ld32_start(sc, a);
                        tmem_ld32_wait(a);
                        drop(a, gone[0]);
                        if (x == 0) {                                    // no maximum yet: that of the first piece
                            float u = -INFINITY, v = -INFINITY;
#pragma unroll
                            for (int c = 0; c < 16; c++) {
                                float &z = c & 1 ? v : u;
                                z = max3_nan(z, __uint_as_float(a[2 * c]), __uint_as_float(a[2 * c + 1]));
                            }
                            m = max3_nan(u, v, v) * g.scale_log2;
                        }
                        const uint64_t off2 = pack_f32x2(-m, -m), scale2 = pack_f32x2(g.scale_log2, g.scale_log2);
                        uint32_t y[2][32];
                        uint64_t sum2 = 0;
                        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            uint32_t (&now)[32] = k & 1 ? b : a;
                            if (k < 3) tmem_ld32_start(sc + 32 * (k + 1), k & 1 ? a : b);
                            if (k > 0) drop(now, gone[k]);
#pragma unroll
                            for (int c = 0; c < 16; c++) {
                                float &z = c & 1 ? t1 : t0;
                                z = max3_nan(z, __uint_as_float(now[2 * c]), __uint_as_float(now[2 * c + 1]));
                                const uint64_t v = fma_f32x2(pack_b32x2(now[2 * c], now[2 * c + 1]), scale2, off2);
                                float p0, p1;
                                if (!masked && c % 16 < TT_POLY) exp2_pair(v, p0, p1);    // (which makes no 0 of -inf)
                                else {
                                    unpack_f32x2(v, p0, p1);
                                    p0 = ex2(p0);
                                    p1 = ex2(p1);
                                }
                                sum2 = add_f32x2(sum2, pack_f32x2(p0, p1));
                                y[k >> 1][16 * (k & 1) + c] = pack2<TYPE>(p0, p1);
                            }
                            if (k < 3) tmem_ld32_wait(k & 1 ? a : b);
                        }
                        const float top = max3_nan(t0, t1, t1) * g.scale_log2;
                        done = !__any_sync(0xffffffffu, j >= 0 && (!(top <= m + TT_SLACK) || m == -INFINITY || top == INFINITY));
                        if (done) {
                            tmem_st32(sc, y[0]);
                            tmem_st32(sc + 32, y[1]);
                            float s0, s1;
                            unpack_f32x2(sum2, s0, s1);
                            l += s0 + s1;
                            tmem_st_wait();
                        }
                    };
                    if (edge) one_pass(std::true_type());
                    else one_pass(std::false_type());
                    if (!done) {
                    float top = -INFINITY;
                    auto piece_max = [&](uint32_t (&x)[32], uint32_t out) {
                        if (edge)
#pragma unroll
                            for (int c = 0; c < 32; c++)
                                if (out >> c & 1u) x[c] = 0xff800000u;
                        float u = top, v = __uint_as_float(x[0]);
#pragma unroll
                        for (int c = 1; c < 31; c += 2) {
                            float &z = (c >> 1) & 1 ? v : u;
                            z = fmaxf(z, fmaxf(__uint_as_float(x[c]), __uint_as_float(x[c + 1])));
                        }
                        top = fmaxf(fmaxf(u, v), __uint_as_float(x[31]));
                    };
                    tmem_ld32_start(sc, a);
                    tmem_ld32_wait(a);
#pragma unroll 1
                    for (int k = 0; k < 4; k += 2) {
                        tmem_ld32_start(sc + 32 * k + 32, b);
                        piece_max(a, k ? gone[2] : gone[0]);
                        tmem_ld32_wait(b);
                        tmem_ld32_start(sc + (k ? 0 : 64), a);          // after the last: the first again, for the weights
                        piece_max(b, k ? gone[3] : gone[1]);
                        tmem_ld32_wait(a);
                    }
                    const float now = top * g.scale_log2;
                    const bool move = now > m + TT_SLACK || (m == -INFINITY && now > m);
                    if (x == 0) m = now;
                    else if (__any_sync(0xffffffffu, move)) {
                        const float f = move ? ex2(m - now) : 1.0f;
                        if (move) m = now;
                        l *= f;
                        // (the scores have come, so the values before them are done)
#pragma unroll 1
                        for (int k = 0; k < HDP / 32; k++) {
                            float o[32];
                            uint32_t y[32];
                            tmem_ld32(tmem + 256 + HDP * t + lanes + 32 * k, o);
#pragma unroll
                            for (int c = 0; c < 32; c++) y[c] = __float_as_uint(o[c] * f);
                            tmem_st32(tmem + 256 + HDP * t + lanes + 32 * k, y);
                        }
                    }
                    const float off = m == -INFINITY ? 0.0f : -m;
                    const uint64_t off2 = pack_f32x2(off, off), scale2 = pack_f32x2(g.scale_log2, g.scale_log2);
                    uint64_t sum2 = 0;
                    auto piece_exp = [&](uint32_t (&x)[32], uint32_t out, uint32_t dst) {
                        if (edge)
#pragma unroll
                            for (int c = 0; c < 32; c++)
                                if (out >> c & 1u) x[c] = 0xff800000u;
                        uint32_t y[16];
#pragma unroll
                        for (int c = 0; c < 16; c++) {
                            float p0, p1;
                            unpack_f32x2(fma_f32x2(pack_b32x2(x[2 * c], x[2 * c + 1]), scale2, off2), p0, p1);
                            p0 = ex2(p0);
                            p1 = ex2(p1);
                            sum2 = add_f32x2(sum2, pack_f32x2(p0, p1));
                            y[c] = pack2<TYPE>(p0, p1);
                        }
                        tmem_st16(dst, y);
                    };
#pragma unroll 1
                    for (int k = 0; k < 4; k += 2) {
                        tmem_ld32_start(sc + 32 * k + 32, b);
                        piece_exp(a, k ? gone[2] : gone[0], sc + 16 * k);
                        tmem_ld32_wait(b);
                        tmem_ld32_start(sc + 64, a);                    // (not used after the last)
                        piece_exp(b, k ? gone[3] : gone[1], sc + 16 * k + 16);
                        tmem_ld32_wait(a);
                    }
                    float s0, s1;
                    unpack_f32x2(sum2, s0, s1);
                    l += s0 + s1;
                    tmem_st_wait();
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[t]);
            }
            if (mine > 0) {
                tree_wait_warp(&pv_done[t], (uint32_t)ends & 1u, &abort_flag, g.err);
                ends++;
                if (lead && (t == 1 || !PAIR)) mbar_arrive(&empty[(pos + ring_v<PAIR>(PAIR ? n - 1 : 2 * mine - 2 + t, n)) % n_slots]);
            } else if (lead && g.q_tma) {
                mbar_arrive(&q_empty);
            }

            // ---- the block's result, or this CTA's part of it
            const bool whole = n == w.units;
            float f0 = 1.0f, f1 = 0.0f;
            if (!PAIR) {
                ml[t][tid] = make_float2(m, l);
                tc_fence_before();
                consumer_sync(256);
                const float2 a = ml[0][tid], b = ml[1][tid];
                m = fmaxf(a.x, b.x);
                const float off = m == -INFINITY ? 0.0f : m;
                f0 = ex2(a.x - off);
                f1 = ex2(b.x - off);
                l = a.y * f0 + b.y * f1;
            }
            tc_fence_after();
            const bool mend = *(volatile int *)&not_finite[item & 1] == item;
            if (alive) {
                const int64_t out = tree_row(g, w.q.t0, w.tok, w.heads, w.head, PAIR ? t : 0, mrow, g.a.ldo);
                const float inv = whole ? (l > 0.0f || l != l ? 1.0f / l : 0.0f) : 1.0f;
                float *part = g.part + (size_t)(2 * blockIdx.x + (first_item ? 0 : 1)) * (hd + 2) * MT + (PAIR ? 128 * t : 0) + mrow;
                if (!whole && (PAIR || t == 0)) {
                    part[(size_t)hd * MT] = m;
                    part[(size_t)(hd + 1) * MT] = l;
                }
                // PAIR: all columns of the thread's row; else half of them, of both streams
                const int c_lo = PAIR ? 0 : t * (HDP / 2), c_hi = min(hd, PAIR ? HDP : c_lo + HDP / 2);
                f0 *= inv;
                f1 *= inv;
#pragma unroll 1
                for (int c0 = c_lo; c0 < c_hi; c0 += 32) {
                    float o[32];
                    tmem_ld32(tmem + 256 + (PAIR ? HDP * t : 0) + lanes + c0, o);
                    if (!PAIR && n > 1) {
                        float o1[32];
                        tmem_ld32(tmem + 256 + HDP + lanes + c0, o1);
#pragma unroll
                        for (int c = 0; c < 32; c++) o[c] = o[c] * f0 + o1[c] * f1;
                    } else {
#pragma unroll
                        for (int c = 0; c < 32; c++) o[c] *= f0;
                    }
                    if (j < 0) continue;
                    if (!whole) {
#pragma unroll
                        for (int c = 0; c < 32; c++)
                            if (c0 + c < hd) part[(size_t)(c0 + c) * MT] = o[c];
                    } else {
#pragma unroll
                        for (int c = 0; c < 32; c += 8) {
                            const float y[8] = {o[c], o[c + 1], o[c + 2], o[c + 3], o[c + 4], o[c + 5], o[c + 6], o[c + 7]};
                            if (c0 + c < hd) tree_store8<TYPE>(g, out + c0 + c, y);
                        }
                    }
                }
                if (mend && j >= 0) {
                    const int lo = max(w.clear, w.tile * TT_KT), hi = min(w.visible, (w.tile + n) * TT_KT);
                    void *dst = whole ? static_cast<void *>(static_cast<uint16_t *>(g.a.out) + out) : part;
                    tree_not_finite<TYPE>(&g, w.q.t0, w.q.s, w.q.base, w.g, j, lo, hi, c_lo, c_hi, dst, whole ? 1 : MT, !whole);
                }
            }
            __syncwarp();
            tc_fence_before();
            if (!PAIR) consumer_sync(256);           // both streams' sums are read: the next item may overwrite them
            if (threadIdx.x == 0) tree_describe(g, w, line, n, first_item);
            __syncwarp();
            first_item = false;
            pos += 2 * n;
            item++;
            if (w.left > 0) tree_next(g, w);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// -------------------------------------------------------------------- host
template <int TYPE, int HDP, bool PAIR>
static int launch_tc(vb_ctx *ctx, TreeArgs &g) {
    constexpr size_t slot = (size_t)HDP / 64 * TT_KT * 128, q = (PAIR ? 2 : 1) * slot;
    const vb_pages &p = g.p;
    const size_t rest = 1024 + q + (PAIR ? 0 : 2 * 128 * sizeof(float2));
    g.stages = (int)std::min<size_t>(TT_SLOTS, (TT_SMEM - rest) / slot);
    const size_t smem = rest + g.stages * slot;
    int rc = tree_prepare(ctx, g, 128, PAIR ? 2 : 1, TT_KT, TT_OVER);
    if (rc) return rc;
    CUtensorMap tk, tv, tq;
    const int64_t rows = (int64_t)p.n_pages * p.n_kv_heads * p.page_rows, layer = (int64_t)g.a.layer * rows * p.head_dim * 2;
    const CUtensorMapDataType dt = p.type == VB_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const int box = std::min(p.page_rows, TT_KT);
    if (!make_map(&tk, static_cast<char *>(p.k) + layer, dt, 2, p.head_dim, rows, 64, box, true) ||
        !make_map(&tv, static_cast<char *>(p.v) + layer, dt, 2, p.head_dim, rows, 64, box, true))
        return set_error(ctx, VB_ERR_BACKEND, "vb_tree_attention: tensor map of the cache refused");
    // queries whose rows TMA can gather: a box is the heads of tile_tokens tokens
    g.q_tma = g.vec && g.chunks == 1;
    if (!g.q_tma) tq = tk;
    else if (!make_map_3d(&tq, g.a.q, dt, p.head_dim, g.a.n_heads, g.a.n_tokens, (int64_t)p.head_dim * 2, g.a.ldq * 2, 64, g.group,
                          g.tile_tokens))
        return set_error(ctx, VB_ERR_BACKEND, "vb_tree_attention: tensor map of the queries refused");
    rc = tree_allow(ctx, reinterpret_cast<const void *>(tree_tc_kernel<TYPE, HDP, PAIR>), TT_SMEM);
    if (rc) return rc;
    VB_CHECK(ctx, pdl_launch(ctx, tree_tc_kernel<TYPE, HDP, PAIR>, dim3(ctx->sm_count), dim3(TT_THREADS), smem, tk, tv, tq, g));
    VB_LAUNCH_CHECK(ctx, "tree_tc");
    return launch_tree_combine(ctx, g);
}

template <int TYPE, int HDP>
static int launch_tc_rows(vb_ctx *ctx, TreeArgs &g) {
    return g.a.max_tokens > std::max(1, 128 / g.group) ? launch_tc<TYPE, HDP, true>(ctx, g) : launch_tc<TYPE, HDP, false>(ctx, g);
}

int launch_tree_tc(vb_ctx *ctx, TreeArgs &g) {
    if (g.a.type == VB_TYPE_F16)
        return g.p.head_dim <= 64 ? launch_tc_rows<TR_F16, 64>(ctx, g) : launch_tc_rows<TR_F16, 128>(ctx, g);
    return g.p.head_dim <= 64 ? launch_tc_rows<TR_BF16, 64>(ctx, g) : launch_tc_rows<TR_BF16, 128>(ctx, g);
}

}  // namespace vb
