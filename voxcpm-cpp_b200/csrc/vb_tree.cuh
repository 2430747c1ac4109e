// vb_tree.cuh -- what the kernels of the drafted-token attention share: the
// arguments, the line of work units and its cut over the CTAs, and small
// device helpers.
#pragma once

#include "vb_common.cuh"
#include "vb_tc.cuh"

namespace vb {

enum { TR_F32 = 0, TR_BF16 = 1, TR_F16 = 2 };

struct TreeArgs {
    vb_tree_args a;
    vb_pages p;
    float scale_log2;                // scale * log2(e): the softmax runs in powers of two
    int group;                       // query heads per K/V head
    int mt;                          // rows per block
    int kt;                          // cache rows per tile
    int stages;
    int vec;                         // 16-byte accesses of q and out
    int *err;
    float *part;                     // [2 * CTAs][head_dim + 2][mt]: sums, then the maximum and the sum of the weights
    struct TreeShare *share;         // [CTAs]
};

// Sequence i of the call.  T = 0: no rows of q (or none that can be named);
// bad: its tokens get zeros.
struct TreeSeq {
    int t0, T, s, len, base, bad;
};

__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs &g, int i) {
    TreeSeq q;
    const vb_tree_args &a = g.a;
    q.t0 = a.start[i];
    const int t1 = a.start[i + 1];
    q.s = a.seqs[i];
    q.T = t1 - q.t0;
    q.bad = 0;
    if (q.t0 < 0 || t1 < q.t0 || t1 > a.n_tokens || q.T > a.max_tokens) {
        q.T = 0;
        q.bad = 1;
        q.len = q.base = 0;
        return q;
    }
    q.len = q.s >= 0 && q.s < g.p.n_seqs ? g.p.length[q.s] : -1;
    q.base = q.len - q.T;
    if (q.base < 0 || (int64_t)q.len > (int64_t)g.p.max_pages * g.p.page_rows ||
        (a.mask && q.T > 32 * (int64_t)a.mask_words)) {
        q.bad = 1;
        q.len = q.base = 0;
    }
    return q;
}

__device__ __forceinline__ int tree_blocks(const TreeArgs &g, const TreeSeq &q) {
    return (q.T * g.group + g.mt - 1) / g.mt;
}

// Rows of the cache that block b of a sequence reads, and its units (at
// least one, so that every output row is written).
__device__ __forceinline__ int tree_visible(const TreeArgs &g, const TreeSeq &q, int b) {
    if (q.bad) return 0;
    if (g.a.mask) return q.len;
    return q.base + min(q.T, ((b + 1) * g.mt + g.group - 1) / g.group);
}

// Of those, the rows that every token of the block sees.
__device__ __forceinline__ int tree_clear(const TreeArgs &g, const TreeSeq &q, int b) {
    return g.a.mask || q.bad ? q.base : q.base + b * g.mt / g.group + 1;
}

__device__ __forceinline__ int tree_units(const TreeArgs &g, int visible) { return max(1, (visible + g.kt - 1) / g.kt); }

__device__ __forceinline__ int64_t tree_seq_units(const TreeArgs &g, const TreeSeq &q) {
    const int nb = tree_blocks(g, q);
    if (g.a.mask || q.bad) return (int64_t)nb * tree_units(g, tree_visible(g, q, 0)) * g.p.n_kv_heads;
    int64_t u = 0;
    for (int b = 0; b < nb; b++) u += tree_units(g, tree_visible(g, q, b));
    return u * g.p.n_kv_heads;
}

// A place in the line of units: the item (i, kv head, block) and the tile.
struct TreeWalk {
    TreeSeq q;
    int i, g, b, nb, visible, clear, units, tile;
    int64_t left;                    // units of this CTA from here on
};

__device__ __forceinline__ void tree_item(const TreeArgs &g, TreeWalk &w) {
    w.visible = tree_visible(g, w.q, w.b);
    w.clear = tree_clear(g, w.q, w.b);
    w.units = tree_units(g, w.visible);
}

__device__ __forceinline__ void tree_next(const TreeArgs &g, TreeWalk &w) {
    w.tile = 0;
    if (++w.b == w.nb) {
        w.b = 0;
        if (++w.g == g.p.n_kv_heads) {
            w.g = 0;
            do w.q = tree_seq(g, ++w.i);
            while (w.q.T == 0);
            w.nb = tree_blocks(g, w.q);
        }
    }
    tree_item(g, w);
}

// The part of the line of units that this CTA works on, found by all its
// threads together (THREADS of them): the first place in w, whose `left` is 0
// when there is none.  `total` and `ctas` describe the whole cut: CTA c has
// the units c * total / ctas up to (c + 1) * total / ctas.
struct TreeCut {
    int64_t scan[32], off;
    int seq;
};

template <int THREADS>
__device__ __forceinline__ void tree_cut(const TreeArgs &g, TreeCut &sh, TreeWalk &w, int64_t &u1, int64_t &total,
                                         int64_t &ctas) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n = g.a.n;
    const int per = (n + THREADS - 1) / THREADS;
    const int i0 = min(n, (int)threadIdx.x * per), i1 = min(n, i0 + per);
    int64_t mine = 0;
    for (int i = i0; i < i1; i++) {
        const TreeSeq q = tree_seq(g, i);
        if (q.bad && blockIdx.x == 0) atomicCAS(g.err, 0, VB_DEV_TREE_SEQ);
        mine += tree_seq_units(g, q);
    }
    int64_t before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += y;
    }
    if (lane == 31) sh.scan[warp] = before;
    before -= mine;
    __syncthreads();
    total = 0;
    for (int k = 0; k < THREADS / 32; k++) {
        if (k < warp) before += sh.scan[k];
        total += sh.scan[k];
    }
    ctas = min((int64_t)gridDim.x, total);
    const int64_t u0 = blockIdx.x < ctas ? blockIdx.x * total / ctas : total;
    u1 = blockIdx.x < ctas ? (blockIdx.x + 1) * total / ctas : total;
    if (u0 >= before && u0 < before + mine) {
        int64_t at = before;
        for (int i = i0; i < i1; i++) {
            const int64_t u = tree_seq_units(g, tree_seq(g, i));
            if (u0 < at + u) {
                sh.seq = i;
                sh.off = u0 - at;
                break;
            }
            at += u;
        }
    }
    if (threadIdx.x == 0) g.share[blockIdx.x].last = -1;
    __syncthreads();
    w.left = u1 - u0;
    if (w.left <= 0) return;
    w.i = sh.seq;
    w.q = tree_seq(g, w.i);
    w.nb = tree_blocks(g, w.q);
    const int64_t head_units = tree_seq_units(g, w.q) / g.p.n_kv_heads;
    w.g = (int)(sh.off / head_units);
    int64_t off = sh.off % head_units;
    w.b = 0;
    tree_item(g, w);
    if (g.a.mask || w.q.bad) {                          // blocks of equal length
        w.b = (int)(off / w.units);
        off %= w.units;
    } else {
        while (off >= w.units) {
            off -= w.units;
            w.b++;
            tree_item(g, w);
        }
    }
    w.tile = (int)off;
}

// An item that goes on in the next CTAs: described by the CTA that holds its
// first unit (`at`), as its last item.
struct TreeShare {
    int i, g, b, slot, last, pad[3];        // last: the CTA of its last unit; -1: no such item
};

__device__ __forceinline__ void tree_describe(const TreeArgs &g, const TreeWalk &w, int64_t at, int64_t total,
                                              int64_t ctas, bool first_item) {
    const int64_t end = at + w.units - 1;
    g.share[blockIdx.x] = {w.i, w.g, w.b, (int)blockIdx.x * 2 + (first_item ? 0 : 1), (int)(((end + 1) * ctas - 1) / total), {}};
}

// Whether token j of the sequence sees draft row d (0 <= d < T).
__device__ __forceinline__ bool tree_sees(const TreeArgs &g, const TreeSeq &q, int j, int d) {
    return g.a.mask ? g.a.mask[(int64_t)(q.t0 + j) * g.a.mask_words + (d >> 5)] >> (d & 31) & 1u : d <= j;
}

template <int TYPE>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if constexpr (TYPE == TR_F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

template <int TYPE>
__device__ __forceinline__ float unpack(uint16_t h) {
    if constexpr (TYPE == TR_F16) return h2f(h);
    else return bf16_to_f(h);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Byte offset of 16-byte chunk c of row r in a [rows][128 B] tile with the
// 128-byte swizzle that TMA writes.
__device__ __forceinline__ uint32_t sw128(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

// A bounded barrier wait; the first that runs out records the error and
// lets every later wait of the CTA return at once.
__device__ __forceinline__ void tree_wait(uint64_t *bar, uint32_t parity, volatile int *abort, int *err) {
    if (mbar_try_wait(bar, parity)) return;
    if (*abort) return;
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity)) {
        if (*abort) return;
        if (clock64() - t0 > WAIT_LIMIT_CYCLES) {
            *abort = 1;
            atomicCAS(err, 0, VB_DEV_TREE_WAIT);
            return;
        }
    }
}

// The same by all lanes of a warp, which go on together: what follows
// (ldmatrix, mma, tcgen05.ld) takes part of its operands from every lane.
__device__ __forceinline__ void tree_wait_warp(uint64_t *bar, uint32_t parity, volatile int *abort, int *err) {
    tree_wait(bar, parity, abort, err);
    __syncwarp();
}

// Values of draft rows that are not finite are taken out of the tiles that
// not every token sees (a zero weight times infinity would reach those that
// do not).  This puts them back: in result columns c0 .. c1-1 of token j, dst
// (`stride` apart) becomes the sum of those that the token does see among
// cache rows lo .. hi-1 (not before the draft), where it sees any.  P: how a
// result is stored.  Rare, and kept out of the kernels' code for that.
template <int TYPE>
__device__ __noinline__ void tree_not_finite(const TreeArgs *g, int t0, int s, int base, int kv, int j, int lo, int hi, int c0,
                                             int c1, void *dst, int64_t stride, int as_float) {
    for (int c = c0; c < c1; c++) {
        float sum = 0.0f;
        bool any = false;
        for (int r = lo; r < hi; r++) {
            const int d = r - base;
            if (!(g->a.mask ? g->a.mask[(int64_t)(t0 + j) * g->a.mask_words + (d >> 5)] >> (d & 31) & 1u : d <= j)) continue;
            int page = g->p.table[(int64_t)s * g->p.max_pages + r / g->p.page_rows];
            if (page < 0 || page >= g->p.n_pages) page = 0;
            const int64_t at = ((((int64_t)g->a.layer * g->p.n_pages + page) * g->p.n_kv_heads + kv) * g->p.page_rows +
                                r % g->p.page_rows) * g->p.head_dim + c;
            const float v = unpack<TYPE>(static_cast<const uint16_t *>(g->p.v)[at]);
            if (isfinite(v)) continue;
            sum += v;
            any = true;
        }
        if (!any) continue;
        if (as_float) static_cast<float *>(dst)[c * stride] = sum;
        else static_cast<uint16_t *>(dst)[c * stride] = (uint16_t)pack2<TYPE>(sum, 0.0f);
    }
}

// 16 bytes of V with the values that are not finite set to zero; found: there were some.
template <int TYPE>
__device__ __forceinline__ uint4 tree_finite(uint4 v, bool &found) {
    const uint32_t inf = TYPE == TR_F16 ? 0x7c00u : 0x7f80u;
    uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if ((x[k] & inf) == inf) {
            x[k] &= 0xffff0000u;
            found = true;
        }
        if ((x[k] >> 16 & inf) == inf) {
            x[k] &= 0xffffu;
            found = true;
        }
    }
    return make_uint4(x[0], x[1], x[2], x[3]);
}

// Eight results of a row, at element `at` of the output.
template <int TYPE>
__device__ __forceinline__ void tree_store8(const TreeArgs &g, int64_t at, const float (&y)[8]) {
    if constexpr (TYPE == TR_F32) {
        float *dst = static_cast<float *>(g.a.out) + at;
        if (g.vec) {
            reinterpret_cast<float4 *>(dst)[0] = make_float4(y[0], y[1], y[2], y[3]);
            reinterpret_cast<float4 *>(dst)[1] = make_float4(y[4], y[5], y[6], y[7]);
        } else {
#pragma unroll
            for (int c = 0; c < 8; c++) dst[c] = y[c];
        }
    } else {
        uint16_t *dst = static_cast<uint16_t *>(g.a.out) + at;
        uint32_t z[4];
#pragma unroll
        for (int c = 0; c < 4; c++) z[c] = pack2<TYPE>(y[2 * c], y[2 * c + 1]);
        if (g.vec) *reinterpret_cast<uint4 *>(dst) = make_uint4(z[0], z[1], z[2], z[3]);
        else {
#pragma unroll
            for (int c = 0; c < 8; c++) dst[c] = (uint16_t)(z[c >> 1] >> (16 * (c & 1)));
        }
    }
}

int launch_tree_tc(vb_ctx *ctx, TreeArgs &g);
int init_tree_tc(vb_ctx *ctx);
int tree_workspace(vb_ctx *ctx, TreeArgs &g);
int launch_tree_combine(vb_ctx *ctx, const TreeArgs &g);

}  // namespace vb
