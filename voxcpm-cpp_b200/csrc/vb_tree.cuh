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
    int tile_rows;                   // rows of a row tile
    int tile_tokens;                 // tokens of a row tile
    int tb;                          // tokens of a block, of one or two row tiles
    int mt;                          // rows of a block's parts: tile_rows for each row tile
    int chunks;                      // blocks that share a token's heads (1 unless group > tile_rows)
    int kt_log2;                     // cache rows per tile, a power of two
    int over;                        // what an item costs beside its tiles, in tiles
    int by_item;                     // `share` goes by item, not by CTA
    int item_blocks;                 // most blocks of a sequence, for that
    int stages;
    int vec;                         // 16-byte accesses of q and out
    int q_tma;                       // tcgen05 kernel: TMA loads the queries
    int *err;
    float *part;                     // [2 * CTAs][head_dim + 2][mt]: sums, then the maximum and the sum of the weights
    struct TreeShare *share;         // [CTAs], or [n][n_kv][item_blocks]
};

// Sequence i of the call.  T = 0: no rows of q (or none that can be named);
// bad: its tokens get zeros.  So do all while an error of a page call waits to
// be read: the newest rows are then not those of the call's tokens.
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
    if (g.p.status[0] != 0 || q.base < 0 || (int64_t)q.len > (int64_t)g.p.max_pages * g.p.page_rows ||
        (a.mask && q.T > 32 * (int64_t)a.mask_words)) {
        q.bad = 1;
        q.len = q.base = 0;
    }
    return q;
}

// A block: tb tokens with the heads of one K/V head (or, where those are more
// than tile_rows, with a chunk of tile_rows of them).  Row r of its row tile
// t is token t * tile_tokens + r / heads, head r % heads.  Tiles of a block:
// those of the cache rows that its last token sees, at least one, so that
// every output row is written.  In the line of units it counts `over` units
// more, before them.  The host refuses calls whose units could pass 2^31.
__device__ __forceinline__ int tree_units(const TreeArgs &g, int visible) {
    return max(1, (visible + (1 << g.kt_log2) - 1) >> g.kt_log2);
}

// sum of floor((a k + b) / 2^s) over k = 0 .. n-1, a and b not negative.
static __device__ __noinline__ uint32_t tree_floor_sum(uint32_t n, int s, uint32_t a, uint32_t b) {
    uint64_t sum = 0, m = (uint64_t)1 << s, aa = a, bb = b, nn = n;
    while (nn) {                                      // Euclid on (a, m)
        sum += (uint64_t)(uint32_t)(aa / m) * (nn * (nn - 1) / 2) + (bb / m) * nn;
        aa %= m;
        bb %= m;
        const uint64_t y = aa * nn + bb;
        if (y < m) break;
        nn = y / m;
        bb = y % m;
        const uint64_t t = m;
        m = aa;
        aa = t;
    }
    return (uint32_t)sum;
}

// Units of the first k token blocks (one chunk, one K/V head).
__device__ __forceinline__ int tree_units_before(const TreeArgs &g, const TreeSeq &q, int k) {
    if (g.a.mask || q.bad) return k * (g.over + tree_units(g, q.len));
    const int kt = 1 << g.kt_log2, whole = min(k, q.T / g.tb);       // blocks of tb tokens
    int u = k * g.over;
    if (k <= 4 || g.tb >= kt) {
        for (int j = 0; j < whole; j++) u += tree_units(g, q.base + (j + 1) * g.tb);
    } else if ((g.tb & (g.tb - 1)) == 0) {
        // tb divides kt: sum of floor((j + c) / r), r = kt / tb
        const int r_log2 = g.kt_log2 - (31 - __clz(g.tb)), c = (q.base + g.tb + kt - 1) / g.tb;
        auto sum = [&](int64_t x) {                   // of floor(i / r) for i < x
            const int64_t m = x >> r_log2;
            return (m * (m - 1) / 2 << r_log2) + m * (x - (m << r_log2));
        };
        u += (int)(sum((int64_t)whole + c) - sum(c));
    } else {
        u += (int)tree_floor_sum(whole, g.kt_log2, g.tb, q.base + g.tb + kt - 1);
    }
    return u + (k > whole ? tree_units(g, q.len) : 0);
}

__device__ __forceinline__ int tree_token_blocks(const TreeArgs &g, const TreeSeq &q) { return (q.T + g.tb - 1) / g.tb; }

// A place in the line of units.
struct TreeWalk {
    TreeSeq q;
    int i, g, b, chunk;              // the item: sequence, K/V head, block, chunk of heads
    int at, pos, left;               // the item's first unit, the place in it, units of this CTA from here on
    int visible, clear, units;       // rows that its last token sees; that every token sees; tiles
    int tok, tokens, heads, head;    // first token and their number, heads and the first of them
    int tile;                        // first tile of this CTA's part
};

__device__ __forceinline__ void tree_item(const TreeArgs &g, TreeWalk &w) {
    w.tok = w.b * g.tb;
    w.tokens = min(g.tb, w.q.T - w.tok);
    const int h0 = w.chunk * g.tile_rows;
    w.heads = min(g.tile_rows, g.group - h0);
    w.head = w.g * g.group + h0;
    const bool chain = !g.a.mask && !w.q.bad;
    w.visible = chain ? w.q.base + w.tok + w.tokens : w.q.len;
    w.clear = chain ? w.q.base + w.tok + 1 : w.q.base;
    w.units = tree_units(g, w.visible);
}

// Takes this CTA's part of the item: its tiles from w.tile on, their number
// (none when only the item's extra units fell to this CTA).
__device__ __forceinline__ int tree_take(const TreeArgs &g, TreeWalk &w) {
    const int n = min(g.over + w.units - w.pos, w.left);
    w.tile = max(0, w.pos - g.over);
    w.pos += n;
    w.left -= n;
    return max(0, w.pos - g.over) - w.tile;
}

__device__ __forceinline__ void tree_next(const TreeArgs &g, TreeWalk &w) {
    w.pos = 0;
    w.at += g.over + w.units;
    if (++w.chunk == g.chunks) {
        w.chunk = 0;
        if (++w.b * g.tb >= w.q.T) {
            w.b = 0;
            if (++w.g == g.p.n_kv_heads) {
                w.g = 0;
                do w.q = tree_seq(g, ++w.i);
                while (w.q.T == 0);
            }
        }
    }
    tree_item(g, w);
}

// The cut of the line: `ctas` CTAs get total / ctas units each, the first
// total % ctas one more.
struct TreeLine {
    int total, ctas, each, more;
    __device__ __forceinline__ int first(int c) const { return c * each + min(c, more); }
    __device__ __forceinline__ int owner(int u) const {
        const int head = more * (each + 1);
        return u < head ? u / (each + 1) : more + (u - head) / each;
    }
};

// The part of the line that this CTA works on, found by all its threads
// together (THREADS of them): the first place in w, whose `left` is 0 when
// there is none.
struct TreeCut {
    TreeSeq q;
    int scan[32], seq, off, b, rest;
};

template <int THREADS>
__device__ __forceinline__ void tree_cut(const TreeArgs &g, TreeCut &sh, TreeWalk &w, TreeLine &line) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = g.a.n, heads = g.p.n_kv_heads * g.chunks;
    const int per = (n + THREADS - 1) / THREADS;
    const int i0 = min(n, (int)threadIdx.x * per), i1 = min(n, i0 + per);
    int mine = 0;
    TreeSeq q;
    for (int i = i0; i < i1; i++) {
        q = tree_seq(g, i);
        if (q.bad && blockIdx.x == 0) atomicCAS(g.err, 0, VB_DEV_TREE_SEQ);
        mine += heads * tree_units_before(g, q, tree_token_blocks(g, q));
    }
    int before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += y;
    }
    if (lane == 31) sh.scan[warp] = before;
    before -= mine;
    if (!g.by_item && threadIdx.x == 0) g.share[blockIdx.x].last = -1;
    __syncthreads();
    line.total = 0;
#pragma unroll
    for (int k = 0; k < THREADS / 32; k++) {
        const int x = sh.scan[k];
        if (k < warp) before += x;
        line.total += x;
    }
    w.left = 0;
    line.ctas = min((int)gridDim.x, line.total);
    if (line.ctas == 0) return;
    line.each = line.total / line.ctas;
    line.more = line.total - line.each * line.ctas;
    const int u0 = line.first(min((int)blockIdx.x, line.ctas)), u1 = line.first(min((int)blockIdx.x + 1, line.ctas));
    if (u0 >= before && u0 < before + mine) {
        int at = before;
        for (int i = i0;; i++) {
            if (per > 1) q = tree_seq(g, i);
            const int u = per > 1 ? heads * tree_units_before(g, q, tree_token_blocks(g, q)) : mine;
            if (u0 < at + u) {
                sh.q = q;
                sh.seq = i;
                sh.off = u0 - at;
                break;
            }
            at += u;
        }
    }
    __syncthreads();
    if (u1 <= u0) return;
    w.left = u1 - u0;
    w.i = sh.seq;
    w.q = sh.q;
    const int nb = tree_token_blocks(g, w.q), each = tree_units_before(g, w.q, nb) * g.chunks;
    w.g = sh.off / each;
    int off = sh.off - w.g * each;
    if (g.a.mask || w.q.bad || nb == 1) {               // blocks of equal length
        const int u = (g.over + tree_units(g, w.q.len)) * g.chunks;
        w.b = off / u;
        off -= w.b * u;
    } else {
        // every thread looks at a few of the blocks
        const int step = (nb + THREADS - 1) / THREADS, k0 = min(nb, (int)threadIdx.x * step), k1 = min(nb, k0 + step);
        int at = tree_units_before(g, w.q, k0) * g.chunks;
        for (int k = k0; k < k1; k++) {
            const int u = (g.over + tree_units(g, w.q.base + min(w.q.T, (k + 1) * g.tb))) * g.chunks;
            if (off >= at && off < at + u) {
                sh.b = k;
                sh.rest = off - at;
            }
            at += u;
        }
        __syncthreads();
        w.b = sh.b;
        off = sh.rest;
    }
    w.chunk = 0;
    tree_item(g, w);
    if (g.chunks > 1) {
        w.chunk = off / (g.over + w.units);
        off -= w.chunk * (g.over + w.units);
        tree_item(g, w);
    }
    w.pos = off;
    w.at = u0 - off;
}

// Where an item's parts are, described by the CTA that holds its first tile:
// for every item, where there are fewer than CTAs, else for a CTA's last item
// when that goes on in the next ones.
struct TreeShare {
    int slot, last;                  // its first part's slot, the CTA of its last tile; -1: nothing to join
    int first;                       // the CTA of its first
    int t0, tok, tokens, heads, head;
};

__device__ __forceinline__ void tree_describe(const TreeArgs &g, const TreeWalk &w, const TreeLine &line, int n, bool first_item) {
    if (w.tile != 0 || (n == w.units && !g.by_item)) return;
    const int at = g.by_item ? (w.i * g.p.n_kv_heads + w.g) * g.item_blocks + w.b * g.chunks + w.chunk : (int)blockIdx.x;
    g.share[at] = {(int)blockIdx.x * 2 + (first_item ? 0 : 1), n == w.units ? -1 : line.owner(w.at + g.over + w.units - 1),
                   (int)blockIdx.x, w.q.t0, w.tok, w.tokens, w.heads, w.head};
}

// Row r of row tile t of a block: its token in the block (-1: no such row)
// and where the row lies in q (ld: its row stride) or out.
__device__ __forceinline__ int tree_token(const TreeArgs &g, int tokens, int heads, int t, int r) {
    const int k = r / heads;
    return k < g.tile_tokens && t * g.tile_tokens + k < tokens ? t * g.tile_tokens + k : -1;
}

__device__ __forceinline__ int64_t tree_row(const TreeArgs &g, int t0, int tok, int heads, int head, int t, int r, int64_t ld) {
    const int k = r / heads;
    return (int64_t)(t0 + tok + t * g.tile_tokens + k) * ld + (int64_t)(head + r - k * heads) * g.p.head_dim;
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
int tree_allow(vb_ctx *ctx, const void *kernel, int bytes);
int tree_prepare(vb_ctx *ctx, TreeArgs &g, int tile_rows, int tiles, int kt, int over);
int launch_tree_combine(vb_ctx *ctx, const TreeArgs &g);

}  // namespace vb
