// vb_qk.cu -- head norms of queries and keys with the position rotation, and
// the store of keys and values into a paged cache, in one pass.
//
// Per token and head: y = x * rsqrt(mean(x^2) + eps) * w, then the pairs
// (a, b) of the first rot_dim values become (a c - b s, a s + b c) with the
// position's (cos, sin).  Everything is held in fp32 and each result rounded
// once, to the output's type.
//
// Mapping: a group of LPH lanes (a power of two) owns head rows of one token.
// A lane holds two pieces of V values whose pairs it rotates itself -- i ..
// with i + rot/2 .. of the first half, or two neighbouring pieces when pairs
// are adjacent -- so the only exchange is the sum of squares over the group.
// V is what 16 bytes hold: 4 fp32 values, 8 of 16 bits (4 where the halves of
// the row do not split into eights).  Longer pieces would leave gaps between
// the lanes of a load.
#include "vb_common.cuh"
#include "vb_kernels.cuh"
#include "vb_tc.cuh"

#include <algorithm>

namespace vb {

constexpr int QK_THREADS = 256;
// Waves of threads that a call is spread over: with 1 | 2 | 8 of them 12,800
// tokens take 45.1 | 45.1 | 47.6 us in fp32 and 38.7 | 34.6 | 40.9 in bf16.
constexpr int QK_WAVES = 2;

struct QKArgs {
    vb_qk_args a;
    vb_pages p;
    int store;              // rows go to the cache
    int vec;                // pointers and strides allow 16-byte accesses
    int vec_w;              // of the weights too
    float inv_dim;          // 1 / head_dim
    int per;                // head rows of a group
    int *err;
};

template <typename T>
struct Elem;
template <>
struct Elem<float> {
    __device__ static float get(float v) { return v; }
    __device__ static float put(float v) { return v; }
};
template <>
struct Elem<__half> {
    __device__ static float get(__half v) { return __half2float(v); }
    __device__ static __half put(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<__nv_bfloat16> {
    __device__ static float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    __device__ static __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};

// V values of a row, as they lie in memory.
template <typename T, int V>
struct Piece {
    T x[V];
};

template <typename T, int V>
__device__ __forceinline__ void load(const T *p, bool vec, Piece<T, V> &v) {
    if (vec) {
        constexpr int N = V * sizeof(T) / 4;          // 32-bit words
        uint32_t w[N];
        if constexpr (N >= 4) {
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const uint4 q = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint32_t *>(p) + i);
                w[i] = q.x, w[i + 1] = q.y, w[i + 2] = q.z, w[i + 3] = q.w;
            }
        } else {
            const uint2 q = *reinterpret_cast<const uint2 *>(p);
            w[0] = q.x, w[1] = q.y;
        }
        memcpy(&v, w, sizeof(v));
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) v.x[i] = p[i];
    }
}

template <typename T, int V>
__device__ __forceinline__ void store(T *p, bool vec, const float (&y)[V]) {
    if (vec) {
        Piece<T, V> v;
#pragma unroll
        for (int i = 0; i < V; i++) v.x[i] = Elem<T>::put(y[i]);
        constexpr int N = V * sizeof(T) / 4;
        uint32_t w[N];
        memcpy(w, &v, sizeof(v));
        if constexpr (N >= 4) {
#pragma unroll
            for (int i = 0; i < N; i += 4)
                *reinterpret_cast<uint4 *>(reinterpret_cast<uint32_t *>(p) + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        } else {
            *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) p[i] = Elem<T>::put(y[i]);
    }
}

// Two fp32 values in a 64-bit register: the arithmetic below runs on pairs,
// which halves its instructions.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b) {
    f32x2 d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ void split(f32x2 d, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(d)); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ f32x2 swapped(f32x2 d) {
    float a, b;
    split(d, a, b);
    return pair(b, a);
}

template <typename T, int V>
__device__ __forceinline__ void widen(const Piece<T, V> &x, f32x2 (&y)[V / 2]) {
#pragma unroll
    for (int i = 0; i < V / 2; i++) y[i] = pair(Elem<T>::get(x.x[2 * i]), Elem<T>::get(x.x[2 * i + 1]));
}

template <typename T, int V>
__device__ __forceinline__ void store2(T *p, bool vec, const f32x2 (&y)[V]) {
    float z[2 * V];
#pragma unroll
    for (int i = 0; i < V; i++) split(y[i], z[2 * i], z[2 * i + 1]);
    store(p, vec, z);
}

// A group takes `per` head rows of one token (q heads, then k, then v), ROWS
// of them at a time with the next ROWS on their way: the token's place, its
// table row and the weights are fetched once for them, and a thread always has
// bytes on their way.  Neighbouring groups take the same rows of neighbouring
// tokens, so a warp's control flow is one.  A CTA of 256 threads needs about 80
// registers a thread with pieces of 4 values and 120 with 8.
//
// Bound by HBM where tokens are many: 12,800 tokens of 16 + 2 heads of 128 take
// 45 to 46 us in fp32 (249 MB, 84 % of the copy rate) and 35 in bf16 (131 MB, 20
// us at that rate), which its instructions bound as well: with pieces of 4
// values, twice as many, it takes 55.  One token is a launch and two trips to
// memory.  With 1 | 2 | 4 rows at a time the two take 52.2 | 45.1 | 53.0 and
// 38.4 | 34.6 | 51.8 us.
constexpr int QK_ROWS = 2;

// ROUND: VB_OUT_BF16.
template <typename T, int V, int LPH, bool ADJACENT, bool ROUND>
__global__ void __launch_bounds__(QK_THREADS, V == 8 ? 2 : 3) qk_norm_rope_kernel(const __grid_constant__ QKArgs g) {
    constexpr int ROWS = QK_ROWS, H = V / 2;
    pdl_trigger();
    pdl_wait();
    const vb_qk_args &a = g.a;
    const int hd = a.head_dim, nq = a.n_heads, nk = a.n_kv_heads;
    const int t = (int)((blockIdx.x * QK_THREADS + threadIdx.x) / LPH), lane = threadIdx.x % LPH;
    const unsigned group = LPH == 32 ? 0xffffffffu : ((1u << LPH) - 1u) << (threadIdx.x % 32 / LPH * LPH);
    if (t >= a.n_tokens) return;                          // whole groups
    const int h_lo = blockIdx.y * g.per, h_hi = min(h_lo + g.per, nq + nk + (g.store ? nk : 0));
    // the lane's two pieces: i0 and i1, rotated with each other or passed on
    const int rot = a.rope ? a.rot_dim : 0, c = V * lane;
    const bool mine = lane < hd / (2 * V);
    int i0, i1;
    bool turn;
    if (ADJACENT) {
        i0 = 2 * c;
        i1 = i0 + V;
        turn = i0 < rot;
    } else {
        turn = c < rot / 2;
        i0 = turn ? c : rot + c - rot / 2;
        i1 = i0 + (turn ? rot / 2 : (hd - rot) / 2);
    }
    // where the token goes, then the rows, then what hangs on the place: two
    // round trips to memory in all
    int pos = a.rope ? a.pos[t] : 0;
    const int seq = g.store ? a.seq[t] : -1, row = g.store ? a.row[t] : 0;
    // an error of a page call that nobody has read: rows may not be where the
    // caller takes them to be, so nothing is stored
    const bool unread = g.store && g.p.status[0] != 0;
    auto fetch = [&](int h, Piece<T, V> (&u)[ROWS], Piece<T, V> (&v)[ROWS]) {
#pragma unroll
        for (int r = 0; r < ROWS; r++, h++) {
            const T *src = h < nq        ? static_cast<const T *>(a.q) + (int64_t)t * a.ldq + h * hd
                           : h < nq + nk ? static_cast<const T *>(a.k) + (int64_t)t * a.ldk + (h - nq) * hd
                                         : static_cast<const T *>(a.v) + (int64_t)t * a.ldv + (h - nq - nk) * hd;
            if (mine && h < h_hi) {
                load(src + i0, g.vec, u[r]);
                load(src + i1, g.vec, v[r]);
            }
        }
    };
    Piece<T, V> x0[ROWS], x1[ROWS];
    fetch(h_lo, x0, x1);
    // an invalid place or position skips the whole token
    const bool off_table = a.rope && (pos < 0 || pos >= a.rope_rows);
    if (off_table) pos = 0;
    int page = 0, held = 0;                               // rows that the sequence holds
    const bool placed = seq >= 0 && seq < g.p.n_seqs && row >= 0 && row / g.p.page_rows < g.p.max_pages;
    if (placed) {
        page = g.p.table[(int64_t)seq * g.p.max_pages + row / g.p.page_rows];
        held = g.p.length[seq];
    }
    // A piece y turns to y * c + z * s: z is the other piece (and s negative for
    // the first) or, where pairs are adjacent, y's own with each pair swapped.
    f32x2 cs_c[ADJACENT ? V : H], cs_s[V], w0[H], w1[H];
    if (turn && mine) {
        Piece<float, 2 * V> cs;
        load(a.rope + (int64_t)pos * rot + (ADJACENT ? i0 : 2 * c), true, cs);
        if constexpr (ADJACENT) {
#pragma unroll
            for (int i = 0; i < V; i++) {
                cs_c[i] = pair(cs.x[2 * i], cs.x[2 * i]);
                cs_s[i] = pair(-cs.x[2 * i + 1], cs.x[2 * i + 1]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < H; i++) {
                cs_c[i] = pair(cs.x[4 * i], cs.x[4 * i + 2]);
                cs_s[i] = pair(-cs.x[4 * i + 1], -cs.x[4 * i + 3]);
                cs_s[H + i] = pair(cs.x[4 * i + 1], cs.x[4 * i + 3]);
            }
        }
    }
    const bool no_row = g.store && seq != -1 && (unread || !placed || row >= held || page < 0 || page >= g.p.n_pages);
    const bool bad = off_table || no_row;
    if (bad && lane == 0) atomicCAS(g.err, 0, off_table ? VB_DEV_QK_POS : VB_DEV_QK_ROW);
    const int64_t pool_head = (int64_t)g.p.page_rows * hd;
    const bool keep = g.store && seq != -1 && !bad;
    const int64_t at = keep ? ((int64_t)a.layer * g.p.n_pages + page) * nk * pool_head + (int64_t)(row % g.p.page_rows) * hd : 0;
    auto weights = [&](const float *w) {                  // (ones where there are none)
        Piece<float, V> u, v;
#pragma unroll
        for (int i = 0; i < V; i++) u.x[i] = v.x[i] = 1.0f;
        if (w && mine) {
            load(w + i0, g.vec_w, u);
            load(w + i1, g.vec_w, v);
        }
        widen(u, w0);
        widen(v, w1);
    };
    if (a.norm) weights(h_lo < nq ? a.q_weight : a.k_weight);
    for (int h = h_lo; h < h_hi; h += ROWS) {
        Piece<T, V> n0[ROWS], n1[ROWS];
        fetch(h + ROWS, n0, n1);
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
            const int hr = h + r;
            if (hr >= h_hi) break;                            // for the whole warp
            const bool is_q = hr < nq, is_v = hr >= nq + nk;
            const int kvh = is_v ? hr - nq - nk : hr - nq;
            if (hr == nq && hr > h_lo && a.norm) weights(a.k_weight);
            f32x2 y0[H] = {}, y1[H] = {};
            if (mine) {
                widen(x0[r], y0);
                widen(x1[r], y1);
            }
            if (!is_v && a.norm) {
                f32x2 sq = 0;
#pragma unroll
                for (int i = 0; i < H; i++) sq = fma2(y0[i], y0[i], fma2(y1[i], y1[i], sq));
                float ss, s2;
                split(sq, ss, s2);
                ss += s2;
#pragma unroll
                for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(group, ss, o);
                const float rs = rsqrtf(ss * g.inv_dim + a.eps);
                const f32x2 rs2 = pair(rs, rs);
#pragma unroll
                for (int i = 0; i < H; i++) {
                    y0[i] = mul2(y0[i], rs2);
                    y1[i] = mul2(y1[i], rs2);
                    y0[i] = mul2(y0[i], w0[i]);
                    y1[i] = mul2(y1[i], w1[i]);
                }
            }
            if (!mine) continue;
            if (turn && !is_v) {
#pragma unroll
                for (int i = 0; i < H; i++) {
                    const f32x2 p0 = y0[i], p1 = y1[i];
                    y0[i] = fma2(p0, cs_c[i], mul2(ADJACENT ? swapped(p0) : p1, cs_s[i]));
                    y1[i] = fma2(p1, cs_c[ADJACENT ? H + i : i], mul2(ADJACENT ? swapped(p1) : p0, cs_s[H + i]));
                }
            }
            auto keep_row = [&]() {
                if (is_q || !keep) return;
                if constexpr (sizeof(T) == 2) {               // of the cache's type
                    uint16_t *pool = static_cast<uint16_t *>(is_v ? g.p.v : g.p.k) + at + kvh * pool_head;
                    store2(reinterpret_cast<T *>(pool) + i0, true, y0);
                    store2(reinterpret_cast<T *>(pool) + i1, true, y1);
                } else if (g.p.type == VB_TYPE_F16) {
                    __half *pool = static_cast<__half *>(is_v ? g.p.v : g.p.k) + at + kvh * pool_head;
                    store2(pool + i0, true, y0);
                    store2(pool + i1, true, y1);
                } else {
                    __nv_bfloat16 *pool = static_cast<__nv_bfloat16 *>(is_v ? g.p.v : g.p.k) + at + kvh * pool_head;
                    store2(pool + i0, true, y0);
                    store2(pool + i1, true, y1);
                }
            };
            if constexpr (ROUND) {
                keep_row();                                   // before: a row of the cache is rounded once, to its type
#pragma unroll
                for (int i = 0; i < H; i++) {
                    float u, v;
                    split(y0[i], u, v);
                    y0[i] = pair(bf16r(u), bf16r(v));
                    split(y1[i], u, v);
                    y1[i] = pair(bf16r(u), bf16r(v));
                }
            }
            if (bad) {
#pragma unroll
                for (int i = 0; i < H; i++) y0[i] = y1[i] = 0;
            }
            T *dst = is_q               ? static_cast<T *>(a.q_out) + (int64_t)t * a.ldq_out + hr * hd
                     : !is_v && a.k_out ? static_cast<T *>(a.k_out) + (int64_t)t * a.ldk_out + kvh * hd
                                        : nullptr;
            if (dst) {
                store2(dst + i0, g.vec, y0);
                store2(dst + i1, g.vec, y1);
            }
            if constexpr (!ROUND) keep_row();
        }
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
            x0[r] = n0[r];
            x1[r] = n1[r];
        }
    }
}

int check_pages(vb_ctx *ctx, const vb_pages *p, const char *who);

template <typename T, int V, bool ADJACENT, bool ROUND = false>
static cudaError_t launch_qk_v(vb_ctx *ctx, QKArgs &g) {
    const int heads = g.a.n_heads + g.a.n_kv_heads * (g.store ? 2 : 1), rows = QK_ROWS;
    int lph = 1;
    while (lph * 2 * V < g.a.head_dim) lph *= 2;
    // as many rows to a group as leave QK_WAVES waves of threads: a token of few
    // is spread over the SMs, one of many shares what it fetches once
    const int64_t room = (int64_t)QK_WAVES * ctx->sm_count * 3 * QK_THREADS / lph;
    int64_t chunks = std::max<int64_t>(1, std::min<int64_t>((heads + rows - 1) / rows, room / std::max(1, g.a.n_tokens)));
    g.per = (int)((heads + chunks - 1) / chunks + rows - 1) / rows * rows;
    const dim3 grid((unsigned)(((int64_t)g.a.n_tokens * lph + QK_THREADS - 1) / QK_THREADS), (unsigned)((heads + g.per - 1) / g.per));
    switch (lph) {
        case 1: return pdl_launch(ctx, qk_norm_rope_kernel<T, V, 1, ADJACENT, ROUND>, grid, dim3(QK_THREADS), 0, g);
        case 2: return pdl_launch(ctx, qk_norm_rope_kernel<T, V, 2, ADJACENT, ROUND>, grid, dim3(QK_THREADS), 0, g);
        case 4: return pdl_launch(ctx, qk_norm_rope_kernel<T, V, 4, ADJACENT, ROUND>, grid, dim3(QK_THREADS), 0, g);
        case 8: return pdl_launch(ctx, qk_norm_rope_kernel<T, V, 8, ADJACENT, ROUND>, grid, dim3(QK_THREADS), 0, g);
        case 16: return pdl_launch(ctx, qk_norm_rope_kernel<T, V, 16, ADJACENT, ROUND>, grid, dim3(QK_THREADS), 0, g);
        default: return pdl_launch(ctx, qk_norm_rope_kernel<T, V, 32, ADJACENT, ROUND>, grid, dim3(QK_THREADS), 0, g);
    }
}

template <typename T>
static cudaError_t launch_qk(vb_ctx *ctx, QKArgs &g) {
    const int rot = g.a.rope ? g.a.rot_dim : 0;
    if constexpr (sizeof(T) == 2)
        if (g.a.head_dim % 16 == 0 && rot % 16 == 0)
            return g.a.adjacent ? launch_qk_v<T, 8, true>(ctx, g) : launch_qk_v<T, 8, false>(ctx, g);
    if constexpr (sizeof(T) == 4)
        if (g.a.flags & VB_OUT_BF16)
            return g.a.adjacent ? launch_qk_v<T, 4, true, true>(ctx, g) : launch_qk_v<T, 4, false, true>(ctx, g);
    return g.a.adjacent ? launch_qk_v<T, 4, true>(ctx, g) : launch_qk_v<T, 4, false>(ctx, g);
}

}  // namespace vb

using namespace vb;

extern "C" int vb_qk_norm_rope(vb_ctx *ctx, const vb_qk_args *in) {
    if (!ctx) return VB_ERR_INVALID_ARG;
    auto bad = [&](const char *why) { return set_error(ctx, VB_ERR_INVALID_ARG, "vb_qk_norm_rope: %s", why); };
    if (!in) return bad("null arguments");
    QKArgs g{};
    g.a = *in;
    vb_qk_args &a = g.a;
    if (a.type != VB_TYPE_F32 && a.type != VB_TYPE_F16 && a.type != VB_TYPE_BF16) return bad("type must be F32, F16 or BF16");
    if (a.n_tokens < 0 || a.n_heads <= 0 || a.n_kv_heads < 0) return bad("bad sizes");
    if (a.head_dim < 8 || a.head_dim > 256 || a.head_dim % 8) return bad("head_dim must be a multiple of 8, at most 256");
    if (a.rot_dim == 0) a.rot_dim = a.head_dim;
    if (a.rot_dim < 0 || a.rot_dim % 8 || a.rot_dim > a.head_dim) return bad("rot_dim must be a multiple of 8, at most head_dim");
    if (a.norm && !(a.eps >= 0.0f)) return bad("negative eps");
    if ((a.flags & ~VB_OUT_BF16) || ((a.flags & VB_OUT_BF16) && a.type != VB_TYPE_F32)) return bad("unknown flags for this type");
    const int64_t qd = (int64_t)a.n_heads * a.head_dim, kd = (int64_t)a.n_kv_heads * a.head_dim;
    if ((double)a.n_tokens * ((double)a.n_heads + 2.0 * a.n_kv_heads) * 32.0 >= 4294967295.0) return bad("too many rows");
    if (!a.ldq) a.ldq = qd;
    if (!a.ldk) a.ldk = kd;
    if (!a.ldv) a.ldv = kd;
    if (!a.ldq_out) a.ldq_out = qd;
    if (!a.ldk_out) a.ldk_out = kd;
    if (a.ldq < qd || a.ldq_out < qd || a.ldk < kd || a.ldv < kd || a.ldk_out < kd) return bad("row stride below the row");
    g.store = a.pages != nullptr;
    if (g.store) {
        int rc = check_pages(ctx, a.pages, "vb_qk_norm_rope");
        if (rc) return rc;
        g.p = *a.pages;
        if (g.p.n_kv_heads != a.n_kv_heads || g.p.head_dim != a.head_dim) return bad("the cache has other heads");
        if (a.layer < 0 || a.layer >= g.p.n_layers) return bad("layer out of range");
        if (a.type != VB_TYPE_F32 && a.type != g.p.type) return bad("the cache has another type");
    }
    if (a.n_tokens == 0) return VB_OK;
    if (!a.q || !a.q_out || (a.n_kv_heads && !a.k) || (a.rope && !a.pos) || (g.store && (!a.v || !a.seq || !a.row)))
        return bad("null pointer");
    const uintptr_t es = a.type == VB_TYPE_F32 ? 4 : 2;
    const uintptr_t all = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.q_out | (uintptr_t)a.k_out |
                          (g.store ? (uintptr_t)a.v : 0);
    if (all % es || ((uintptr_t)a.pos | (uintptr_t)a.q_weight | (uintptr_t)a.k_weight | (uintptr_t)a.seq |
                     (uintptr_t)a.row) % 4 || (uintptr_t)a.rope % 16)
        return bad("misaligned pointer");
    const int64_t lanes = 16 / (int64_t)es;
    g.vec = all % 16 == 0 && (a.ldq | a.ldk | a.ldv | a.ldq_out | a.ldk_out) % lanes == 0;
    g.vec_w = ((uintptr_t)a.q_weight | (uintptr_t)a.k_weight) % 16 == 0;
    g.inv_dim = 1.0f / (float)a.head_dim;
    g.err = ctx->op_error;
    cudaError_t e = a.type == VB_TYPE_F32   ? launch_qk<float>(ctx, g)
                    : a.type == VB_TYPE_F16 ? launch_qk<__half>(ctx, g)
                                            : launch_qk<__nv_bfloat16>(ctx, g);
    VB_CHECK(ctx, e);
    VB_LAUNCH_CHECK(ctx, "qk_norm_rope");
    return VB_OK;
}
