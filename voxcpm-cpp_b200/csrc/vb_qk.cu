// vb_qk.cu -- head norms of queries and keys with the position rotation, and
// the store of keys and values into a paged cache, in one pass.
//
// Per token and head: y = x * rsqrt(mean(x^2) + eps) * w, then the pairs
// (a, b) of the first rot_dim values become (a c - b s, a s + b c) with the
// position's (cos, sin).  Everything is held in fp32 and each result rounded
// once, to the output's type.
//
// Mapping: a group of LPH lanes (a power of two, at least head_dim / 8) owns
// one head row.  A lane holds two pieces of four values whose pairs it
// rotates itself -- i .. i+3 with i + rot/2 .. of the first half, or two
// neighbouring pieces when pairs are adjacent -- so the only exchange is the
// sum of squares over the group.  Rows of q, k and v are items of one grid.
#include "vb_common.cuh"
#include "vb_kernels.cuh"
#include "vb_tc.cuh"

namespace vb {

constexpr int QK_THREADS = 256;

struct QKArgs {
    vb_qk_args a;
    vb_pages p;
    int store;              // rows go to the cache
    int vec;                // pointers and strides allow 4-value accesses
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

template <typename T>
struct alignas(4 * sizeof(T)) Vec4 {
    T x[4];
};

template <typename T>
__device__ __forceinline__ void load4(const T *p, bool vec, float (&v)[4]) {
    if (vec) {
        const Vec4<T> t = *reinterpret_cast<const Vec4<T> *>(p);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = Elem<T>::get(t.x[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = Elem<T>::get(p[i]);
    }
}

template <typename T>
__device__ __forceinline__ void store4(T *p, bool vec, const float (&v)[4]) {
    if (vec) {
        Vec4<T> t;
#pragma unroll
        for (int i = 0; i < 4; i++) t.x[i] = Elem<T>::put(v[i]);
        *reinterpret_cast<Vec4<T> *>(p) = t;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) p[i] = Elem<T>::put(v[i]);
    }
}

template <typename T, int LPH>
__global__ void __launch_bounds__(QK_THREADS) qk_norm_rope_kernel(const __grid_constant__ QKArgs g) {
    pdl_trigger();
    pdl_wait();
    const vb_qk_args &a = g.a;
    const int hd = a.head_dim, nq = a.n_heads, nk = a.n_kv_heads;
    const int heads = nq + nk + (g.store ? nk : 0);
    const int64_t item = ((int64_t)blockIdx.x * QK_THREADS + threadIdx.x) / LPH;
    const int lane = threadIdx.x % LPH;
    const unsigned group = LPH == 32 ? 0xffffffffu : ((1u << LPH) - 1u) << (threadIdx.x % 32 / LPH * LPH);
    if (item >= (int64_t)a.n_tokens * heads) return;      // whole groups
    const int t = (int)(item / heads), h = (int)(item % heads);
    const bool is_q = h < nq, is_v = h >= nq + nk;
    const int kvh = is_v ? h - nq - nk : h - nq;

    // where the token goes; an invalid place or position skips the whole token
    int pos = 0;
    if (a.rope) {
        pos = a.pos[t];
        if (pos < 0 || pos >= a.rope_rows) {
            if (lane == 0) {
                atomicCAS(g.err, 0, VB_DEV_QK_POS);
            }
            pos = -1;
        }
    }
    int64_t pool_row = -1;
    bool bad = pos < 0;
    if (g.store) {
        const int s = a.seq[t], r = a.row[t];
        if (s != -1) {
            int page = -1;
            if (s >= 0 && s < g.p.n_seqs && r >= 0 && r / g.p.page_rows < g.p.max_pages)
                page = g.p.table[(int64_t)s * g.p.max_pages + r / g.p.page_rows];
            if (page < 0 || page >= g.p.n_pages) {
                if (lane == 0) atomicCAS(g.err, 0, VB_DEV_QK_ROW);
                bad = true;
            } else {
                pool_row = (((int64_t)a.layer * g.p.n_pages + page) * nk) * g.p.page_rows + r % g.p.page_rows;
            }
        }
    }
    if (is_v && (pool_row < 0 || bad)) return;

    const T *src = is_q ? static_cast<const T *>(a.q) + (int64_t)t * a.ldq + (int64_t)h * hd
                        : static_cast<const T *>(is_v ? a.v : a.k) + (int64_t)t * (is_v ? a.ldv : a.ldk) +
                              (int64_t)kvh * hd;
    // the lane's two pieces: i0 and i1, rotated with each other or passed on
    const int rot = a.rope ? a.rot_dim : 0, c4 = 4 * lane;
    const bool mine = lane < hd / 8;
    int i0, i1;
    bool turn;
    if (a.adjacent) {
        i0 = 2 * c4;
        i1 = i0 + 4;
        turn = i0 < rot;
    } else {
        turn = c4 < rot / 2;
        i0 = turn ? c4 : rot + c4 - rot / 2;
        i1 = i0 + (turn ? rot / 2 : (hd - rot) / 2);
    }
    float x0[4] = {}, x1[4] = {};
    if (mine && !bad) {
        load4(src + i0, g.vec, x0);
        load4(src + i1, g.vec, x1);
    }
    if (!is_v) {
        if (a.norm) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) ss = fmaf(x0[i], x0[i], fmaf(x1[i], x1[i], ss));
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(group, ss, o);
            const float rs = rsqrtf(ss / (float)hd + a.eps);
            const float *w = is_q ? a.q_weight : a.k_weight;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x0[i] *= rs;
                x1[i] *= rs;
                if (w && mine) {
                    x0[i] *= w[i0 + i];
                    x1[i] *= w[i1 + i];
                }
            }
        }
        if (turn && mine && !bad) {
            const float *cs = a.rope + (int64_t)pos * rot;
            if (a.adjacent) {
                const float4 u = *reinterpret_cast<const float4 *>(cs + i0);      // pairs i0/2, i0/2 + 1
                const float4 v = *reinterpret_cast<const float4 *>(cs + i0 + 4);
                const float cc[4] = {u.x, u.z, v.x, v.z}, sn[4] = {u.y, u.w, v.y, v.w};
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float p0 = x0[2 * i], q0 = x0[2 * i + 1], p1 = x1[2 * i], q1 = x1[2 * i + 1];
                    x0[2 * i] = p0 * cc[i] - q0 * sn[i];
                    x0[2 * i + 1] = p0 * sn[i] + q0 * cc[i];
                    x1[2 * i] = p1 * cc[2 + i] - q1 * sn[2 + i];
                    x1[2 * i + 1] = p1 * sn[2 + i] + q1 * cc[2 + i];
                }
            } else {
                const float4 u = *reinterpret_cast<const float4 *>(cs + 2 * c4);
                const float4 v = *reinterpret_cast<const float4 *>(cs + 2 * c4 + 4);
                const float cc[4] = {u.x, u.z, v.x, v.z}, sn[4] = {u.y, u.w, v.y, v.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float p0 = x0[i], p1 = x1[i];
                    x0[i] = p0 * cc[i] - p1 * sn[i];
                    x1[i] = p0 * sn[i] + p1 * cc[i];
                }
            }
        }
    }
    if (!mine) return;
    if (sizeof(T) == 4 && (a.flags & VB_OUT_BF16)) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x0[i] = bf16r(x0[i]);
            x1[i] = bf16r(x1[i]);
        }
    }
    if (bad) {
#pragma unroll
        for (int i = 0; i < 4; i++) x0[i] = x1[i] = 0.0f;
    }
    T *dst = is_q ? static_cast<T *>(a.q_out) + (int64_t)t * a.ldq_out + (int64_t)h * hd
             : !is_v && a.k_out ? static_cast<T *>(a.k_out) + (int64_t)t * a.ldk_out + (int64_t)kvh * hd
                                : nullptr;
    if (dst) {
        store4(dst + i0, g.vec, x0);
        store4(dst + i1, g.vec, x1);
    }
    if (is_q || pool_row < 0 || bad) return;
    const int64_t at = (pool_row + (int64_t)kvh * g.p.page_rows) * hd;
    if (g.p.type == VB_TYPE_F16) {
        __half *pool = static_cast<__half *>(is_v ? g.p.v : g.p.k) + at;
        store4(pool + i0, true, x0);
        store4(pool + i1, true, x1);
    } else {
        __nv_bfloat16 *pool = static_cast<__nv_bfloat16 *>(is_v ? g.p.v : g.p.k) + at;
        store4(pool + i0, true, x0);
        store4(pool + i1, true, x1);
    }
}

int check_pages(vb_ctx *ctx, const vb_pages *p, const char *who);

template <typename T>
static cudaError_t launch_qk(vb_ctx *ctx, const QKArgs &g) {
    const int hd = g.a.head_dim;
    const int64_t items = (int64_t)g.a.n_tokens * (g.a.n_heads + g.a.n_kv_heads * (g.store ? 2 : 1));
    const int lph = hd <= 32 ? 4 : hd <= 64 ? 8 : hd <= 128 ? 16 : 32;
    const unsigned grid = (unsigned)((items * lph + QK_THREADS - 1) / QK_THREADS);
    switch (lph) {
        case 4: return pdl_launch(ctx, qk_norm_rope_kernel<T, 4>, dim3(grid), dim3(QK_THREADS), 0, g);
        case 8: return pdl_launch(ctx, qk_norm_rope_kernel<T, 8>, dim3(grid), dim3(QK_THREADS), 0, g);
        case 16: return pdl_launch(ctx, qk_norm_rope_kernel<T, 16>, dim3(grid), dim3(QK_THREADS), 0, g);
        default: return pdl_launch(ctx, qk_norm_rope_kernel<T, 32>, dim3(grid), dim3(QK_THREADS), 0, g);
    }
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
    if ((int64_t)a.n_tokens * (a.n_heads + 2 * (int64_t)a.n_kv_heads) * 32 / QK_THREADS >= INT32_MAX) return bad("too many rows");
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
    g.vec = all % (4 * es) == 0 && (a.ldq | a.ldk | a.ldv | a.ldq_out | a.ldk_out) % 4 == 0;
    g.err = ctx->op_error;
    cudaError_t e = a.type == VB_TYPE_F32   ? launch_qk<float>(ctx, g)
                    : a.type == VB_TYPE_F16 ? launch_qk<__half>(ctx, g)
                                            : launch_qk<__nv_bfloat16>(ctx, g);
    VB_CHECK(ctx, e);
    VB_LAUNCH_CHECK(ctx, "qk_norm_rope");
    return VB_OK;
}
