// vb_tree.cu -- attention of drafted tokens over a paged cache.
//
// For token j of sequence i and query head h of K/V head g:
//   o = sum_r p_r v_r / sum_r p_r,  p_r = exp(scale * q.k_r - max)
// over the rows before the draft and the draft rows that j's mask names.
//
// One warp owns one (token, head): a lane holds head dimensions lane,
// lane + 32, ..., scores are warp sums, and the maximum and sum run along.
#include "vb_common.cuh"
#include "vb_kernels.cuh"
#include "vb_tc.cuh"

namespace vb {

constexpr int TR_WARPS = 8;

struct TreeArgs {
    vb_tree_args a;
    vb_pages p;
    float scale;
    int *err;
};

template <typename T>
__device__ __forceinline__ float to_f(T v) { return (float)v; }

template <typename Q, typename C>
__global__ void __launch_bounds__(TR_WARPS * 32) tree_attention_kernel(const __grid_constant__ TreeArgs g) {
    pdl_trigger();
    pdl_wait();
    constexpr int U = 8;
    const vb_tree_args &a = g.a;
    const vb_pages &p = g.p;
    const int lane = threadIdx.x & 31;
    const int64_t item = (int64_t)blockIdx.x * TR_WARPS + (threadIdx.x >> 5);
    if (item >= (int64_t)a.n * a.max_tokens * a.n_heads) return;
    const int h = (int)(item % a.n_heads), j = (int)(item / a.n_heads % a.max_tokens);
    const int i = (int)(item / a.n_heads / a.max_tokens);
    const int t0 = a.start[i], T = a.start[i + 1] - t0, s = a.seqs[i];
    const int hd = p.head_dim;
    if (t0 < 0 || T < 0 || T > a.max_tokens || t0 > a.n_tokens - T) {
        if (lane == 0) atomicCAS(g.err, 0, VB_DEV_TREE_SEQ);
        return;
    }
    if (j >= T) return;
    const int len = s >= 0 && s < p.n_seqs ? p.length[s] : -1;
    Q *out = static_cast<Q *>(const_cast<void *>(a.out)) + (int64_t)(t0 + j) * a.ldo + (int64_t)h * hd;
    const int base = len - T;
    if (base < 0 || (int64_t)len > (int64_t)p.max_pages * p.page_rows || (a.mask && T > 32 * a.mask_words)) {
        if (lane == 0) atomicCAS(g.err, 0, VB_DEV_TREE_SEQ);
        for (int d = lane; d < hd; d += 32) out[d] = Q(0.0f);
        return;
    }
    const Q *q = static_cast<const Q *>(a.q) + (int64_t)(t0 + j) * a.ldq + (int64_t)h * hd;
    const uint32_t *mask = a.mask ? a.mask + (int64_t)(t0 + j) * a.mask_words : nullptr;
    float qv[U], o[U], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int u = 0; u < U; u++) {
        qv[u] = lane + 32 * u < hd ? to_f(q[lane + 32 * u]) : 0.0f;
        o[u] = 0.0f;
    }
    const int kvh = h / (a.n_heads / p.n_kv_heads);
    const int last = mask ? len : base + j + 1;
    for (int r = 0; r < last; r++) {
        if (mask && r >= base && !(mask[(r - base) >> 5] >> ((r - base) & 31) & 1u)) continue;
        const int page = p.table[(int64_t)s * p.max_pages + r / p.page_rows];
        if (page < 0 || page >= p.n_pages) {
            if (lane == 0) atomicCAS(g.err, 0, VB_DEV_TREE_PAGE);
            continue;
        }
        const int64_t at = ((((int64_t)a.layer * p.n_pages + page) * p.n_kv_heads + kvh) * p.page_rows +
                            r % p.page_rows) * hd;
        const C *k = static_cast<const C *>(p.k) + at, *v = static_cast<const C *>(p.v) + at;
        float sc = 0.0f;
#pragma unroll
        for (int u = 0; u < U; u++)
            if (lane + 32 * u < hd) sc = fmaf(qv[u], to_f(k[lane + 32 * u]), sc);
        sc = warp_sum(sc) * g.scale;
        const float mn = fmaxf(m, sc), ms = mn == -INFINITY ? 0.0f : mn;
        const float al = expf(m - ms), e = expf(sc - ms);
        m = mn;
        l = fmaf(l, al, e);
#pragma unroll
        for (int u = 0; u < U; u++)
            if (lane + 32 * u < hd) o[u] = fmaf(o[u], al, e * to_f(v[lane + 32 * u]));
    }
#pragma unroll
    for (int u = 0; u < U; u++)
        if (lane + 32 * u < hd) out[lane + 32 * u] = Q(l > 0.0f || l != l ? o[u] / l : 0.0f);
}

int check_pages(vb_ctx *ctx, const vb_pages *p, const char *who);

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
    const int64_t qd = (int64_t)a.n_heads * g.p.head_dim;
    if (!a.ldq) a.ldq = qd;
    if (!a.ldo) a.ldo = qd;
    if (a.ldq < qd || a.ldo < qd) return bad("row stride below the row");
    if (!(a.scale >= 0.0f)) return bad("negative scale");
    g.scale = a.scale == 0.0f ? 1.0f / sqrtf((float)g.p.head_dim) : a.scale;
    if (a.mask && a.mask_words <= 0) return bad("mask without words");
    if (a.n == 0 || a.n_tokens == 0 || a.max_tokens == 0) return VB_OK;
    if (!a.q || !a.out || !a.seqs || !a.start) return bad("null pointer");
    const int64_t items = (int64_t)a.n * a.max_tokens * a.n_heads;
    if (items / TR_WARPS >= INT32_MAX) return bad("too many rows");
    g.err = ctx->op_error;
    const dim3 grid((unsigned)((items + TR_WARPS - 1) / TR_WARPS)), block(TR_WARPS * 32);
    cudaError_t e = a.type == VB_TYPE_F32 ? pdl_launch(ctx, tree_attention_kernel<float, __nv_bfloat16>, grid, block, 0, g)
                    : a.type == VB_TYPE_F16 ? pdl_launch(ctx, tree_attention_kernel<__half, __half>, grid, block, 0, g)
                                            : pdl_launch(ctx, tree_attention_kernel<__nv_bfloat16, __nv_bfloat16>, grid, block, 0, g);
    VB_CHECK(ctx, e);
    VB_LAUNCH_CHECK(ctx, "tree_attention");
    return VB_OK;
}
