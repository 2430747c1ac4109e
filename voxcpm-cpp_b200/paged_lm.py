"""A transformer stack over a paged cache that steps drafted tokens.

The blocks are those of vb.LM (RMSNorm, fused q/k/v projection, LongRoPE,
attention, SwiGLU, bf16 rounding after each) put together from the public
calls, with the cache in pages that sequences share:

    pages_extend    room for the step's rows
    qk_norm_rope    each block's q and k turned, k and v into their pages
    tree_attention  each drafted token against the cache and its ancestors
    pages_keep      after verification: the accepted path moves up, the rest
                    of the draft is dropped
    pages_fork      a candidate that shares its parent's pages until it writes
    pages_truncate  a finished sequence gives its pages back

A step's tokens are a prompt or a decode token (a chain), or a tree of drafted
tokens that one call verifies.  Run as a program it drafts over a small random
stack and checks that the tree's results are those of its paths one by one:

    python voxcpm-cpp_b200/paged_lm.py
"""
from __future__ import annotations

import numpy as np

import vcpm_b200 as vb


def tree(parents):
    """(depth of each token, mask words) of a draft: parents[j] is the draft
    place of token j's parent, below j, or -1 for a child of the sequence's
    last row.  Bit r of token j's words: row r is j or one of its ancestors."""
    n = len(parents)
    depth, seen = [], np.zeros((n, n), bool)
    for j, p in enumerate(parents):
        if not -1 <= p < j:
            raise ValueError("a parent comes before its children")
        depth.append(depth[p] + 1 if p >= 0 else 0)
        if p >= 0:
            seen[j] = seen[p]
        seen[j, j] = True
    bits = np.zeros((n, -(-n // 32) * 32), bool)
    bits[:, :n] = seen
    return depth, np.packbits(bits, axis=1, bitorder="little").view("<u4").view(np.int32)


class PagedLM:
    """vb.LM's blocks over a vb.Pages cache.  layers: the host weights that
    vb.LM takes; the context's stream has to be torch's (set_stream(1) for
    the default one)."""

    def __init__(self, ctx, cfg, layers, final_norm=None, *, seqs, pages, page_rows=64, most_rows):
        import torch
        self.ctx, self.cfg, self.torch = ctx, cfg, torch
        self.dev = f"cuda:{ctx.device}"
        H, hd = cfg.hidden, cfg.head_dim
        self.qd, self.kd = cfg.n_heads * hd, cfg.n_kv_heads * hd
        rows = lambda w, n: np.ascontiguousarray(w).reshape(n, -1)  # noqa: E731
        f32 = lambda x: torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(self.dev)  # noqa: E731
        self.layers = []
        for x in layers:
            qkv = np.concatenate([rows(x["q"], self.qd), rows(x["k"], self.kd), rows(x["v"], self.kd)])
            weight = lambda K, N, w: ctx.weight(cfg.wtype, K, N, w)  # noqa: E731
            self.layers.append(dict(qkv=weight(H, self.qd + 2 * self.kd, qkv), o=weight(self.qd, H, x["o"]),
                                    gate=weight(H, cfg.ffn, x["gate"]), up=weight(H, cfg.ffn, x["up"]),
                                    down=weight(cfg.ffn, H, x["down"]), attn_norm=f32(x["attn_norm"]),
                                    ffn_norm=f32(x["ffn_norm"])))
        self.final_norm = None if final_norm is None else f32(final_norm)
        self.scale = cfg.scale_depth / np.sqrt(cfg.n_layers) if cfg.scale_depth > 0 else 1.0
        self.cache = vb.Pages.empty(ctx, cfg.n_layers, pages, cfg.n_kv_heads, page_rows, hd, seqs,
                                    -(-most_rows // page_rows))
        self.rope = None
        if not cfg.no_rope:
            self.rope = torch.from_numpy(vb.rope_table(hd, cfg.rope_theta, hd == 128, most_rows)).to(self.dev)
        ctx.pages_init(self.cache)

    def ints(self, x):
        return self.torch.as_tensor(np.asarray(x, np.int32), device=self.dev)

    def step(self, x, seqs, parents):
        """x float32 [tokens][hidden]: the tokens of seqs[0], then seqs[1], ...;
        parents[i]: the number of tokens of a chain, or the parents of a
        drafted tree (see tree()).  Returns the last block's output, normed."""
        torch, ctx, cfg, p = self.torch, self.ctx, self.cfg, self.cache
        chain = all(isinstance(a, int) for a in parents)
        parents = [list(range(-1, a - 1)) if isinstance(a, int) else list(a) for a in parents]
        counts = [len(a) for a in parents]
        T, H = sum(counts), cfg.hidden
        if tuple(x.shape) != (T, H) or x.dtype != torch.float32:
            raise ValueError(f"x: float32 [{T}][{H}] is wanted")
        trees = [tree(a) for a in parents]
        words = max([m.shape[1] for _, m in trees] + [1])
        mask = None if chain else self.ints(np.concatenate([np.pad(m, ((0, 0), (0, words - m.shape[1]))) for _, m in trees]))
        ids, start = self.ints(seqs), self.ints(np.cumsum([0] + counts))
        of = self.ints(np.repeat(np.arange(len(seqs)), counts)).long()
        before = p.length[ids.long()][of]                     # rows of a token's sequence so far
        place = before + self.ints([j for n in counts for j in range(n)])
        pos = before + self.ints([d for depth, _ in trees for d in depth])
        token_seq = ids[of].contiguous()
        ctx.pages_extend(p, ids, self.ints(counts))

        new = lambda n: torch.empty((T, n), dtype=torch.float32, device=self.dev)  # noqa: E731
        qd, kd, F = self.qd, self.kd, cfg.ffn
        h, n1, qkv, q, att = x.clone(), new(H), new(qd + 2 * kd), new(qd), new(qd)
        a, gate, up, act = new(H), new(F), new(F), new(F)
        for i, L in enumerate(self.layers):
            ctx.rms_norm(h, L["attn_norm"], n1, H, T, cfg.eps, vb.OUT_BF16)
            ctx.matmul(L["qkv"], n1, T, qkv, vb.OUT_BF16)
            ctx.qk_norm_rope(vb.QKArgs(qkv[:, :qd], qkv[:, qd:qd + kd], qkv[:, qd + kd:], heads=cfg.n_heads,
                                       kv_heads=cfg.n_kv_heads, head_dim=cfg.head_dim, q_out=q, rope=self.rope,
                                       pos=None if self.rope is None else pos, flags=vb.OUT_BF16, pages=p, layer=i,
                                       seq=token_seq, row=place))
            ctx.tree_attention(vb.TreeArgs(q, p, i, ids, start, att, heads=cfg.n_heads, max_tokens=max(counts + [1]),
                                           mask=mask))
            ctx.matmul(L["o"], att, T, a, vb.OUT_BF16)
            ctx.residual_add(h, a, self.scale, h, T * H)
            ctx.rms_norm(h, L["ffn_norm"], n1, H, T, cfg.eps, vb.OUT_BF16)
            ctx.matmul(L["gate"], n1, T, gate, vb.OUT_BF16)
            ctx.matmul(L["up"], n1, T, up, vb.OUT_BF16)
            ctx.swiglu(gate, up, act, T * F)
            ctx.matmul(L["down"], act, T, a, vb.OUT_BF16)
            ctx.residual_add(h, a, self.scale, h, T * H)
        if self.final_norm is None:
            return h
        ctx.rms_norm(h, self.final_norm, n1, H, T, cfg.eps, vb.OUT_BF16)
        return n1

    def keep(self, seqs, drafted, paths):
        """Of the last drafted[i] rows of seqs[i] keep the accepted path."""
        most = max([len(a) for a in paths] + [1])
        path = np.zeros((len(paths), most), np.int32)
        for i, a in enumerate(paths):
            path[i, :len(a)] = a
        self.ctx.pages_keep(self.cache, self.ints(seqs), self.ints(drafted), self.ints([len(a) for a in paths]), self.ints(path))

    def fork(self, src, dst):
        self.ctx.pages_fork(self.cache, self.ints(src), self.ints(dst))

    def truncate(self, seqs, length):
        self.ctx.pages_truncate(self.cache, self.ints(seqs), self.ints(length))

    def check(self):
        """Raises if a call since the last check met a full pool or bad numbers."""
        # both are read, and so cleared, first: a step behind a failed page call
        # records errors of its own
        rc, error, request, free = self.ctx.pages_status(self.cache)
        device_rc, code = self.ctx.device_status()
        if rc or device_rc:
            said = ([f"pages: error {error} in request {request}"] if rc else []) + ([f"device error {code}"] if device_rc else [])
            raise vb.VBError(rc or device_rc, "; ".join(said))
        return free

    def close(self):
        for L in self.layers:
            for k in ("qkv", "o", "gate", "up", "down"):
                L[k].release()
        self.layers = []


def main():
    import torch
    rng = np.random.default_rng(0)
    cfg = vb.LMConfig(512, 16, 2, 128, 1024, 4, 1e-5, 10000.0, 0, 0.0, vb.TYPE_F16)
    w = lambda n, k: (rng.standard_normal((n, k)) * 0.02).astype(np.float16)  # noqa: E731
    qd, kd = cfg.n_heads * cfg.head_dim, cfg.n_kv_heads * cfg.head_dim
    layers = [dict(q=w(qd, 512), k=w(kd, 512), v=w(kd, 512), o=w(512, qd), gate=w(1024, 512), up=w(1024, 512),
                   down=w(512, 1024), attn_norm=np.ones(512, np.float32), ffn_norm=np.ones(512, np.float32))
              for _ in range(cfg.n_layers)]
    ctx = vb.Context(0)
    ctx.set_stream(1)
    lm = PagedLM(ctx, cfg, layers, np.ones(512, np.float32), seqs=8, pages=64, page_rows=16, most_rows=512)
    rows = lambda n: torch.from_numpy(rng.standard_normal((n, 512)).astype(np.float32)).cuda().bfloat16().float()  # noqa: E731

    lm.step(rows(120), [0, 1], [70, 50])                      # two prompts
    draft = rows(7)
    parents = [-1, 0, 0, 1, 2, 2, -1]
    paths = [[0, 1, 3], [0, 2, 4], [0, 2, 5], [6]]
    lm.fork([0] * 4, [2, 3, 4, 5])                            # candidates that share sequence 0's pages
    by_tree = lm.step(draft, [0], [parents])
    worst = 0.0
    for s, path in zip((2, 3, 4, 5), paths):
        alone = lm.step(draft[path].contiguous(), [s], [len(path)])
        worst = max(worst, float((by_tree[path] - alone).norm() / alone.norm()))
    lm.keep([0], [7], [[0, 2, 5]])                            # the path that was accepted
    x = rows(1)
    after = torch.cat([lm.step(x, [0], [1]), lm.step(x, [4], [1])])
    again = float((after[0] - after[1]).norm() / after[1].norm())
    lm.truncate([0, 1, 2, 3, 4, 5], [0] * 6)
    free = lm.check()
    print(f"tree against its paths: {worst:.1e}; the token after the kept path: {again:.1e}; free pages {free} of 64")
    lm.close()
    ctx.close()
    return worst, again, free


if __name__ == "__main__":
    main()
