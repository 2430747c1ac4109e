"""Plain statements of the paged-cache operators for the tests: a page pool
kept in Python lists, and the attention and head norms in 64 bits."""
import numpy as np


class PoolModel:
    """The bookkeeping of vb_pages and the rows themselves, one value of
    `data` per (layer, k or v, page, head, row): numpy [L][2][pages][kv][P][hd]."""

    def __init__(self, data, n_seqs, max_pages):
        self.data = data
        self.P, self.n_pages = data.shape[4], data.shape[2]
        self.table = np.full((n_seqs, max_pages), -1, np.int32)
        self.length = np.zeros(n_seqs, np.int32)
        self.refs = np.zeros(self.n_pages, np.int32)

    def held(self, s):
        return -(-int(self.length[s]) // self.P)

    def extend(self, seqs, rows):
        free = [p for p in range(self.n_pages) if self.refs[p] == 0]
        for s, r in zip(seqs, rows):
            n, have = int(self.length[s]), self.held(s)
            if r and n % self.P and self.refs[self.table[s, have - 1]] > 1:
                old, new = self.table[s, have - 1], free.pop(0)
                self.data[:, :, new, :, :n % self.P] = self.data[:, :, old, :, :n % self.P]
                self.refs[old] -= 1
                self.refs[new] = 1
                self.table[s, have - 1] = new
            for c in range(have, -(-(n + r) // self.P)):
                self.table[s, c] = free.pop(0)
                self.refs[self.table[s, c]] = 1
            self.length[s] = n + r

    def truncate(self, seqs, cut):
        for s, n in zip(seqs, cut):
            n = min(int(n), int(self.length[s]))
            for c in range(-(-n // self.P), self.held(s)):
                self.refs[self.table[s, c]] -= 1
                self.table[s, c] = -1
            self.length[s] = n

    def fork(self, src, dst):
        self.truncate(dst, [0] * len(dst))
        for s, d in zip(src, dst):
            self.table[d] = self.table[s]
            self.length[d] = self.length[s]
            for p in self.table[s, :self.held(s)]:
                self.refs[p] += 1

    def keep(self, seqs, drafted, kept, path):
        for i, s in enumerate(seqs):
            base = int(self.length[s]) - drafted[i]
            for j in range(kept[i]):
                a, b = base + path[i][j], base + j
                if a != b:
                    self.data[:, :, self.table[s, b // self.P], :, b % self.P] = \
                        self.data[:, :, self.table[s, a // self.P], :, a % self.P]
            self.truncate([s], [base + kept[i]])


def attention(q, k, v, seen, scale):
    """q [T][hd], k, v [rows][hd], seen bool [T][rows], in 64 bits; a row that
    sees nothing gives zeros, unseen rows never enter."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    out = np.zeros((q.shape[0], v.shape[1]))
    if np.isfinite(k).all() and np.isfinite(v).all():         # nothing to keep out: all tokens at once
        s = np.where(seen, (q @ k.T) * scale, -np.inf)
        some = seen.any(1)
        e = np.exp(s[some] - s[some].max(1, keepdims=True)) if some.any() else s[some]
        out[some] = (e @ v) / e.sum(1, keepdims=True)
        return out
    for t in range(q.shape[0]):
        at = np.nonzero(seen[t])[0]
        if not at.size:
            continue
        s = (k[at] @ q[t]) * scale
        e = np.exp(s - s.max())
        out[t] = (e @ v[at]) / e.sum()
    return out


def tree_mask(parents):
    """bool [T][T]: token j sees itself and its ancestors (parent -1: none)."""
    t = len(parents)
    m = np.zeros((t, t), bool)
    for j, p in enumerate(parents):
        if p >= 0:
            m[j] = m[p]
        m[j, j] = True
    return m


def pack_mask(mask, words):
    """int32 [T][words] of a bool [T][<= 32*words] mask."""
    full = np.zeros((mask.shape[0], 32 * words), np.uint64)
    full[:, :mask.shape[1]] = mask
    return (full.reshape(mask.shape[0], words, 32) << np.arange(32, dtype=np.uint64)).sum(2).astype(np.uint32).view(np.int32)


def qk(x, w, eps, cs, rot, adjacent, norm):
    """Head norm and rotation of x [T][heads][hd] in 64 bits; cs [T][rot]."""
    y = np.asarray(x, np.float64)
    if norm:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps)
        if w is not None:
            y = y * np.asarray(w, np.float64)
    if cs is None:
        return y
    y = y.copy()
    i = np.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if adjacent else (i, i + rot // 2)
    c, s = (np.asarray(cs, np.float64)[:, None, j::2] for j in (0, 1))
    ya, yb = y[..., a], y[..., b]
    y[..., a], y[..., b] = ya * c - yb * s, ya * s + yb * c
    return y
