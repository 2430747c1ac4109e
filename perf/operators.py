"""Cases of the paged-cache operators: the head norms and rotation that write the cache (qk), the attention of drafted tokens
that reads it (tree), and the page operations between the two (pages).

`run` computes them in elementary torch operations where `own` is false, and through the framework's entry points where it is
true.  Head counts and widths are those of the framework's stacks (16 query heads on 2 K/V heads of 128, 28 layers, prompts of
200 and 256 tokens, batches of up to 64 utterances) and generic ones beside them."""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5


# ------------------------------------------------------------------ cases
def _qk(name, tokens, seqs, type, past=0, heads=16, kv_heads=2, head_dim=128, rot=128, adjacent=False, page_rows=16):
    return dict(name=name, op="qk", type=type, seqs=seqs, tokens=tokens, past=past, heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, rot=rot, adjacent=adjacent, page_rows=page_rows)


def _tree(name, seqs, drafted, rows, type, ragged=False, chain=False, heads=16, kv_heads=2, head_dim=128, page_rows=16):
    return dict(name=name, op="tree", type=type, seqs=seqs, drafted=drafted, rows=rows, ragged=ragged, chain=chain,
                heads=heads, kv_heads=kv_heads, head_dim=head_dim, page_rows=page_rows)


def _pages(name, kind, seqs, rows, drafted=0, children=0, layers=28, kv_heads=2, head_dim=128, page_rows=16):
    return dict(name=name, op="pages", kind=kind, seqs=seqs, rows=rows, drafted=drafted, children=children, layers=layers,
                kv_heads=kv_heads, head_dim=head_dim, page_rows=page_rows)


def listed():
    return [
        # one token of one utterance between its projections and its attention: latency
        _qk("qk_token", 1, 1, "f32", past=383),
        # 16 drafted tokens of each of 64 utterances
        _qk("qk_drafts", 16, 64, "bf16", past=1021),
        # the 200-token prompts of 64 utterances in one call: bandwidth
        _qk("qk_prompts", 200, 64, "f32"),
        # one decode token over a short cache: latency
        _tree("tree_token", 1, 1, 384, "f32"),
        # up to 25 drafted tokens for each of 8 utterances of different lengths
        _tree("tree_drafts", 8, 25, 2000, "bf16", ragged=True),
        # an odd head layout, odd lengths, fp16, pages of 32
        _tree("tree_odd", 5, 13, 3001, "f16", ragged=True, heads=12, kv_heads=4, head_dim=96, page_rows=32),
        # one drafted tree at the end of a very long cache
        _tree("tree_long", 1, 48, 131072, "bf16", page_rows=64),
        # one decode token for each of 64 long sequences: the cache is read at memory speed
        _tree("tree_decode64", 64, 1, 8192, "f32", page_rows=64),
        # a whole prompt, each token seeing those before it: matrix products
        _tree("tree_prompt", 1, 4096, 4096, "bf16", chain=True),
        # four candidates forked off one utterance, each about to write eight rows
        _pages("pages_fork", "fork", 1, 1003, drafted=8, children=4),
        # a step's end for 64 utterances: 16 drafted rows, the accepted path of each is kept
        _pages("pages_keep", "keep", 64, 700, drafted=16),
        # a half-empty pool moves into a smaller one
        _pages("pages_compact", "compact", 64, 1000, layers=28, page_rows=64),
    ]


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6e12, w["flops"] / 1e15)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["qk", "tree", "tree", "pages"])
    heads, kv_heads = rng.choice([(16, 2), (16, 2), (32, 8), (8, 8), (12, 4)])
    head_dim, page_rows = rng.choice([64, 96, 128, 128, 256]), rng.choice([16, 32, 64, 128])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    if op == "qk":
        rot, seqs = rng.choice([head_dim, head_dim, head_dim // 2]), _log(rng, 1, 64)
        case = _qk("", _log(rng, 1, 256), seqs, rng.choice(list(TYPES)), rng.randrange(4096), heads, kv_heads, head_dim, rot,
                   rng.random() < 0.3, page_rows)
        shrink = "tokens"
    elif op == "tree":
        chain, seqs = rng.random() < 0.4, _log(rng, 1, 64)
        drafted = _log(rng, 1, 2048 if chain else 64)
        rows = drafted if chain and rng.random() < 0.5 else max(drafted, _log(rng, 1, 131072))
        case = _tree("", seqs, drafted, rows, rng.choice(list(TYPES)), rng.random() < 0.5, chain, heads, kv_heads, head_dim, page_rows)
        # the plain form holds whole score matrices
        while case["seqs"] * case["drafted"] * heads * case["rows"] > 5e8:
            case["seqs" if case["seqs"] > 1 else "rows"] = max(1, case["seqs" if case["seqs"] > 1 else "rows"] // 2)
        case["drafted"] = min(case["drafted"], case["rows"])
        shrink = "rows"
    else:
        kind = rng.choice(["fork", "keep", "compact"])
        case = _pages("", kind, _log(rng, 1, 8 if kind == "fork" else 64), _log(rng, 1, 4096), _log(rng, 1, 64), _log(rng, 1, 16),
                      rng.choice([1, 8, 28]), kv_heads, head_dim, page_rows)
        if kind != "fork":
            case["children"] = 0
        if kind == "compact":
            case["drafted"] = 0
        shrink = "rows"
    while _cost(case) > most and case[shrink] > 1:
        case[shrink] = max(1, case[shrink] // 2)
    if op == "tree":
        case["drafted"] = min(case["drafted"], case["rows"])
    del case["name"]
    return case


# ------------------------------------------------- sizes that follow from a case
def _lengths(case):
    """(rows held, drafted tokens) of each sequence: the case's own, or spread below them where it is ragged."""
    n, t, rows = case["seqs"], case["drafted"], case["rows"]
    if not case.get("ragged"):
        return [rows] * n, [t] * n
    drafted = [t if i == 0 else 1 + (t - 1) * ((i * 5) % n) // n for i in range(n)]
    return [max(d, rows - (rows * 3 // 4) * ((i * 3) % n) // n) for i, d in enumerate(drafted)], drafted


def _up(a, b):
    return -(-a // b)


def _path_lengths(case):
    return [1 + (i * 7) % min(6, case["drafted"]) for i in range(case["seqs"])]


def work(case):
    hd, kv = case["head_dim"], case["kv_heads"]
    if case["op"] == "qk":
        t, h, size = case["tokens"] * case["seqs"], case["heads"], TYPES[case["type"]].itemsize
        table = 4 * case["rot"] * case["tokens"]
        return {"bytes": t * (2 * h + 2 * kv) * hd * size + t * 2 * kv * hd * 2 + table + 12 * t, "flops": t * (h + kv) * hd * 8}
    if case["op"] == "tree":
        lens, drafted = _lengths(case)
        h, size = case["heads"], TYPES[case["type"]].itemsize
        seen = sum((r - t) * t + t * (t + 1) // 2 for r, t in zip(lens, drafted))
        return {"bytes": sum(lens) * 2 * kv * hd * 2 + 2 * sum(drafted) * h * hd * size, "flops": 4 * seen * h * hd}
    row = case["layers"] * 2 * kv * hd * 2          # one position over all layers
    n, p = case["seqs"], case["page_rows"]
    pages = _up(case["rows"], p)
    if case["kind"] == "fork":
        c = n * case["children"]
        return {"bytes": 2 * c * (case["rows"] % p) * row + c * pages * 16, "flops": 0}
    if case["kind"] == "keep":
        return {"bytes": 2 * sum(k - 1 for k in _path_lengths(case)) * row + n * 64, "flops": 0}
    return {"bytes": 2 * n * pages * p * row + n * pages * 24, "flops": 0}


# ----------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cache(g, lens, room, n_seqs, spare, layers, kv, page_rows, hd, dtype):
    """A paged cache whose sequences hold `lens` rows in pages scattered over the pool; `room`: most rows of a sequence."""
    held = [_up(x, page_rows) for x in lens]
    most, total = max(1, _up(room, page_rows)), sum(held)
    n_pages = total + spare
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((n_seqs, most), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    cols = torch.arange(most, device="cuda")
    count = torch.tensor(held + [0] * (n_seqs - len(held)), device="cuda")
    table[cols < count[:, None]] = order[:total]
    refs[order[:total].long()] = 1
    shape = (layers, n_pages, kv, page_rows, hd)
    return dict(k=torch.randn(shape, generator=g, device="cuda", dtype=dtype), v=torch.randn(shape, generator=g, device="cuda", dtype=dtype),
                table=table, length=_ints(list(lens) + [0] * (n_seqs - len(lens))), refs=refs,
                status=torch.zeros(4, dtype=torch.int32, device="cuda"))


def _rope(rows, rot):
    """(cos, sin) pairs of positions 0..rows-1."""
    angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
        -2.0 * torch.arange(rot // 2, device="cuda", dtype=torch.float64) / rot)
    return torch.stack((angle.cos(), angle.sin()), -1).flatten(1).float()


def _tree_bits(drafted, words, seed):
    """Bit r of token j: row r of the draft is j itself or one of its ancestors."""
    state, rows = seed * 2654435761 + 12345, []
    for t in drafted:
        bits = []
        for j in range(t):
            state = (state * 6364136223846793005 + 1442695040888963407) % (1 << 64)
            up = j - 1 - (state >> 33) % min(j + 1, 4)          # -1: a child of the sequence's last row
            bits.append((1 << j) | (bits[up] if up >= 0 else 0))
        rows += bits
    flat = [(b >> (32 * w)) & 0xFFFFFFFF for b in rows for w in range(words)]
    return _ints([x - (1 << 32) if x >> 31 else x for x in flat]).reshape(len(rows), words)


def prepare(case, seed):
    g = _gen(seed)
    hd, kv, p = case["head_dim"], case["kv_heads"], case["page_rows"]
    st = {"case": case}
    if case["op"] == "qk":
        n, t, h, dtype = case["seqs"], case["tokens"], case["heads"], TYPES[case["type"]]
        rows, total = case["past"] + t, n * t
        pool = torch.bfloat16 if dtype == torch.float32 else dtype
        st["cache"] = _cache(g, [rows] * n, rows, n, 3, 2, kv, p, hd, pool)
        st["qkv"] = torch.randn(total, (h + 2 * kv) * hd, generator=g, device="cuda", dtype=dtype) * 3   # rows of a fused projection
        st["qw"], st["kw"] = (1 + 0.2 * torch.randn(hd, generator=g, device="cuda") for _ in range(2))
        st["rope"] = _rope(rows, case["rot"])
        st["seq"] = torch.arange(total, device="cuda", dtype=torch.int32) // t
        st["row"] = torch.arange(total, device="cuda", dtype=torch.int32) % t + case["past"]
        st["out"] = torch.empty(total, h * hd, dtype=dtype, device="cuda")
    elif case["op"] == "tree":
        lens, drafted = _lengths(case)
        n, h, dtype, total = case["seqs"], case["heads"], TYPES[case["type"]], sum(drafted)
        pool = torch.bfloat16 if dtype == torch.float32 else dtype
        st["cache"] = _cache(g, lens, max(lens), n, 3, 2, kv, p, hd, pool)
        st["q"] = torch.randn(total, h * hd, generator=g, device="cuda", dtype=dtype)
        starts = [0]
        for d in drafted:
            starts.append(starts[-1] + d)
        st["start"], st["most"], st["longest"] = _ints(starts), max(drafted), max(lens)
        st["seqs"] = torch.arange(n, device="cuda", dtype=torch.int32)
        st["mask"] = None if case["chain"] else _tree_bits(drafted, _up(max(drafted), 32), seed)
        st["out"] = torch.empty(total, h * hd, dtype=dtype, device="cuda")
    else:
        n, rows, t, layers, kids = case["seqs"], case["rows"], case["drafted"], case["layers"], case["children"]
        pages = _up(rows, p)
        if case["kind"] == "fork":
            spare = n * kids * (_up(t, p) + 2)
            st["cache"] = _cache(g, [rows] * n, rows + t, n * (1 + kids), spare, layers, kv, p, hd, torch.bfloat16)
            st["src"] = torch.arange(n * kids, device="cuda", dtype=torch.int32) // kids
            st["dst"] = torch.arange(n * kids, device="cuda", dtype=torch.int32) + n
            st["more"] = _ints([t] * (n * kids))
        elif case["kind"] == "keep":
            st["cache"] = _cache(g, [rows] * n, rows + t, n, n * (_up(t, p) + 1), layers, kv, p, hd, torch.bfloat16)
            st["seqs"] = torch.arange(n, device="cuda", dtype=torch.int32)
            st["more"], st["kept"] = _ints([t] * n), _ints(_path_lengths(case))
            most = max(_path_lengths(case))
            # the path of each sequence: rising row numbers of its draft
            pick = torch.rand(n, t, generator=g, device="cuda").argsort(1)[:, :most]
            inside = torch.arange(most, device="cuda") < st["kept"][:, None]
            st["path"] = torch.where(inside, pick, t).sort(1).values.to(torch.int32).contiguous()
            st["before"] = _ints([rows] * n)
        else:
            st["cache"] = _cache(g, [rows] * n, rows, n, n * pages, layers, kv, p, hd, torch.bfloat16)
            st["into"] = _cache(g, [], rows, n, n * pages + 1, layers, kv, p, hd, torch.bfloat16)
    return st


# ------------------------------------------------------------ plain forms
def _plain_qk(st):
    c, case = st["cache"], st["case"]
    hd, h, kv, rot = case["head_dim"], case["heads"], case["kv_heads"], case["rot"]
    x = st["qkv"].float().unflatten(1, (h + 2 * kv, hd))
    weight = torch.cat((st["qw"].expand(h, hd), st["kw"].expand(kv, hd)))
    y = x[:, :h + kv]
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * weight
    cs = st["rope"][st["row"].long()][:, None]
    cos, sin, turn = cs[..., 0::2], cs[..., 1::2], y[..., :rot]
    a, b = (turn[..., 0::2], turn[..., 1::2]) if case["adjacent"] else (turn[..., :rot // 2], turn[..., rot // 2:])
    a, b = a * cos - b * sin, a * sin + b * cos
    turn = torch.stack((a, b), -1).flatten(-2) if case["adjacent"] else torch.cat((a, b), -1)
    y = torch.cat((turn, y[..., rot:]), -1)
    st["out"].copy_(y[:, :h].flatten(1))
    p = case["page_rows"]
    page, slot = c["table"][st["seq"].long(), st["row"].long() // p].long(), st["row"].long() % p
    for pool, new in ((c["k"], y[:, h:]), (c["v"], x[:, h + kv:])):
        pool[1].transpose(1, 2)[page, slot] = new.to(pool.dtype)
    return {"q": st["out"], "k": c["k"][1], "v": c["v"][1]}


def _plain_tree(st):
    c, case = st["cache"], st["case"]
    hd, h, kv, p, n = case["head_dim"], case["heads"], case["kv_heads"], case["page_rows"], case["seqs"]
    t, rows, start = st["most"], st["longest"], st["start"].long()
    pages = c["table"][st["seqs"].long(), :_up(rows, p)].long().clamp(min=0)
    k, v = (x[1][pages].permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :rows].float() for x in (c["k"], c["v"]))    # [n][kv][rows][hd]
    token = torch.arange(t, device="cuda")
    count, held = start[1:] - start[:-1], c["length"][st["seqs"].long()].long()
    at = (start[:-1, None] + token).clamp(max=st["q"].shape[0] - 1)
    real = token < count[:, None]
    row = torch.arange(rows, device="cuda")
    drafted = row - (held - count)[:, None]                                          # place in the draft, negative before it
    if st["mask"] is None:
        seen = drafted[:, None] <= token[:, None]
    else:
        word = (drafted // 32).clamp(0, st["mask"].shape[1] - 1)
        bits = st["mask"][at].gather(2, word[:, None].expand(n, t, rows))
        seen = (drafted < 0)[:, None] | ((bits >> (drafted % 32)[:, None]) & 1).bool()
    seen = seen & (row < held[:, None])[:, None]                                      # [n][t][rows]
    q = st["q"][at].float().reshape(n, t, kv, h // kv, hd).permute(0, 2, 3, 1, 4)      # [n][kv][group][t][hd]
    s = (q.flatten(2, 3) @ k.transpose(2, 3)).unflatten(2, (h // kv, t)) * (1.0 / math.sqrt(hd))
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    e = (s - top.masked_fill(top == -math.inf, 0)).exp()
    total = e.sum(-1, keepdim=True)
    o = (e.flatten(2, 3) @ v).unflatten(2, (h // kv, t)) / total.masked_fill(total == 0, 1)
    st["out"].copy_(o.permute(0, 3, 1, 2, 4).flatten(2)[real])
    return {"o": st["out"]}


def _plain_truncate(c, seqs, new, p):
    i = seqs.long()
    cols = torch.arange(c["table"].shape[1], device="cuda")
    before, new = c["length"][i].long(), torch.minimum(new.long(), c["length"][i].long())
    gone = (cols >= ((new + p - 1) // p)[:, None]) & (cols < ((before + p - 1) // p)[:, None])
    rows = c["table"][i]
    c["refs"].index_add_(0, rows[gone].long(), torch.full_like(rows[gone], -1))
    c["table"][i] = rows.masked_fill(gone, -1)
    c["length"][i] = new.to(torch.int32)


def _plain_fork(c, src, dst, p):
    _plain_truncate(c, dst, torch.zeros_like(dst), p)
    rows = c["table"][src.long()]
    named = rows[rows >= 0]
    c["refs"].index_add_(0, named.long(), torch.ones_like(named))
    c["table"][dst.long()] = rows
    c["length"][dst.long()] = c["length"][src.long()]


def _plain_extend(c, seqs, more, p):
    i, more = seqs.long(), more.long()
    held = c["length"][i].long()
    have, want = (held + p - 1) // p, (held + more + p - 1) // p
    last = c["table"][i, (have - 1).clamp(min=0)].long()
    part = (held % p != 0) & (more > 0)
    earlier = ((last[:, None] == last) & part[:, None] & part).tril(-1).sum(1)        # requests before this one that left the page
    own_page = part & (c["refs"][last.clamp(min=0)] - earlier > 1)
    need = want - have + own_page
    first, begin = need.cumsum(0) - need, have - own_page.long()
    free = (c["refs"] == 0).nonzero()[:, 0]
    cols = torch.arange(c["table"].shape[1], device="cuda")
    fill = (cols >= begin[:, None]) & (cols < want[:, None])
    rows = c["table"][i]
    new = free[(first[:, None] + cols - begin[:, None]).clamp(0, free.numel() - 1)].to(torch.int32)
    c["table"][i] = torch.where(fill, new, rows)
    a, b, tail = last[own_page], free[first[own_page]], (held % p)[own_page]
    take = (torch.arange(p, device="cuda") < tail[:, None])[None, :, None, :, None]
    for pool in (c["k"], c["v"]):
        pool[:, b] = torch.where(take, pool[:, a], pool[:, b])
    c["refs"].index_add_(0, a, torch.full_like(a, -1).to(torch.int32))
    c["refs"][new[fill].long()] = 1
    c["length"][i] = (held + more).to(torch.int32)


def _plain_keep(c, seqs, drafted, kept, path, p):
    i = seqs.long()
    base = c["length"][i].long() - drafted.long()
    place = torch.arange(path.shape[1], device="cuda")
    inside = place < kept[:, None]
    who = i[:, None].expand_as(path)[inside]
    src, dst = (base[:, None] + path)[inside], (base[:, None] + place)[inside]
    page = lambda r: c["table"][who, r // p].long()  # noqa: E731
    for pool in (c["k"], c["v"]):
        rows = pool.transpose(2, 3)                                                   # [layers][pages][page rows][kv][hd]
        rows[:, page(dst), dst % p] = rows[:, page(src), src % p]
    _plain_truncate(c, seqs, base + kept, p)


def _plain_compact(c, to):
    live = c["refs"] > 0
    number, n = live.cumsum(0) - 1, int(live.sum())
    to["k"][:, :n], to["v"][:, :n] = c["k"][:, live], c["v"][:, live]
    to["refs"].zero_()
    to["refs"][:n] = c["refs"][live]
    to["table"].copy_(torch.where(c["table"] >= 0, number[c["table"].long().clamp(min=0)].to(torch.int32), -1))
    to["length"].copy_(c["length"])


def _plain_pages(st):
    c, case = st["cache"], st["case"]
    p, kind = case["page_rows"], case["kind"]
    if kind == "fork":
        _plain_fork(c, st["src"], st["dst"], p)
        _plain_extend(c, st["dst"], st["more"], p)
    elif kind == "keep":
        _plain_extend(c, st["seqs"], st["more"], p)
        _plain_keep(c, st["seqs"], st["more"], st["kept"], st["path"], p)
        _plain_truncate(c, st["seqs"], st["before"], p)
    else:
        _plain_compact(c, st["into"])


# ---------------------------------------------------- the framework's calls
_context = None


def _framework():
    """The binding and this process's context, on torch's stream."""
    global _context
    if _context is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "voxcpm-cpp_b200"))
        import vcpm_b200 as vb
        ctx = vb.Context(torch.cuda.current_device())
        ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)     # 1: the legacy default stream
        _context = (vb, ctx)
    return _context


def _bind(st):
    """The argument records that a program builds once for its buffers."""
    vb, ctx = _framework()
    case = st["case"]
    pages = lambda c: vb.Pages(c["k"], c["v"], c["table"], c["length"], c["refs"], c["status"])  # noqa: E731
    st["pages"] = pages(st["cache"])
    if case["op"] == "qk":
        h, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
        q, k, v = st["qkv"].split((h * hd, kv * hd, kv * hd), 1)
        st["args"] = vb.QKArgs(q, k, v, heads=h, kv_heads=kv, head_dim=hd, rope=st["rope"], pos=st["row"], q_out=st["out"],
                               q_weight=st["qw"], k_weight=st["kw"], norm=True, eps=EPS, rot_dim=case["rot"], adjacent=case["adjacent"],
                               pages=st["pages"], layer=1, seq=st["seq"], row=st["row"])
    elif case["op"] == "tree":
        st["args"] = vb.TreeArgs(st["q"], st["pages"], 1, st["seqs"], st["start"], st["out"], heads=case["heads"],
                                 max_tokens=st["most"], mask=st["mask"])
    elif case["kind"] == "compact":
        st["into_pages"] = pages(st["into"])


def _own_pages(ctx, st):
    c, kind = st["pages"], st["case"]["kind"]
    if kind == "fork":
        ctx.pages_fork(c, st["src"], st["dst"])
        ctx.pages_extend(c, st["dst"], st["more"])
    elif kind == "keep":
        ctx.pages_extend(c, st["seqs"], st["more"])
        ctx.pages_keep(c, st["seqs"], st["more"], st["kept"], st["path"])
        ctx.pages_truncate(c, st["seqs"], st["before"])
    else:
        ctx.pages_compact(c, st["into_pages"])


def run(st):
    op = st["case"]["op"]
    if not own:
        if op == "qk":
            return _plain_qk(st)
        if op == "tree":
            return _plain_tree(st)
        _plain_pages(st)
    else:
        ctx = _framework()[1]
        if "pages" not in st:
            _bind(st)
        if op == "qk":
            ctx.qk_norm_rope(st["args"])
            return {"q": st["out"], "k": st["cache"]["k"][1], "v": st["cache"]["v"][1]}
        if op == "tree":
            ctx.tree_attention(st["args"])
            return {"o": st["out"]}
        _own_pages(ctx, st)
    c = st["into"] if st["case"]["kind"] == "compact" else st["cache"]
    # rows only move: their bits are compared
    return {"k": c["k"].view(torch.int16), "v": c["v"].view(torch.int16), "table": c["table"], "length": c["length"], "refs": c["refs"]}


# ------------------------------------------------------- exact, in 64 bits
def _exact_qk(case, st):
    hd, h, kv, rot, p = case["head_dim"], case["heads"], case["kv_heads"], case["rot"], case["page_rows"]
    x = st["qkv"].double().reshape(-1, h + 2 * kv, hd)
    out = torch.empty_like(x)
    pair = torch.arange(rot // 2, device="cuda")
    lo, hi = (2 * pair, 2 * pair + 1) if case["adjacent"] else (pair, pair + rot // 2)
    cs = st["rope"].double()[st["row"].long()]
    for j in range(h + 2 * kv):
        z = x[:, j]
        if j < h + kv:
            z = z / (z.pow(2).sum(1, keepdim=True) / hd + EPS).sqrt() * (st["qw"] if j < h else st["kw"]).double()
            w = z.clone()
            w[:, lo] = z[:, lo] * cs[:, 2 * pair] - z[:, hi] * cs[:, 2 * pair + 1]
            w[:, hi] = z[:, lo] * cs[:, 2 * pair + 1] + z[:, hi] * cs[:, 2 * pair]
            z = w
        out[:, j] = z
    res = {"q": out[:, :h].reshape(x.shape[0], h * hd)}
    page = st["cache"]["table"][st["seq"].long(), torch.div(st["row"], p, rounding_mode="floor").long()].long()
    for name, first in (("k", h), ("v", h + kv)):
        pool = st["cache"][name][1].double()
        for g in range(kv):
            pool[page, g, (st["row"] % p).long()] = out[:, first + g]
        res[name] = pool
    return res


def _exact_tree(case, st):
    hd, h, kv, p = case["head_dim"], case["heads"], case["kv_heads"], case["page_rows"]
    lens, drafted = _lengths(case)
    out, first = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda"), 0
    for i, (rows, t) in enumerate(zip(lens, drafted)):
        pages = st["cache"]["table"][i, :_up(rows, p)].long()
        seen = torch.ones(t, rows, dtype=torch.bool, device="cuda")
        j = torch.arange(t, device="cuda")
        if st["mask"] is None:
            seen[:, rows - t:] = j[:, None] >= j
        else:
            bits = st["mask"][first:first + t]
            seen[:, rows - t:] = (bits[:, j // 32] >> (j % 32)) & 1 == 1
        for a in range(h):
            g = a // (h // kv)
            k = st["cache"]["k"][1, pages, g].reshape(-1, hd)[:rows].double()
            v = st["cache"]["v"][1, pages, g].reshape(-1, hd)[:rows].double()
            q = st["q"][first:first + t, a * hd:(a + 1) * hd].double()
            s = (q @ k.T / math.sqrt(hd)).masked_fill(~seen, -math.inf)
            out[first:first + t, a * hd:(a + 1) * hd] = torch.softmax(s, 1) @ v
        first += t
    return {"o": out}


def exact(case, seed):
    if case["op"] == "pages":
        return None
    st = prepare(case, seed)
    return _exact_qk(case, st) if case["op"] == "qk" else _exact_tree(case, st)
