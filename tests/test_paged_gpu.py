"""GPU tests of the paged-cache operators through the C ABI: the page calls
against a pool kept in Python, the head norms and the drafted-token attention
against their formulas in 64 bits, and every refusal.

Tolerances.  Page calls move bits: equal.  Head norms and rotation: fp32
arithmetic on a few values, 2^-20 relative to the row's largest value, plus
half a unit of the output's type (2^-12 fp16, 2^-9 bf16).  Attention: with
S = scale * max sum|q_i k_i|, a score is off by at most 2^-16 S (operands of
the fp32 form are held to 2^-17 or better; fp32 sums add less), a
weight by twice that relatively; weights of the 16-bit forms are rounded to
the cache's type (2^-8 bf16, 2^-11 fp16 bounds both the rounding and the
output's), those of the fp32 form held to 2^-16: absolute error below
max|v| * (4 * 2^-16 S + r), r = 2^-14, 2^-7, 2^-10."""
import numpy as np
import pytest

import paged_model as M

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import vcpm_b200 as vb  # noqa: E402

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    c = vb.Context(0)
    c.set_stream(1)          # torch's default stream
    yield c
    c.close()


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def new_cache(ctx, layers=2, pages=40, kv=2, P=16, hd=64, seqs=6, most=10, dtype=torch.bfloat16, seed=0):
    c = vb.Pages.empty(ctx, layers, pages, kv, P, hd, seqs, most, dtype)
    g = torch.Generator(device="cuda").manual_seed(seed)
    c.k.normal_(generator=g)
    c.v.normal_(generator=g)
    return c


def rows_of(c):
    """numpy int16 [L][2][pages][kv][P][hd]."""
    return torch.stack((c.k, c.v), 1).view(torch.int16).cpu().numpy()


def assert_state(c, m):
    torch.cuda.synchronize()
    assert np.array_equal(c.table.cpu().numpy(), m.table)
    assert np.array_equal(c.length.cpu().numpy(), m.length)
    assert np.array_equal(c.refs.cpu().numpy(), m.refs)
    assert np.array_equal(rows_of(c), m.data)


# ------------------------------------------------------------------ page calls
@pytest.mark.parametrize("seed,layers,kv,P,hd", [(0, 2, 2, 16, 64), (1, 1, 1, 16, 8), (2, 3, 4, 32, 96), (3, 1, 2, 64, 256)])
def test_page_calls_match_a_pool_in_python(ctx, seed, layers, kv, P, hd):
    rng = np.random.default_rng(seed)
    n_seqs, most, pages = 6, 6, 24
    c = new_cache(ctx, layers, pages, kv, P, hd, n_seqs, most, seed=seed)
    m = M.PoolModel(rows_of(c), n_seqs, most)
    done = set()
    for _ in range(80):
        op = rng.choice(["extend", "extend", "fork", "keep", "truncate"])
        seqs = rng.permutation(n_seqs)[:rng.integers(1, 4)]
        if op == "extend":
            rows = [int(rng.choice([0, 1, 3, P, 2 * P - 1])) for _ in seqs]
            if any(m.length[s] + r > most * P for s, r in zip(seqs, rows)):
                continue
            need = sum(-(-(int(m.length[s]) + r) // P) - m.held(s) + 1 for s, r in zip(seqs, rows))
            if need > (m.refs == 0).sum():
                continue
            ctx.pages_extend(c, ints(seqs), ints(rows))
            m.extend(seqs, rows)
        elif op == "fork":
            src = [int(rng.choice([s for s in range(n_seqs) if s not in seqs])) for _ in seqs]
            ctx.pages_fork(c, ints(src), ints(seqs))
            m.fork(src, seqs)
        elif op == "truncate":
            cut = [int(rng.integers(0, most * P + 1)) for _ in seqs]
            ctx.pages_truncate(c, ints(seqs), ints(cut))
            m.truncate(seqs, cut)
        else:
            drafted = [int(rng.integers(0, min(20, m.length[s]) + 1)) for s in seqs]
            kept = [int(rng.integers(0, min(d, 12) + 1)) for d in drafted]
            path = np.full((len(seqs), 12), -7, np.int32)
            ok = True
            for i, s in enumerate(seqs):
                path[i, :kept[i]] = np.sort(rng.permutation(drafted[i])[:kept[i]])
                base = int(m.length[s]) - drafted[i]
                ok &= all(m.refs[m.table[s, (base + j) // P]] == 1 for j in range(kept[i]) if path[i, j] != j)
            if not ok:
                continue
            ctx.pages_keep(c, ints(seqs), ints(drafted), ints(kept), ints(path))
            m.keep(seqs, drafted, kept, path)
        done.add(op)
        assert_state(c, m)
    assert ctx.pages_status(c) == (0, 0, 0, int((m.refs == 0).sum()))
    assert done == {"extend", "fork", "keep", "truncate"}


def test_last_holder_of_a_shared_page_keeps_it(ctx):
    c = new_cache(ctx)
    m = M.PoolModel(rows_of(c), 6, 10)
    for f, a in (("extend", ([0], [21])), ("fork", ([0, 0, 0], [1, 2, 3])), ("truncate", ([0], [0])),
                 ("extend", ([3, 1, 2], [1, 1, 20]))):
        getattr(ctx, "pages_" + f)(c, *(ints(x) for x in a))
        getattr(m, f)(*a)
        assert_state(c, m)
    assert m.refs[m.table[2, 1]] == 1 and m.table[2, 1] == 1      # the third request kept page 1


def test_many_requests_and_a_large_pool(ctx):
    """More requests than threads of the plan, free pages beyond its first scan step."""
    n, P = 1500, 16
    c = new_cache(ctx, 1, 20000, 1, P, 8, n, 8)
    m = M.PoolModel(rows_of(c), n, 8)
    order = np.random.default_rng(3).permutation(n)
    for seqs, rows in ((order, (order * 7) % 100), (order[::-1][:1100].copy(), np.full(1100, 17))):
        ctx.pages_extend(c, ints(seqs), ints(rows))
        m.extend(seqs, rows)
    ctx.pages_truncate(c, ints(order[:700]), ints(np.zeros(700)))
    m.truncate(order[:700], np.zeros(700, int))
    ctx.pages_fork(c, ints(order[700:1400]), ints(order[:700]))
    m.fork(order[700:1400], order[:700])
    ctx.pages_extend(c, ints(order), ints(np.full(n, 5)))
    m.extend(order, np.full(n, 5))
    assert_state(c, m)


@pytest.mark.parametrize("pages", [7, 40, 64])
def test_compact(ctx, pages):
    c = new_cache(ctx)
    m = M.PoolModel(rows_of(c), 6, 10)
    for f, a in (("extend", ([0, 1, 2], [37, 16, 90])), ("fork", ([0, 0], [3, 4])), ("truncate", ([2, 1], [0, 3])),
                 ("extend", ([3], [20]))):
        getattr(ctx, "pages_" + f)(c, *(ints(x) for x in a))
        getattr(m, f)(*a)
    to = new_cache(ctx, pages=pages, most=12, seed=9)
    before = rows_of(to)
    to.table.fill_(5)
    to.refs.fill_(3)
    ctx.pages_compact(c, to)
    live = np.nonzero(m.refs)[0]
    number = np.full(m.n_pages + 1, -1)
    number[live] = np.arange(live.size)
    assert_state(c, m)                                            # unchanged
    want = before.copy()
    want[:, :, :live.size] = m.data[:, :, live]
    assert np.array_equal(rows_of(to), want)
    table = np.full((6, 12), -1)
    table[:, :10] = number[m.table]
    assert np.array_equal(to.table.cpu().numpy(), table)
    assert np.array_equal(to.length.cpu().numpy(), m.length)
    assert np.array_equal(to.refs.cpu().numpy(), np.pad(m.refs[live], (0, pages - live.size)))


def start_state(ctx):
    """Sequence 0 holds 40 rows, 1 is its fork, 2 holds 5."""
    c = new_cache(ctx, pages=8, most=4)
    m = M.PoolModel(rows_of(c), 6, 4)
    for f, a in (("extend", ([0, 2], [40, 5])), ("fork", ([0], [1]))):
        getattr(ctx, "pages_" + f)(c, *(ints(x) for x in a))
        getattr(m, f)(*a)
    return c, m


@pytest.mark.parametrize("call,args,error,request_", [
    ("extend", ([0, 6], [1, 1]), vb.PAGES_SEQ, 1),
    ("extend", ([0, -1], [1, 1]), vb.PAGES_SEQ, 1),
    ("extend", ([0, 2, 0], [1, 1, 1]), vb.PAGES_SEQ, 2),
    ("extend", ([0, 2], [1, -1]), vb.PAGES_COUNT, 1),
    ("extend", ([0, 2], [1, 60]), vb.PAGES_LONG, 1),
    ("extend", ([0, 3], [1, 2 ** 31 - 1]), vb.PAGES_LONG, 1),
    ("extend", ([2, 3, 4], [40, 33, 1]), vb.PAGES_FULL, 1),
    ("fork", ([0, 2], [3, 3]), vb.PAGES_SEQ, 1),
    ("fork", ([0, 1], [1, 3]), vb.PAGES_SEQ, 1),
    ("fork", ([9], [3]), vb.PAGES_SEQ, 0),
    ("truncate", ([0, 6], [1, 1]), vb.PAGES_SEQ, 1),
    ("truncate", ([0, 2], [1, -3]), vb.PAGES_COUNT, 1),
    ("keep", ([2, 7], [1, 1], [1, 1], [[0], [0]]), vb.PAGES_SEQ, 1),
    ("keep", ([2], [6], [1], [[0]]), vb.PAGES_COUNT, 0),
    ("keep", ([2], [3], [2], [[0]]), vb.PAGES_COUNT, 0),
    ("keep", ([2], [1], [2], [[0, 1]]), vb.PAGES_COUNT, 0),
    ("keep", ([2], [4], [3], [[1, 1, 2]]), vb.PAGES_PATH, 0),
    ("keep", ([2], [4], [1], [[4]]), vb.PAGES_PATH, 0),
    ("keep", ([2, 1], [4, 4], [1, 1], [[1], [1]]), vb.PAGES_SHARED, 1),
])
def test_errors_change_nothing_and_stay_until_read(ctx, call, args, error, request_):
    c, m = start_state(ctx)
    getattr(ctx, "pages_" + call)(c, *(ints(x) for x in args))
    assert_state(c, m)
    ctx.pages_extend(c, ints([2]), ints([1]))                     # held back by the error
    assert_state(c, m)
    rc, got, req, free = ctx.pages_status(c)
    assert (rc, got, req, free) == (vb.VB_ERR_BACKEND, error, request_, int((m.refs == 0).sum()))
    assert "paged cache" in ctx.last_error()
    assert ctx.pages_status(c)[:2] == (0, 0)
    ctx.pages_extend(c, ints([2]), ints([1]))
    m.extend([2], [1])
    assert_state(c, m)


def test_compact_into_a_pool_too_small(ctx):
    c, m = start_state(ctx)
    to = new_cache(ctx, pages=3, most=4)
    kept = (rows_of(to), to.refs.clone())
    ctx.pages_compact(c, to)
    assert ctx.pages_status(c)[:2] == (vb.VB_ERR_BACKEND, vb.PAGES_FULL)
    assert np.array_equal(rows_of(to), kept[0]) and torch.equal(to.refs, kept[1])
    assert_state(c, m)


def test_a_broken_table_is_reported(ctx):
    c, m = start_state(ctx)
    c.table[2, 0] = 1000
    ctx.pages_extend(c, ints([2]), ints([1]))
    assert ctx.pages_status(c)[:2] == (vb.VB_ERR_BACKEND, vb.PAGES_TABLE)


def test_empty_calls(ctx):
    c, m = start_state(ctx)
    none = ints([])
    ctx.pages_extend(c, none, none)
    ctx.pages_fork(c, none, none)
    ctx.pages_truncate(c, none, none)
    ctx.pages_keep(c, none, none, none, ints(np.zeros((0, 3))))
    ctx.pages_keep(c, ints([2]), ints([0]), ints([0]), ints(np.zeros((1, 0))))
    assert_state(c, m)
    ctx.pages_init(c)
    torch.cuda.synchronize()
    assert not c.length.any() and not c.refs.any() and bool((c.table == -1).all())


def test_steps_replay_from_a_graph(ctx):
    """extend, keep and truncate captured once run again on the device's own state."""
    c = new_cache(ctx)
    m = M.PoolModel(rows_of(c), 6, 10)
    ctx.pages_extend(c, ints([0, 1]), ints([10, 30]))
    m.extend([0, 1], [10, 30])
    seqs, t, kept, path = ints([0, 1]), ints([5, 5]), ints([2, 3]), ints([[0, 3, 0], [1, 2, 4]])

    def step():
        ctx.pages_extend(c, seqs, t)
        ctx.pages_keep(c, seqs, t, kept, path)

    own = torch.cuda.Stream()
    step()
    m.extend([0, 1], [5, 5])
    m.keep([0, 1], [5, 5], [2, 3], path.cpu().numpy())
    torch.cuda.synchronize()
    ctx.set_stream(own.cuda_stream)
    ctx.graph_begin()
    step()
    g = ctx.graph_end()
    for _ in range(4):
        ctx.graph_launch(g)
        m.extend([0, 1], [5, 5])
        m.keep([0, 1], [5, 5], [2, 3], path.cpu().numpy())
    ctx.sync()
    ctx.graph_destroy(g)
    ctx.set_stream(1)
    assert_state(c, m)


@pytest.mark.parametrize("change", [dict(page_rows=8), dict(page_rows=48), dict(page_rows=2048), dict(head_dim=12),
                                    dict(head_dim=264), dict(type=vb.TYPE_F32), dict(n_seqs=20000), dict(n_pages=0),
                                    dict(k=0), dict(table=0), dict(n_pages=2 ** 30), dict(refs=4)])
def test_cache_views_that_are_refused(ctx, change):
    c = new_cache(ctx)
    for name, value in change.items():
        setattr(c.c, name, c.refs.data_ptr() + 4 if name == "refs" else value)
    with pytest.raises(vb.VBError) as e:
        ctx.pages_extend(c, ints([0]), ints([1]))
    assert e.value.code == vb.VB_ERR_INVALID_ARG


def test_refused_calls(ctx):
    c, other = new_cache(ctx), new_cache(ctx, hd=32)
    for call in (lambda: ctx.pages_compact(c, other), lambda: ctx.pages_compact(c, c),
                 lambda: ctx.pages_compact(c, new_cache(ctx, most=9)),
                 lambda: ctx.pages_extend(c, ints(range(7)), ints(range(7)))):
        with pytest.raises(vb.VBError) as e:
            call()
        assert e.value.code == vb.VB_ERR_INVALID_ARG
    with pytest.raises(ValueError):
        ctx.pages_extend(c, ints([0, 1]), ints([1]))


# ------------------------------------------------- head norms and rotation
def qk_case(ctx, type, T, nh, nkv, hd, rot=0, adjacent=False, norm=True, weights=True, store=True, P=16, pad=0, seed=0,
            flags=0, pool=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[type]
    width = (nh + 2 * nkv) * hd + pad
    big = (torch.randn(T, width, generator=g, device="cuda") * 3).to(dtype)
    q, k, v = (big[:, a * hd:b * hd] for a, b in ((0, nh), (nh, nh + nkv), (nh + nkv, nh + 2 * nkv)))
    rows = 3 * P
    rope = torch.from_numpy(vb.rope_table(rot or hd, 10000.0, False, rows)).cuda()
    w = [1 + 0.3 * torch.randn(hd, generator=g, device="cuda") for _ in range(2)] if weights else [None, None]
    out, kout = torch.full((T, nh * hd), 7.0, dtype=dtype, device="cuda"), torch.full((T, nkv * hd), 7.0, dtype=dtype, device="cuda")
    n_seqs = max(1, -(-T // (rows - 1)))
    c = None
    seq, row = torch.arange(T) // (rows - 1), torch.arange(T) % (rows - 1) + 1
    if store:
        c = new_cache(ctx, 2, 3 * n_seqs + 2, nkv, P, hd, n_seqs, 3, pool or (torch.bfloat16 if type == "f32" else dtype))
        ctx.pages_extend(c, ints(np.arange(n_seqs)), ints([rows] * n_seqs))
    args = vb.QKArgs(q, k, v, heads=nh, kv_heads=nkv, head_dim=hd, q_out=out, k_out=kout, rope=rope, pos=ints(row), q_weight=w[0],
                     k_weight=w[1], norm=norm, eps=1e-5, rot_dim=rot, adjacent=adjacent, flags=flags, pages=c, layer=1,
                     seq=ints(seq), row=ints(row))
    wn = [None if x is None else x.cpu().numpy() for x in w]
    cs = rope.cpu().numpy()[row.numpy()]
    ref = [M.qk(x.float().cpu().numpy().reshape(T, -1, hd), y, 1e-5, cs, rot or hd, adjacent, norm) for x, y in ((q, wn[0]), (k, wn[1]))]
    return args, out, kout, c, v, ref, (seq, row)


HALF = {torch.float32: 0.0, torch.float16: 2.0 ** -12, torch.bfloat16: 2.0 ** -9}


def assert_rows(got, ref, dtype):
    got = got.float().cpu().numpy().astype(np.float64).reshape(ref.shape)
    top = np.abs(ref).max(-1, keepdims=True)
    assert np.all(np.abs(got - ref) <= top * 2.0 ** -20 + np.abs(ref) * 2.0 * HALF[dtype])


@pytest.mark.parametrize("type", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,nh,nkv,hd,rot,adjacent,norm,weights,pad", [
    (1, 16, 2, 128, 0, False, True, True, 0),
    (200, 16, 2, 128, 0, False, False, False, 0),
    (47, 3, 1, 64, 32, False, True, True, 4),
    (33, 4, 4, 96, 48, True, True, False, 3),         # rows that no 4-value access fits
    (5, 2, 1, 256, 128, True, True, True, 0),
    (9, 5, 5, 8, 0, False, True, True, 1),
    (7, 2, 2, 40, 24, False, True, True, 0),
    (95, 8, 2, 80, 16, False, True, True, 0),
])
def test_qk_norm_rope(ctx, type, T, nh, nkv, hd, rot, adjacent, norm, weights, pad):
    args, out, kout, c, v, (rq, rk), (seq, row) = qk_case(ctx, type, T, nh, nkv, hd, rot, adjacent, norm, weights, True, 16, pad)
    before = rows_of(c)
    ctx.qk_norm_rope(args)
    assert ctx.device_status() == (0, 0)
    assert_rows(out, rq, out.dtype)
    assert_rows(kout, rk, out.dtype)
    page = c.table.long().cpu()[seq, row // 16]
    k_rows, v_rows = (x[1][page, :, row % 16] for x in (c.k.cpu(), c.v.cpu()))
    assert torch.equal(k_rows.reshape(T, -1), kout.cpu().to(c.k.dtype))
    assert torch.equal(v_rows.reshape(T, -1), v.cpu().to(c.k.dtype))
    after = rows_of(c)
    written = np.zeros(after.shape[2:5], bool)
    written[page[:, None], np.arange(nkv)[None], (row % 16)[:, None]] = True
    assert np.array_equal(after[0], before[0]) and np.array_equal(after[1][:, ~written], before[1][:, ~written])


def test_qk_is_in_place_when_asked(ctx):
    args, out, kout, c, v, (rq, rk), _ = qk_case(ctx, "bf16", 13, 4, 2, 128)
    args.c.q_out, args.c.ldq_out = args.c.q, args.c.ldq
    args.c.k_out, args.c.ldk_out = args.c.k, args.c.ldk
    ctx.qk_norm_rope(args)
    assert_rows(args._keep[0], rq, torch.bfloat16)
    assert_rows(args._keep[1], rk, torch.bfloat16)


def test_qk_without_norm_is_rope_neox_and_kv_write(ctx):
    """The framework's own rotation and cache rounding, bit for bit."""
    T, nh, nkv, hd = 21, 16, 2, 128
    args, out, kout, c, v, _, (seq, row) = qk_case(ctx, "f32", T, nh, nkv, hd, norm=False, weights=False, flags=vb.OUT_BF16)
    table = torch.from_numpy(vb.rope_table(hd, 10000.0, True, 64)).cuda()
    args.c.rope, args.c.rope_rows = table.data_ptr(), 64
    want = args._keep[0].contiguous()
    ctx.rope_neox(want, hd, nh, T, args._keep[6], 10000.0)
    ctx.qk_norm_rope(args)
    torch.cuda.synchronize()
    # a product may be contracted with the sum here: one bf16 unit at most, and rarely
    d = (out != want).float().mean().item()
    assert d < 1e-3 and torch.allclose(out, want, rtol=2.0 ** -7, atol=1e-6)


def test_qk_skips_tokens_without_a_place(ctx):
    args, out, kout, c, v, (rq, rk), (seq, row) = qk_case(ctx, "f32", 6, 2, 1, 64)
    s, r = ints([0, -1, 1, 0, 0, 0]), ints([1, 2, 3, 48, -1, 6])
    pos = ints([1, 2, 3, 4, 5, 48])
    args.c.seq, args.c.row, args.c.pos = s.data_ptr(), r.data_ptr(), pos.data_ptr()
    before = rows_of(c)
    ctx.qk_norm_rope(args)
    rc, code = ctx.device_status()
    assert rc == vb.VB_ERR_BACKEND and code in (vb.DEV_QK_ROW, vb.DEV_QK_POS)
    assert ctx.device_status() == (0, 0)
    got = out.cpu().numpy()
    assert not got[2:].any()                                      # no such sequence, row past the table, negative row, no such position
    assert_rows(out[:2], rq[:2], torch.float32)                   # sequence -1: computed, not stored
    after = rows_of(c)
    page = int(c.table[0, 0])
    after[1][:, page, 0, 1] = before[1][:, page, 0, 1]
    assert np.array_equal(after, before)


@pytest.mark.parametrize("change", [
    dict(type=vb.TYPE_Q8_0), dict(type=vb.TYPE_F16), dict(head_dim=12), dict(head_dim=512), dict(rot_dim=20), dict(rot_dim=72),
    dict(n_heads=0), dict(n_tokens=-1), dict(layer=2), dict(layer=-1), dict(n_kv_heads=1), dict(ldq=100), dict(q=0),
    dict(v=0), dict(seq=0), dict(pos=0), dict(flags=6), dict(q_out=2), dict(rope=8)])
def test_qk_refusals(ctx, change):
    args = qk_case(ctx, "f32", 4, 2, 2, 64)[0]
    if change == dict(type=vb.TYPE_F16):
        args.c.ldq = args.c.ldk = args.c.ldv = args.c.ldq_out = args.c.ldk_out = 0     # F16 rows over a BF16 cache
    for name, value in change.items():
        setattr(args.c, name, value)
    with pytest.raises(vb.VBError) as e:
        ctx.qk_norm_rope(args)
    assert e.value.code == vb.VB_ERR_INVALID_ARG and "vb_qk_norm_rope" in ctx.last_error()


# ------------------------------------------------ drafted-token attention
R = {"f32": 2.0 ** -14, "bf16": 2.0 ** -7, "f16": 2.0 ** -10}


def tree_case(ctx, type, lens, drafted, nh, nkv, hd, P, mask="tree", seed=0, layers=2, extra_words=0, q_scale=1.0, pad=0,
              pool_dtype=None):
    rng = np.random.default_rng(seed)
    dtype = TYPES[type]
    cd = torch.bfloat16 if type == "f32" else dtype
    n = len(lens)
    most = max(1, -(-max(lens) // P)) + 1
    pages = sum(-(-x // P) for x in lens) + 4
    c = new_cache(ctx, layers, pages, nkv, P, hd, n + 1, most, cd, seed)
    order = rng.permutation(pages).astype(np.int32)
    table, at = np.full((n + 1, most), -1, np.int32), 0
    seqs = rng.permutation(n + 1)[:n].astype(np.int32)
    length = np.zeros(n + 1, np.int32)
    for i, x in enumerate(lens):
        m = -(-x // P)
        table[seqs[i], :m] = order[at:at + m]
        at += m
        length[seqs[i]] = x
    c.table.copy_(ints(table))
    c.length.copy_(ints(length))
    total = sum(drafted)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = (torch.randn(total, nh * hd + pad, generator=g, device="cuda") * q_scale).to(dtype)[:, :nh * hd]
    out = torch.full((total, nh * hd + pad), 3.0, dtype=dtype, device="cuda")[:, :nh * hd]
    words = -(-max(list(drafted) + [1]) // 32) + extra_words
    bits, seen = [], []
    for x, t in zip(lens, drafted):
        if mask == "chain":
            b = np.tril(np.ones((t, t), bool))
        elif mask == "tree":
            b = M.tree_mask([j - 1 - int(rng.integers(0, min(j, 4) + 1)) for j in range(t)])
        else:
            b = rng.random((t, t)) < 0.3                          # any bits, empty rows among them
        bits.append(b)
        seen.append(np.concatenate((np.ones((t, x - t), bool), b), 1))
    packed = None
    if mask != "chain":
        packed = np.concatenate([M.pack_mask(b, words) for b in bits]) if total else np.zeros((0, words), np.int32)
        # bits past a sequence's draft say nothing
        if mask == "tree":
            for i, t in enumerate(drafted):
                rows = slice(sum(drafted[:i]), sum(drafted[:i + 1]))
                if t % 32 and t:
                    packed[rows, t // 32] |= np.int32(-1) << np.int32(t % 32)
        packed = ints(packed)
    start = ints(np.cumsum([0] + list(drafted)))
    args = vb.TreeArgs(q, c, layers - 1, ints(seqs), start, out, heads=nh, max_tokens=max(list(drafted) + [1]), mask=packed)
    return dict(args=args, q=q, out=out, c=c, table=table, seqs=seqs, seen=seen, lens=lens, drafted=drafted, nh=nh, nkv=nkv,
                hd=hd, P=P, layer=layers - 1, type=type)


def tree_ref(t):
    """(formula in 64 bits, error bound) of every output."""
    hd, P, scale = t["hd"], t["P"], 1.0 / np.sqrt(t["hd"])
    k, v = (x[t["layer"]].float().cpu().numpy() for x in (t["c"].k, t["c"].v))
    q = t["q"].float().cpu().numpy()
    ref, tol, first = np.zeros((q.shape[0], t["nh"] * hd)), np.zeros((q.shape[0], t["nh"] * hd)), 0
    for i, (n, d) in enumerate(zip(t["lens"], t["drafted"])):
        pages = t["table"][t["seqs"][i], :-(-n // P)]
        for h in range(t["nh"]):
            g = h // (t["nh"] // t["nkv"])
            kk, vv = (x[pages, g].reshape(-1, hd)[:n] for x in (k, v))
            qq = q[first:first + d, h * hd:(h + 1) * hd]
            ref[first:first + d, h * hd:(h + 1) * hd] = M.attention(qq, kk, vv, t["seen"][i], scale)
            if n and d:
                s = scale * (np.abs(qq) @ np.abs(np.where(np.isfinite(kk), kk, 0)).T).max()
                big = np.abs(np.where(np.isfinite(vv), vv, 0)).max()
                tol[first:first + d, h * hd:(h + 1) * hd] = big * (4 * 2.0 ** -16 * s + R[t["type"]])
        first += d
    return ref, tol


def check_tree(ctx, t):
    ctx.tree_attention(t["args"])
    assert ctx.device_status() == (0, 0)
    ref, tol = tree_ref(t)
    got = t["out"].float().cpu().numpy().astype(np.float64)
    assert np.all(np.isfinite(got))
    assert np.all(np.abs(got - ref) <= tol), float(np.max(np.abs(got - ref) - tol))
    if np.linalg.norm(ref) > 0:                                   # the bound above is for the worst case; on average far less
        rel = np.linalg.norm(got - ref) / np.linalg.norm(ref)
        assert rel < {"f32": 1e-5, "bf16": 5e-3, "f16": 7e-4}[t["type"]]


@pytest.mark.parametrize("type", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens,drafted,nh,nkv,hd,P,mask", [
    ([384], [1], 16, 2, 128, 16, "tree"),                          # a decode step
    ([1], [1], 16, 2, 128, 16, "chain"),                           # the first row
    ([1, 16, 17, 63, 64, 65, 127, 128, 129, 500], [1] * 10, 8, 2, 128, 16, "chain"),
    ([40, 7, 0, 300, 33], [25, 7, 0, 1, 13], 16, 2, 128, 16, "tree"),      # a draft and nothing before it, no tokens, no rows
    ([70, 12], [64, 12], 4, 4, 64, 32, "any"),                     # rows that see nothing
    ([50, 3], [9, 3], 6, 2, 96, 64, "any"),
    ([300], [40], 8, 1, 256, 128, "tree"),
    ([90, 200], [33, 5], 5, 5, 80, 16, "tree"),
    ([77], [20], 3, 1, 8, 16, "tree"),
    ([150, 31], [150, 31], 16, 2, 128, 16, "chain"),               # prompts
    ([400], [130], 16, 2, 128, 64, "chain"),                       # a prompt's later piece
    ([333], [100], 16, 2, 128, 1024, "tree"),
    ([2500], [3], 16, 2, 128, 32, "tree"),
    ([600, 2000, 100], [70, 16, 17], 16, 1, 64, 16, "tree"),       # 16 heads on one
    ([100, 37], [3, 2], 72, 1, 64, 16, "tree"),                    # more heads on one than a block has rows
    ([90, 200, 16], [2, 1, 16], 300, 1, 32, 16, "any"),
    ([1000], [37], 24, 2, 128, 32, "chain"),                       # blocks of whole tokens, not of a power of two
])
def test_tree_attention(ctx, type, lens, drafted, nh, nkv, hd, P, mask):
    check_tree(ctx, tree_case(ctx, type, lens, drafted, nh, nkv, hd, P, mask))


@pytest.mark.parametrize("hd", [8, 64, 96, 128, 256])
@pytest.mark.parametrize("drafted,nh,nkv", [(1, 1, 1), (4, 2, 2), (3, 1, 1), (1, 8, 2), (2, 4, 2), (1, 3, 1), (1, 10, 2), (5, 2, 2), (2, 4, 1),
                                            (8, 1, 1), (1, 16, 2), (2, 6, 2), (7, 1, 1), (9, 1, 1), (3, 3, 1)])
def test_tree_fp32_of_few_rows(ctx, drafted, nh, nkv, hd):
    """Blocks of up to 4, 8 and 16 rows, within one CTA and across several."""
    check_tree(ctx, tree_case(ctx, "f32", [drafted + 3, 2700, drafted], [drafted, drafted, drafted], nh, nkv, hd, 16, "any", seed=11))


@pytest.mark.parametrize("type,hd", [("f32", 64), ("f32", 128), ("f32", 256), ("bf16", 128), ("bf16", 256), ("f16", 256)])
@pytest.mark.parametrize("drafted,nh,nkv", [(17, 1, 1), (4, 16, 2), (11, 6, 2), (8, 8, 1), (31, 4, 1), (65, 2, 1), (70, 16, 2), (3, 200, 1)])
def test_tree_blocks_of_more_rows(ctx, type, hd, drafted, nh, nkv):
    """Every size of a block of rows, filled and not."""
    check_tree(ctx, tree_case(ctx, type, [drafted + 5, 1500, drafted], [drafted, drafted, drafted], nh, nkv, hd, 16, "any", seed=12))


@pytest.mark.parametrize("type,hd", [("bf16", 128), ("f16", 96), ("bf16", 64)])
@pytest.mark.parametrize("mask", ["any", "chain"])
@pytest.mark.parametrize("lens,drafted", [
    ([700, 40, 129, 1025, 2000, 385], [48, 16, 17, 33, 15, 1]), ([9000], [48]),
    ([33 + 3 * i for i in range(60)], [(7 * i) % 33 for i in range(60)]), ([260, 300], [129, 40])])
def test_tree_blocks_of_one_and_two_row_tiles(ctx, type, hd, mask, lens, drafted):
    """Full blocks, blocks of one row tile and both of them after one another in a CTA; queries by TMA and by threads."""
    check_tree(ctx, tree_case(ctx, type, lens, drafted, 16, 2, hd, 16, mask, seed=13))
    check_tree(ctx, tree_case(ctx, type, lens, drafted, 16, 2, hd, 16, mask, seed=14, pad=3))


@pytest.mark.parametrize("type", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens,drafted,P", [([30000], [2], 64), ([9000, 20000], [1, 1], 16), ([25000, 100], [40, 3], 32)])
def test_tree_many_tiles_for_each_cta(ctx, type, lens, drafted, P):
    """Calls one after another, each CTA working through many tiles of the ring."""
    t = tree_case(ctx, type, lens, drafted, 8, 1, 128, P, seed=8)
    for _ in range(8):
        ctx.tree_attention(t["args"])
    check_tree(ctx, t)


@pytest.mark.parametrize("type", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("drafted", [1, 8, 40])
def test_tree_rings_go_round(ctx, type, drafted):
    """Every CTA goes many times round its ring of tiles, faster than they come."""
    t = tree_case(ctx, type, [200000], [drafted], 2 if drafted > 1 else 1, 1, 128, 64, seed=9, layers=1)
    for _ in range(12):
        ctx.tree_attention(t["args"])
    check_tree(ctx, t)


@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_tree_many_sequences_and_long_chains(ctx, type):
    rng = np.random.default_rng(1)
    lens = rng.integers(0, 60, 900)
    check_tree(ctx, tree_case(ctx, type, lens.tolist(), [int(min(x, d)) for x, d in zip(lens, rng.integers(0, 9, 900))], 2, 1, 8, 16, seed=1))
    # more blocks of tokens than threads in a CTA, in the middle of other sequences
    check_tree(ctx, tree_case(ctx, type, [40, 3300, 9], [4, 3250, 9], 8, 1, 8, 16, "chain", seed=2))
    if type == "bf16":
        check_tree(ctx, tree_case(ctx, type, [3100], [3100], 256, 1, 8, 64, "chain", seed=3))


@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_tree_strided_rows_and_wide_masks(ctx, type):
    check_tree(ctx, tree_case(ctx, type, [90, 64], [30, 20], 4, 2, 128, 16, extra_words=3, pad=8))
    check_tree(ctx, tree_case(ctx, type, [90, 64], [30, 20], 4, 2, 128, 16, pad=3))


@pytest.mark.parametrize("type", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("drafted", [5, 40])
def test_tree_unseen_rows_may_hold_anything(ctx, type, drafted):
    """NaN and infinities past the end, in free pages and in draft rows that a token does not see stay out of its result."""
    t = tree_case(ctx, type, [75, 48 + drafted], [drafted, drafted], 8, 2, 128, 16, "any", seed=4)
    bad = [1, drafted - 1]                                        # draft rows nobody sees, except the last token
    for i in range(2):
        t["seen"][i][:, -drafted:][:-1, bad] = False
        t["seen"][i][-1, -drafted:][bad] = False
    packed = np.concatenate([M.pack_mask(s[:, -drafted:], -(-drafted // 32)) for s in t["seen"]])
    t["args"]._keep[5].copy_(ints(packed))
    used = np.zeros((t["c"].k.shape[1], 16), bool)
    for i, n in enumerate(t["lens"]):
        for r in range(n):
            if r - (n - drafted) not in bad:
                used[t["table"][t["seqs"][i], r // 16], r % 16] = True
    hole = torch.from_numpy(~used).cuda()
    for x, val in ((t["c"].k, float("nan")), (t["c"].v, float("inf"))):
        x[1].masked_fill_(hole[:, None, :, None], val)
    x = t["c"].v[1]
    x[..., 3].masked_fill_(hole[:, None], float("nan"))
    check_tree(ctx, t)


@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_tree_seen_infinities_show(ctx, type):
    """An infinite value that a token sees is in its result, and in no other's."""
    t = tree_case(ctx, type, [60], [20], 2, 2, 64, 16, "tree", seed=2)
    seen = t["seen"][0][:, 40:]
    r = 7
    page, slot = t["table"][t["seqs"][0], (40 + r) // 16], (40 + r) % 16
    t["c"].v[1, page, :, slot, 5] = float("inf")
    ctx.tree_attention(t["args"])
    assert ctx.device_status() == (0, 0)
    got = t["out"].float().cpu().numpy().reshape(20, 2, 64)
    assert np.array_equal(np.isinf(got[:, :, 5]), np.repeat(seen[:, r:r + 1], 2, 1))
    t["c"].v[1, page, :, slot, 5] = 0.0
    ref, tol = tree_ref(t)
    keep = np.ones((20, 2, 64), bool)
    keep[:, :, 5] = ~seen[:, r:r + 1]
    keep = keep.reshape(20, -1)
    assert np.all((np.abs(got.reshape(20, -1) - ref) <= tol)[keep])


@pytest.mark.parametrize("type", ["f32", "bf16", "f16"])
def test_tree_large_scores(ctx, type):
    """Scores in the hundreds: one row takes all the weight."""
    t = tree_case(ctx, type, [700], [12], 8, 2, 128, 16, seed=6, q_scale=40.0)
    ctx.tree_attention(t["args"])
    ref, tol = tree_ref(t)
    got = t["out"].float().cpu().numpy()
    assert np.all(np.isfinite(got)) and np.all(np.abs(got - ref) <= tol)


def test_tree_scale(ctx):
    t = tree_case(ctx, "f32", [200], [6], 4, 2, 64, 16, seed=7)
    t["args"].c.scale = 0.5
    ctx.tree_attention(t["args"])
    got = t["out"].cpu().numpy()
    t["q"].mul_(0.5 * 8.0)                                        # the same scores at the default scale
    ref, tol = tree_ref(t)
    assert np.all(np.abs(got - ref) <= tol)


@pytest.mark.parametrize("type,lens,drafted", [("f32", [3000, 70], [2, 20]), ("bf16", [5000, 1300], [48, 16]), ("bf16", [700], [700])])
def test_tree_gives_the_same_bits_again(ctx, type, lens, drafted):
    t = tree_case(ctx, type, lens, drafted, 16, 2, 128, 16, "chain")
    got = []
    for _ in range(3):
        t["out"].fill_(1.0)
        ctx.tree_attention(t["args"])
        torch.cuda.synchronize()
        got.append(t["out"].clone())
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


@pytest.mark.parametrize("type,drafted", [("f32", 2), ("bf16", 1), ("bf16", 9), ("f16", 40)])
def test_steps_replayed_from_a_graph(ctx, type, drafted):
    """extend, attention and keep captured once: each replay finds the lengths of the one before, with the bits of direct calls."""
    dtype = TYPES[type]
    own = torch.cuda.Stream()
    both = [new_cache(ctx, pages=60, P=16, hd=128, most=30, dtype=torch.bfloat16 if type == "f32" else dtype, seed=5) for _ in range(2)]
    n = 2
    seqs, rows, kept = ints([3, 1]), ints([drafted] * n), ints([1, min(drafted, 2)])
    path, start = ints([[drafted - 1, 0], [0, drafted - 1]]), ints([0, drafted, 2 * drafted])
    mask = ints(M.pack_mask(np.tile(M.tree_mask([j - 1 - (j > 2) for j in range(drafted)]), (n, 1)), -(-drafted // 32)))
    q = torch.randn(n * drafted, 16 * 128, device="cuda").to(dtype)
    got = [torch.zeros_like(q) for _ in both]
    args = [vb.TreeArgs(q, c, 1, seqs, start, o, heads=16, max_tokens=drafted, mask=mask) for c, o in zip(both, got)]

    def step(i):
        ctx.pages_extend(both[i], seqs, rows)
        ctx.tree_attention(args[i])
        ctx.pages_keep(both[i], seqs, rows, kept, path)

    for c in both:
        ctx.pages_init(c)
        ctx.pages_extend(c, seqs, ints([100, 37]))
    torch.cuda.synchronize()
    ctx.set_stream(own.cuda_stream)
    step(0)
    step(1)
    ctx.sync()
    ctx.graph_begin()
    step(1)
    g = ctx.graph_end()
    for _ in range(4):
        step(0)
        ctx.graph_launch(g)
        ctx.sync()
        assert torch.equal(got[0], got[1]) and torch.equal(both[0].length, both[1].length) and bool(got[1].any())
    ctx.graph_destroy(g)
    ctx.set_stream(1)
    assert both[0].length.tolist() == [0, 37 + 5 * min(drafted, 2), 0, 105, 0, 0]
    assert ctx.device_status() == (0, 0) and all(ctx.pages_status(c)[0] == 0 for c in both)


def test_tree_past_32_bit_offsets(ctx):
    """A layer whose rows lie past 2^31 elements of the pool."""
    nkv, P, hd, pages = 2, 64, 128, 70000
    k, v = (torch.empty(3, pages, nkv, P, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    new = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    c = vb.Pages(k, v, new(1, 3), new(1), new(pages), new(4))
    table = np.array([[69990, 3, 69999]], np.int32)
    c.table.copy_(ints(table))
    c.length.fill_(150)
    for p in table[0]:
        k[2, p].normal_()
        v[2, p].normal_()
    q = torch.randn(4, 16 * hd, device="cuda")
    out = torch.zeros_like(q)
    rope = torch.from_numpy(vb.rope_table(hd, 10000.0, False, 150)).cuda()
    args = vb.TreeArgs(q, c, 2, ints([0]), ints([0, 4]), out, heads=16, max_tokens=4)
    kv = torch.randn(4, 2 * nkv * hd, device="cuda")
    place = ints([146, 147, 148, 149])
    qk = vb.QKArgs(q, kv[:, :nkv * hd], kv[:, nkv * hd:], heads=16, kv_heads=nkv, head_dim=hd, q_out=q, rope=rope, pos=place,
                   pages=c, layer=2, seq=ints([0] * 4), row=place)
    ctx.qk_norm_rope(qk)
    ctx.tree_attention(args)
    assert ctx.device_status() == (0, 0)
    small = [x[2, table[0].tolist()].float().cpu().numpy() for x in (k, v)]
    assert np.array_equal(small[1][2, :, 18:22].transpose(1, 0, 2).reshape(4, -1), kv[:, nkv * hd:].bfloat16().float().cpu().numpy())
    for h in range(16):
        kk, vv = (x[:, h // 8].reshape(-1, hd)[:150] for x in small)
        ref = M.attention(q[:, h * hd:(h + 1) * hd].cpu().numpy(), kk, vv, np.tril(np.ones((4, 150), bool), 146), hd ** -0.5)
        got = out[:, h * hd:(h + 1) * hd].cpu().numpy()
        assert np.linalg.norm(got - ref) <= 1e-5 * np.linalg.norm(ref)


@pytest.mark.parametrize("what,code", [("length", vb.DEV_TREE_SEQ), ("seq", vb.DEV_TREE_SEQ), ("long", vb.DEV_TREE_SEQ),
                                       ("most", vb.DEV_TREE_SEQ), ("words", vb.DEV_TREE_SEQ), ("page", vb.DEV_TREE_PAGE)])
@pytest.mark.parametrize("drafted", [4, 40])
def test_tree_bad_device_values_are_reported(ctx, what, code, drafted):
    """The other sequence's tokens come out right."""
    t = tree_case(ctx, "bf16", [120, 90], [drafted, drafted], 8, 2, 128, 16, "tree", seed=3)
    a, s = t["args"], int(t["seqs"][0])
    if what == "length":
        t["c"].length[s] = drafted - 1
    elif what == "seq":
        a._keep[2][0] = 99
    elif what == "long":
        t["c"].length[s] = 10 ** 6
    elif what == "most":
        a._keep[3][0] = -1                                        # a start before the rows of q
    elif what == "words":
        a.c.mask_words, a.c.max_tokens = 1, 64
        if drafted <= 32:
            pytest.skip("one word holds the draft")
    else:
        t["c"].table[s, 2] = t["c"].k.shape[1]
    ctx.tree_attention(a)
    assert ctx.device_status() == (vb.VB_ERR_BACKEND, code)
    assert ctx.device_status() == (0, 0)
    if what == "words":
        return
    ref, tol = tree_ref(t | {"table": np.where(t["table"] >= t["c"].k.shape[1], 0, t["table"])})
    got = t["out"].float().cpu().numpy()
    assert np.all((np.abs(got - ref) <= tol)[drafted:])
    if what in ("length", "seq", "long"):
        assert not got[:drafted].any()


@pytest.mark.parametrize("change", [
    dict(type=vb.TYPE_Q8_0), dict(type=vb.TYPE_F16), dict(layer=2), dict(layer=-1), dict(n=-1), dict(n_tokens=-1),
    dict(max_tokens=-1), dict(n_heads=0), dict(n_heads=5), dict(ldq=8), dict(ldo=8), dict(scale=-1.0),
    dict(scale=float("nan")), dict(mask_words=0), dict(q=0), dict(out=0), dict(seqs=0), dict(start=0), dict(pages=0)])
def test_tree_refusals(ctx, change):
    t = tree_case(ctx, "f32", [20], [4], 4, 2, 64, 16)
    for name, value in change.items():
        setattr(t["args"].c, name, value)
    with pytest.raises(vb.VBError) as e:
        ctx.tree_attention(t["args"])
    assert e.value.code == vb.VB_ERR_INVALID_ARG and "vb_tree_attention" in ctx.last_error()


def test_tree_empty_calls(ctx):
    t = tree_case(ctx, "f32", [20, 30], [0, 0], 4, 2, 64, 16)
    ctx.tree_attention(t["args"])
    t["args"].c.n = 0
    ctx.tree_attention(t["args"])
    assert ctx.device_status() == (0, 0)


def test_captured_steps_outlive_larger_calls():
    """Calls that need larger workspaces come between a step's capture and its replays."""
    ctx, own = vb.Context(0), torch.cuda.Stream()                 # (a new context: its workspaces are still small)
    ctx.set_stream(own.cuda_stream)
    g0 = torch.Generator(device="cuda").manual_seed(3)
    both = [new_cache(ctx, pages=60, P=16, hd=128, most=30, seed=5) for _ in range(2)]
    seqs, one, path = ints([3, 1]), ints([1, 1]), ints([[0], [0]])
    q = torch.randn(2, 16 * 128, generator=g0, device="cuda")
    att, y = ([torch.zeros(n, 2048, device="cuda") for _ in both] for n in (2, 16))
    args = [vb.TreeArgs(q, c, 1, seqs, ints([0, 1, 2]), o, heads=16, max_tokens=1) for c, o in zip(both, att)]
    w = ctx.weight(vb.TYPE_F16, 2048, 2048, np.random.default_rng(0).standard_normal((2048, 2048)).astype(np.float16))
    x = torch.randn(64, 2048, generator=g0, device="cuda")
    prompt = tree_case(ctx, "bf16", [700], [700], 16, 2, 128, 16, "chain")
    wide, to = (new_cache(ctx, 1, 200000, 1, 16, 8, 2, 8) for _ in range(2))
    torch.cuda.synchronize()

    def step(i):
        ctx.pages_extend(both[i], seqs, one)
        ctx.tree_attention(args[i])
        ctx.pages_keep(both[i], seqs, one, one, path)
        ctx.matmul(w, x, 16, y[i])

    for c in both:
        ctx.pages_init(c)
        ctx.pages_extend(c, seqs, ints([100, 300]))
    step(0)
    step(1)
    ctx.sync()
    ctx.graph_begin()
    step(1)
    g = ctx.graph_end()
    ctx.tree_attention(prompt["args"])
    ctx.pages_compact(wide, to)
    ctx.matmul(w, x, 64, torch.zeros(64, 2048, device="cuda"))
    ctx.sync()
    others = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(32)]
    torch.cuda.synchronize()
    for _ in range(3):
        step(0)
        ctx.graph_launch(g)
        ctx.sync()
        assert torch.equal(att[0], att[1]) and torch.equal(y[0], y[1]) and bool(att[1].any()) and bool(y[1].any())
    assert all(bool(o.isnan().all()) for o in others)
    ref, tol = tree_ref(prompt)
    assert np.all(np.abs(prompt["out"].float().cpu().numpy() - ref) <= tol)
    assert ctx.device_status() == (0, 0) and all(ctx.pages_status(c)[0] == 0 for c in both)
    ctx.graph_destroy(g)
    w.release()
    ctx.close()


@pytest.mark.parametrize("call", ["fork", "truncate"])
def test_an_error_in_a_call_of_many_requests_changes_nothing(ctx, call):
    """CTAs of a later wave start while the first record the error."""
    n, most, half = 12000, 1024, 6000
    c = new_cache(ctx, 1, 16, 1, 16, 8, n, most)
    row = torch.arange(n, device="cuda", dtype=torch.int32) % 8
    c.table[:, :3] = row[:, None]
    c.length.fill_(40)
    c.refs[:8] = 3 * n // 8
    before = [x.clone() for x in (c.table, c.length, c.refs, c.k, c.v)]
    seqs = np.arange(half)
    for at in (half - 1, 0, half // 2):
        a = seqs + half if call == "fork" else seqs.copy()
        b = seqs.copy() if call == "fork" else np.zeros(half, int)
        (a if call == "fork" else b)[at] = -1                     # a source out of range, a negative length
        getattr(ctx, "pages_" + call)(c, ints(a), ints(b))
        assert ctx.pages_status(c)[1:3] == (vb.PAGES_SEQ if call == "fork" else vb.PAGES_COUNT, at)
        assert all(torch.equal(x, y) for x, y in zip((c.table, c.length, c.refs, c.k, c.v), before))


@pytest.mark.parametrize("type,hd,drafted,nh,nkv,before", [
    ("f32", 64, 40, 8, 2, 300), ("f32", 128, 40, 8, 2, 20000), ("f32", 128, 20, 8, 2, 20000), ("f32", 128, 2, 8, 2, 9000),
    ("f32", 256, 10, 8, 2, 9000), ("bf16", 256, 40, 32, 2, 300), ("f16", 256, 40, 32, 2, 20000), ("bf16", 256, 40, 8, 2, 9000),
    ("bf16", 128, 40, 16, 2, 20000), ("f16", 64, 12, 16, 2, 9000), ("bf16", 128, 1, 16, 2, 9000)])
def test_tree_seen_infinities_show_in_every_form(ctx, type, hd, drafted, nh, nkv, before):
    """Every size of a block, held by one CTA and by several; calls one after another give the same."""
    t = tree_case(ctx, type, [before + drafted, drafted + 9], [drafted, drafted], nh, nkv, hd, 16, "any" if drafted > 1 else "tree", seed=15)
    bad = [(0, 0, 3), (0, drafted - 1, hd - 1), (1, drafted // 2, 0)]       # sequence, draft row, column
    for value in (float("inf"), float("nan")):
        for i, r, col in bad:
            at = t["lens"][i] - drafted + r
            t["c"].v[1, t["table"][t["seqs"][i], at // 16], :, at % 16, col] = value
        got = []
        for _ in range(3):
            ctx.tree_attention(t["args"])
            torch.cuda.synchronize()
            got.append(t["out"].float().cpu().numpy().reshape(2, drafted, nh, hd))
        assert ctx.device_status() == (0, 0)
        want = np.zeros((2, drafted, hd), bool)
        for i, r, col in bad:
            want[i, :, col] |= t["seen"][i][:, t["lens"][i] - drafted + r]
        for x in got:
            assert np.array_equal(~np.isfinite(x), np.broadcast_to(want[:, :, None], x.shape))
            assert np.array_equal(np.isnan(x), ~np.isfinite(x) & np.isnan(value))
    for i, r, col in bad:
        at = t["lens"][i] - drafted + r
        t["c"].v[1, t["table"][t["seqs"][i], at // 16], :, at % 16, col] = 0.0
    ref, tol = tree_ref(t)
    ok = np.abs(got[-1].reshape(ref.shape) - ref) <= tol
    assert np.all(ok | np.broadcast_to(want[:, :, None], got[0].shape).reshape(ref.shape))


@pytest.mark.parametrize("type,drafted", [("f32", 1), ("bf16", 1), ("f16", 12), ("f32", 30), ("bf16", 48)])
@pytest.mark.parametrize("hd,P", [(64, 64), (64, 128), (64, 1024), (128, 128), (128, 1024)])
def test_tree_tiles_of_few_boxes(ctx, type, drafted, hd, P):
    """Tiles whose copies leave some of the loading warps without one, many of them in a row: whole pages, and sequences of a
    few rows, after one another."""
    long = tree_case(ctx, type, [40000 + drafted], [drafted], 2, 1, hd, P, seed=16, layers=1)
    short = tree_case(ctx, type, [drafted + i % 30 for i in range(400)], [drafted] * 400, 2, 1, hd, P, seed=17, layers=1)
    for t in (long, short):
        for _ in range(4):
            ctx.tree_attention(t["args"])
        check_tree(ctx, t)


def step_args(c, seq, place, nh=4, seed=0):
    """(norm and store, attention) of one sequence's tokens at `place`."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    kv, hd, n = c.k.shape[2], c.k.shape[4], len(place)
    qkv = torch.randn(n, (nh + 2 * kv) * hd, generator=g, device="cuda")
    q, out = torch.full((n, nh * hd), 7.0, device="cuda"), torch.full((n, nh * hd), 7.0, device="cuda")
    store = vb.QKArgs(qkv[:, :nh * hd], qkv[:, nh * hd:(nh + kv) * hd], qkv[:, (nh + kv) * hd:], heads=nh, kv_heads=kv,
                      head_dim=hd, q_out=q, pages=c, layer=1, seq=ints([seq] * n), row=ints(place))
    return store, vb.TreeArgs(q, c, 1, ints([seq]), ints([0, n]), out, heads=nh, max_tokens=n), qkv, q, out


def test_a_step_after_a_failed_extend_writes_nowhere(ctx):
    """A fork cut back into a shared page cannot be extended: its rows do not land on its parent's."""
    c = new_cache(ctx, pages=5, most=4)
    m = M.PoolModel(rows_of(c), 6, 4)
    for f, a in (("extend", ([0], [40])), ("fork", ([0], [1])), ("truncate", ([1], [35])), ("extend", ([2], [32]))):
        getattr(ctx, "pages_" + f)(c, *(ints(x) for x in a))
        getattr(m, f)(*a)
    ctx.pages_extend(c, ints([1]), ints([2]))                     # wants a page of its own, and there is none
    store, attend, qkv, q, out = step_args(c, 1, [35, 36])
    ctx.qk_norm_rope(store)
    assert ctx.device_status() == (vb.VB_ERR_BACKEND, vb.DEV_QK_ROW)
    ctx.tree_attention(attend)
    assert ctx.device_status() == (vb.VB_ERR_BACKEND, vb.DEV_TREE_SEQ)
    assert not q.any() and not out.any()
    assert_state(c, m)
    # the error is read and the rows are still not held
    assert ctx.pages_status(c)[:3] == (vb.VB_ERR_BACKEND, vb.PAGES_FULL, 0)
    ctx.qk_norm_rope(store)
    assert ctx.device_status() == (vb.VB_ERR_BACKEND, vb.DEV_QK_ROW)
    assert_state(c, m)
    # with a page free the same step goes through, on a copy of the shared one
    for f, a in (("truncate", ([2], [0])), ("extend", ([1], [2]))):
        getattr(ctx, "pages_" + f)(c, *(ints(x) for x in a))
        getattr(m, f)(*a)
    ctx.qk_norm_rope(store)
    ctx.tree_attention(attend)
    assert ctx.device_status() == (0, 0) and bool(out.any())
    kv = qkv[:, 4 * 64:].bfloat16().view(torch.int16).cpu().numpy().reshape(2, 2, 2, 64)
    for t, row in enumerate((35, 36)):
        m.data[1, :, m.table[1, row // 16], :, row % 16] = kv[t]
    assert m.table[1, 2] != m.table[0, 2]
    assert_state(c, m)


def test_rows_are_stored_while_they_are_held(ctx):
    """Rows at and past a sequence's length are skipped, whatever its page holds; shared ones that it holds are stored."""
    c = new_cache(ctx)
    ctx.pages_extend(c, ints([0]), ints([21]))
    ctx.pages_fork(c, ints([0]), ints([1]))
    ctx.pages_truncate(c, ints([0]), ints([20]))
    store, _, qkv, q, _ = step_args(c, 0, [18, 19, 20, 31])
    before = rows_of(c)
    ctx.qk_norm_rope(store)
    assert ctx.device_status() == (vb.VB_ERR_BACKEND, vb.DEV_QK_ROW)
    assert torch.equal(q[:2], qkv[:2, :4 * 64]) and not q[2:].any()
    kv = qkv[:, 4 * 64:].bfloat16().view(torch.int16).cpu().numpy().reshape(4, 2, 2, 64)
    page = int(c.table[1, 1])
    before[1, :, page, :, 2], before[1, :, page, :, 3] = kv[0], kv[1]
    assert np.array_equal(rows_of(c), before)


@pytest.mark.parametrize("length", [-5, -40, -2 ** 31, 65, 2 ** 31 - 1])
@pytest.mark.parametrize("call,args", [("extend", ([2], [1])), ("extend", ([0], [0])), ("keep", ([2], [3], [2], [[1, 2]])),
                                       ("keep", ([0], [0], [0], [[0]]))])
def test_a_broken_length_is_reported(ctx, call, args, length):
    """A length that is no number of rows leads nowhere outside the table."""
    c, m = start_state(ctx)                                       # 4 pages of 16 rows for a sequence
    seq = args[0][0]
    c.length[seq] = length
    m.length[seq] = length
    getattr(ctx, "pages_" + call)(c, *(ints(x) for x in args))
    assert ctx.pages_status(c)[:3] == (vb.VB_ERR_BACKEND, vb.PAGES_LONG, 0)
    assert_state(c, m)


@pytest.mark.parametrize("type,drafted,nh", [("f32", 1, 2), ("f32", 40, 8), ("bf16", 1, 2), ("bf16", 12, 16), ("bf16", 40, 16),
                                             ("f16", 40, 16), ("f16", 12, 16)])
@pytest.mark.parametrize("row", [0, 4, 20, 70, 130, 5003])
def test_tree_infinite_scores_show(ctx, type, drafted, nh, row):
    """An infinite score leaves no weight that can be named: NaN, wherever its row lies in the cache and however it is cut.  A
    row whose score is minus infinity has no weight (fp32 queries: their terms' products with it cancel to NaN)."""
    t = tree_case(ctx, type, [9000 + drafted], [drafted], nh, 1, 128, 16, "tree", seed=18)
    t["q"][:, 5::128] = t["q"][:, 5::128].abs() + 1               # each head's value 5 is positive
    page, at = t["table"][t["seqs"][0], row // 16], row % 16
    t["c"].k[1, page, 0, at, 5] = float("inf")
    ctx.tree_attention(t["args"])
    assert ctx.device_status() == (0, 0)
    assert bool(t["out"].isnan().all())
    if type == "f32":
        return
    t["c"].k[1, page, 0, at, 5] = float("-inf")
    ctx.tree_attention(t["args"])
    t["c"].k[1, page, 0, at] = 0
    t["seen"][0][:, row] = False
    ref, tol = tree_ref(t)
    got = t["out"].float().cpu().numpy()
    assert np.all(np.abs(got - ref) <= tol)


@pytest.mark.parametrize("type", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd,row", [(128, 0), (128, 4), (128, 20), (64, 9), (64, 40)])
def test_tree_infinite_scores_show_in_whole_items(ctx, type, hd, row):
    """The same in items that a CTA holds alone, after a tile that every token sees."""
    n, drafted = 600, 20
    t = tree_case(ctx, type, [128 + drafted] * n, [drafted] * n, 16, 1, hd, 16, "tree", seed=19)
    t["q"][:, 5::hd] = t["q"][:, 5::hd].abs() + 1
    with_inf = np.arange(n) % 3 == 1
    t["c"].k[1, t["table"][t["seqs"][with_inf], row // 16], 0, row % 16, 5] = float("inf")
    ctx.tree_attention(t["args"])
    assert ctx.device_status() == (0, 0)
    nan = t["out"].isnan().cpu().numpy().reshape(n, -1)
    assert nan[with_inf].all() and not nan[~with_inf].any()


@pytest.mark.parametrize("pool", ["bf16", "f16"])
def test_qk_rounds_cache_rows_once(ctx, pool):
    """Results rounded to bf16 beside a cache of another type: its rows come from the unrounded values."""
    args, out, kout, c, v, (rq, rk), (seq, row) = qk_case(ctx, "f32", 40, 4, 2, 64, flags=vb.OUT_BF16, pool=TYPES[pool])
    plain = qk_case(ctx, "f32", 40, 4, 2, 64, pool=TYPES[pool])
    ctx.qk_norm_rope(args)
    ctx.qk_norm_rope(plain[0])
    torch.cuda.synchronize()
    assert torch.equal(out, plain[1].bfloat16().float()) and torch.equal(kout, plain[2].bfloat16().float())
    page = c.table.long().cpu()[seq, row // 16]
    k_rows, v_rows = (x[1].cpu()[page, :, row % 16].reshape(40, -1) for x in (c.k, c.v))
    assert torch.equal(k_rows, plain[2].cpu().to(TYPES[pool])) and torch.equal(v_rows, v.cpu().to(TYPES[pool]))


def test_every_error_is_reported_once(ctx):
    """The report clears the word before what the next call records."""
    bad, good = (tree_case(ctx, "f32", [20], [4], 4, 2, 64, 16) for _ in range(2))
    bad["args"]._keep[2][0] = 99
    own = torch.cuda.Stream()
    torch.cuda.synchronize()
    ctx.set_stream(own.cuda_stream)
    for _ in range(100):
        ctx.tree_attention(bad["args"])
        assert ctx.device_status() == (vb.VB_ERR_BACKEND, vb.DEV_TREE_SEQ)
        ctx.tree_attention(bad["args"])
        assert ctx.device_status() == (vb.VB_ERR_BACKEND, vb.DEV_TREE_SEQ)
        ctx.tree_attention(good["args"])
        assert ctx.device_status() == (0, 0)
    ctx.set_stream(1)


def terms_case(ctx, T, group, hd, rows):
    """fp32 queries over `rows` rows of zeros before a draft that no token sees; row r of the cache: put(r, k, v)."""
    t = tree_case(ctx, "f32", [rows + T], [T], group, 1, hd, 16, "any", seed=20)
    t["args"]._keep[5].zero_()
    t["args"].c.scale = 1.0
    t["c"].k[1], t["c"].v[1] = 0, 0
    t["q"].zero_()

    def put(r, k, v):
        at = (1, int(t["table"][t["seqs"][0], r // 16]), 0, r % 16)
        t["c"].k[at][:2] = torch.tensor(k, device="cuda")
        t["c"].v[at] = v
    return t, put


FP32_FORMS = [(1, 2, 64), (2, 2, 128), (1, 4, 256), (2, 3, 64), (1, 8, 128), (4, 2, 256), (1, 12, 64), (2, 8, 128), (1, 16, 256),
              (3, 8, 64), (3, 8, 128), (3, 8, 256), (10, 8, 64), (10, 8, 128), (20, 8, 64), (20, 8, 128), (20, 8, 256)]


@pytest.mark.parametrize("T,group,hd", FP32_FORMS)
def test_tree_fp32_queries_keep_their_third_term(ctx, T, group, hd):
    """Two rows whose scores differ by what a query value's third bf16 term adds.

    Scores of 46 (in powers of two): their products and the sum of the terms are exact here, the scale's product is rounded to
    2^-19, so the difference of two scores is off by 2^-18, its weight's logarithm by 2^-18 ln 2 and the result by half of that,
    1.3e-6; the power and the sums add less than 5e-7.  Without the term the result is 0 in place of 6.1e-5."""
    t, put = terms_case(ctx, T, group, hd, 2)
    put(0, (1.0, 0.0), 1.0)
    put(1, (0.0, 1.0), -1.0)
    t["q"][:, 0::hd], t["q"][:, 1::hd] = 32 * (1 + 2.0 ** -9 + 2.0 ** -18), 32 * (1 + 2.0 ** -9)
    ctx.tree_attention(t["args"])
    assert ctx.device_status() == (0, 0)
    assert np.all(np.abs(t["out"].cpu().numpy().astype(np.float64) - np.tanh(16 * 2.0 ** -18)) <= 1.8e-6)


@pytest.mark.parametrize("T,group,hd", FP32_FORMS)
def test_tree_fp32_weights_keep_their_third_term(ctx, T, group, hd):
    """32 rows of one weight, of which three bf16 terms are 1/2, 2^-10 and 2^-19, beside a row of weight 1.

    result = 32 p / (1 + 32 p): an error of p itself shrinks to a 17th, the sums of 33 values and the division round a few
    times to 2^-24: 1e-6 holds them.  Without the third term the result is off by 2^-18 of it, 3.6e-6."""
    t, put = terms_case(ctx, T, group, hd, 33)
    for r in range(33):
        put(r, (float(r == 16), 0.0), float(r != 16))
    p = 0.5 * (1 + 2.0 ** -9 + 2.0 ** -18)
    t["q"][:, 0::hd] = -np.log(p)
    ctx.tree_attention(t["args"])
    assert ctx.device_status() == (0, 0)
    assert np.all(np.abs(t["out"].cpu().numpy().astype(np.float64) - 32 * p / (1 + 32 * p)) <= 1e-6)


@pytest.mark.parametrize("rows,pages", [(16, 2 ** 27 - 1), (16, 2 ** 27 - 64), (1024, 2 ** 21 - 1)])
def test_sequences_of_2_to_the_31_rows_are_refused(ctx, rows, pages):
    """A length rounded up to pages or tiles stays a 32-bit number."""
    c = new_cache(ctx)
    c.c.page_rows, c.c.max_pages, c.c.n_pages = rows, pages, 1
    for call in (lambda: ctx.pages_extend(c, ints([0]), ints([1])), lambda: ctx.pages_truncate(c, ints([0]), ints([0]))):
        with pytest.raises(vb.VBError) as e:
            call()
        assert e.value.code == vb.VB_ERR_INVALID_ARG and "too large" in ctx.last_error()
