"""The stack over the paged cache against the CPU oracle's stack, by the same
gate as the other stacks (synth.assert_envelope): prompts, drafted trees path
by path, what is kept of them, and forks."""
import contextlib

import numpy as np
import pytest

import oracle as O
import synth as S

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import paged_lm as PL  # noqa: E402
import vcpm_b200 as vb  # noqa: E402

H, NH, NKV, HD, F, LAYERS = 512, 4, 2, 128, 1024, 2


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    c = vb.Context(0)
    c.set_stream(1)
    yield c
    c.close()


def rows(n):
    return O.bf16_round(S.normal((n, H)))


class Refs:
    """The oracle's stack in both of its accumulations."""

    def __init__(self, wtype, no_rope):
        self.layers = [S.layer(wtype, H, NH, NKV, HD, F) for _ in range(LAYERS)]
        self.fn = S.normal(H, 0.02, 1.0)
        self.cfg = O.LMConfig(H, NH, NKV, HD, F, LAYERS, 1e-5, 10000.0, no_rope, 0.0)
        self.olayers = [S.oracle_layer(wtype, L) for L in self.layers]

    def last(self, steps):
        """Outputs of the last of a sequence's steps (arrays of rows)."""
        got = []
        for f32 in (False, True):
            cache, pos = O.KVCache(LAYERS, 256, NKV, HD), 0
            with O.f32_accumulation() if f32 else contextlib.nullcontext():
                for x in steps:
                    y = O.lm_forward(self.cfg, self.olayers, self.fn, cache, x, len(x), pos)
                    pos += len(x)
            got.append(y)
        return got


@pytest.mark.parametrize("wtype,no_rope", [(O.TYPE_Q8_0, 0), (O.TYPE_F16, 0), (O.TYPE_F16, 1)])
def test_stack_over_pages(ctx, wtype, no_rope):
    ref = Refs(wtype, no_rope)
    cfg = vb.LMConfig(H, NH, NKV, HD, F, LAYERS, 1e-5, 10000.0, no_rope, 0.0, wtype)
    lm = PL.PagedLM(ctx, cfg, ref.layers, ref.fn, seqs=4, pages=24, page_rows=16, most_rows=128)
    up = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    a, b, draft, tail = rows(23), rows(9), rows(6), rows(1)
    got = lm.step(up(np.concatenate([a, b])), [2, 0], [23, 9]).cpu().numpy()
    S.assert_envelope(got[:23], *ref.last([a]))
    S.assert_envelope(got[23:], *ref.last([b]))
    lm.fork([2], [1])
    # sequence 2 drafts a tree, sequence 0 a chain, in one step
    got = lm.step(up(np.concatenate([draft, tail])), [2, 0], [[-1, 0, 0, 1, 2, -1], [-1]]).cpu().numpy()
    for path in ([0, 1, 3], [0, 2, 4], [5]):
        S.assert_envelope(got[path], *ref.last([a, draft[path]]))
    S.assert_envelope(got[6:], *ref.last([b, tail]))
    lm.keep([2, 0], [6, 1], [[0, 2, 4], []])
    # the kept path, the dropped token and the fork each go on
    got = lm.step(up(np.concatenate([tail, tail, tail])), [2, 0, 1], [1, 1, 1]).cpu().numpy()
    S.assert_envelope(got[:1], *ref.last([a, draft[[0, 2, 4]], tail]))
    S.assert_envelope(got[1:2], *ref.last([b, tail]))
    S.assert_envelope(got[2:], *ref.last([a, tail]))
    lm.truncate([0, 1, 2], [0, 0, 0])
    assert lm.check() == 24
    lm.close()


def test_program(ctx):
    worst, again, free = PL.main()
    assert worst <= 1.5e-2 and again <= 1.5e-2 and free == 64


def test_refusals(ctx):
    with pytest.raises(ValueError):
        PL.tree([0])
    ref = Refs(O.TYPE_F16, 1)
    cfg = vb.LMConfig(H, NH, NKV, HD, F, LAYERS, 1e-5, 10000.0, 1, 0.0, O.TYPE_F16)
    lm = PL.PagedLM(ctx, cfg, ref.layers, seqs=1, pages=1, page_rows=16, most_rows=16)
    with pytest.raises(ValueError):
        lm.step(torch.zeros((2, H), device="cuda"), [0], [1])
    lm.step(torch.zeros((17, H), device="cuda"), [0], [17])   # more rows than the pool has
    with pytest.raises(vb.VBError):
        lm.check()
    lm.close()


def test_a_check_says_what_came_since_the_last(ctx):
    """A failed step, a check that raises, then a step that fits: the next check passes."""
    ref = Refs(O.TYPE_F16, 1)
    cfg = vb.LMConfig(H, NH, NKV, HD, F, LAYERS, 1e-5, 10000.0, 1, 0.0, O.TYPE_F16)
    lm = PL.PagedLM(ctx, cfg, ref.layers, ref.fn, seqs=2, pages=2, page_rows=16, most_rows=32)
    a, b = rows(20), rows(16)
    lm.step(torch.from_numpy(a).cuda(), [0], [20])
    lm.step(torch.from_numpy(b).cuda(), [1], [16])            # no page is left
    with pytest.raises(vb.VBError, match="pages: error 4 in request 0; device error"):
        lm.check()
    assert lm.check() == 0
    lm.truncate([0], [0])
    got = lm.step(torch.from_numpy(b).cuda(), [1], [16]).cpu().numpy()
    assert lm.check() == 1
    S.assert_envelope(got, *ref.last([b]))
    lm.close()
