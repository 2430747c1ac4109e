"""CPU checks of the paged-cache part of the C ABI: the argument records match
the header's layout, null arguments are refused without a device, and the
rotation table is the one that the oracle rotates with."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest

import oracle as O
import paged_model as M
import vcpm_b200 as vb

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("name,record", [("vb_pages", vb.PagesC), ("vb_qk_args", vb.QKArgsC), ("vb_tree_args", vb.TreeArgsC)])
def test_records_match_the_header(tmp_path, name, record):
    src = tmp_path / "layout.c"
    fields = "".join(f'printf("%s %zu\\n", "{f}", offsetof({name}, {f}));' for f, _ in record._fields_)
    src.write_text('#include <stdio.h>\n#include "vcpm_b200.h"\nint main(void) { printf("size %zu\\n", sizeof(' + name + "));" + fields +
                   " return 0; }\n")
    exe = tmp_path / "layout"
    subprocess.check_call(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    want = dict(line.split() for line in subprocess.check_output([str(exe)], text=True).splitlines())
    assert int(want.pop("size")) == C.sizeof(record)
    assert {f: int(o) for f, o in want.items()} == {f: getattr(record, f).offset for f, _ in record._fields_}


def test_null_arguments_are_refused_without_a_device():
    L = vb.lib()
    assert L.vb_pages_init(None, None) == vb.VB_ERR_INVALID_ARG
    assert L.vb_pages_extend(None, None, 0, None, None) == vb.VB_ERR_INVALID_ARG
    assert L.vb_pages_fork(None, None, 0, None, None) == vb.VB_ERR_INVALID_ARG
    assert L.vb_pages_keep(None, None, 0, None, None, None, None, 0) == vb.VB_ERR_INVALID_ARG
    assert L.vb_pages_truncate(None, None, 0, None, None) == vb.VB_ERR_INVALID_ARG
    assert L.vb_pages_compact(None, None, None) == vb.VB_ERR_INVALID_ARG
    assert L.vb_pages_status(None, None, None, None, None) == vb.VB_ERR_INVALID_ARG
    assert L.vb_qk_norm_rope(None, None) == vb.VB_ERR_INVALID_ARG
    assert L.vb_tree_attention(None, None) == vb.VB_ERR_INVALID_ARG


@pytest.mark.parametrize("args", [(0, 1e4, 0, 4), (63, 1e4, 0, 4), (64, 1e4, 1, 4), (64, -1.0, 0, 4), (64, 1e4, 0, -1)])
def test_rope_table_refusals(args):
    out = np.zeros(1024, np.float32)
    assert vb.lib().vb_rope_table(*args, out.ctypes.data) == vb.VB_ERR_INVALID_ARG
    assert vb.lib().vb_rope_table(64, 1e4, 0, 4, None) == vb.VB_ERR_INVALID_ARG


@pytest.mark.parametrize("hd,longrope", [(64, False), (128, True)])
def test_rope_table_is_the_oracles(hd, longrope):
    table = vb.rope_table(hd, 10000.0, longrope, 512)
    factors = O.longrope_short_factors() if longrope else None
    for pos in (0, 1, 2, 5, 63, 64, 200, 511):
        assert np.array_equal(table[pos], O.rope_cache(pos, hd, 10000.0, factors))


def test_pool_model_shares_and_copies():
    m = M.PoolModel(np.arange(2 * 2 * 4 * 1 * 16 * 8).reshape(2, 2, 4, 1, 16, 8), 3, 2)
    m.extend([0], [20])
    m.fork([0], [1])
    assert m.refs.tolist() == [2, 2, 0, 0]
    m.extend([1], [1])
    assert m.refs.tolist() == [2, 1, 1, 0] and np.array_equal(m.data[:, :, 2, :, :4], m.data[:, :, 1, :, :4])
    m.truncate([0], [0])
    assert m.refs.tolist() == [1, 0, 1, 0]


def test_broadcast_rows_are_refused():
    """A row stride of 0 means packed rows to the library: a broadcast tensor would be read past its end."""
    torch = pytest.importorskip("torch")
    for t in (torch.zeros(1, 16).expand(3, 16), torch.zeros(64).as_strided((3, 16), (8, 1))):
        with pytest.raises(ValueError, match="rows of their own"):
            vb._rows(t, 16, "q")
    for t, ld in ((torch.zeros(3, 20)[:, :16], 20), (torch.zeros(1, 16).expand(1, 16), 16), (torch.zeros(3, 16), 16)):
        assert vb._rows(t, 16, "q") == (t.data_ptr(), ld)


def test_host_tensors_are_refused():
    """Their addresses would fault on the device."""
    torch = pytest.importorskip("torch")
    new = lambda *s, dtype=torch.int32: torch.zeros(s, dtype=dtype)  # noqa: E731
    q, k = new(3, 16, dtype=torch.float32), new(3, 8, dtype=torch.float32)
    with pytest.raises(ValueError, match="CUDA"):
        vb.Pages(new(1, 2, 1, 16, 8, dtype=torch.bfloat16), new(1, 2, 1, 16, 8, dtype=torch.bfloat16), new(1, 2), new(1), new(2), new(4))
    with pytest.raises(ValueError, match="CUDA"):
        vb.QKArgs(q, k, k, heads=2, kv_heads=1, head_dim=8, q_out=q)
    with pytest.raises(ValueError, match="CUDA"):
        vb._count(new(2), new(2))
    with pytest.raises(ValueError, match="pos"):
        vb.QKArgs(q, k, k, heads=2, kv_heads=1, head_dim=8, q_out=q, rope=new(4, 8, dtype=torch.float32))


def test_the_cubic_of_the_powers():
    """2^f on [-1/2, 1/2] by the polynomial of the tcgen05 attention kernel: its stated relative error holds."""
    src = open(os.path.join(ROOT, "voxcpm-cpp_b200", "csrc", "vb_tree_tc.cu")).read()
    body = src[src.index("void exp2_pair"):]
    coef = [float(x) for x in re.findall(r"pack_f32x2\((0\.\d+)f, \1f\)", body[:body.index("\n}\n")])]
    assert len(coef) == 4                                         # cubic first
    f = np.linspace(-0.5, 0.5, 200001)
    assert np.max(np.abs(np.polyval(coef, f) / np.exp2(f) - 1)) < 7.6e-5
