"""include/dsca_b200_dense.h and its Python callers without a GPU: exported symbols, struct layouts, refusals, and
the 64-bit definitions that the GPU tests compare with."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

import dense_ref as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"dsca_gated_ffn_args": "GatedFfnArgs", "dsca_gated_ffn_backward_args": "GatedFfnBackwardArgs",
           "dsca_quantize_rows_args": "QuantizeRowsArgs", "dsca_int8_linear_args": "Int8LinearArgs",
           "dsca_gated_ffn_int8_args": "GatedFfnInt8Args"}


def _header():
    return open(os.path.join(ROOT, "include", "dsca_b200_dense.h")).read()


def test_symbols_and_constants(lib):
    from dsca_moe_b200 import _lib as L

    src = re.sub(r"/\*.*?\*/", " ", _header(), flags=re.S)
    assert set(re.findall(r"\b(dsca_[a-z0-9_]+)\s*\(", src)) == set(L.EXPORTED_DENSE)
    for name in L.EXPORTED_DENSE:
        assert hasattr(lib, name), name
    for c, v in (("DSCA_DENSE_MAX_DIM", L.DENSE_MAX_DIM), ("DSCA_DENSE_MAX_ROWS", L.DENSE_MAX_ROWS),
                 ("DSCA_DENSE_FEW_TOKENS", L.DENSE_FEW_TOKENS), ("DSCA_DENSE_FEW_BYTES", L.DENSE_FEW_BYTES)):
        assert int(re.search(rf"#define {c} (\d+)", src).group(1)) == v
    assert set(re.findall(r"\}\s*(dsca_[a-z0-9_]+)\s*;", src)) == set(STRUCTS)


def test_struct_layouts(tmp_path):
    from dsca_moe_b200 import _lib as L

    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "dsca_b200_dense.h"', "int main(void) {"]
    want = []
    for c, py in STRUCTS.items():
        cls = getattr(L, py)
        lines.append(f'  printf("%zu ", sizeof({c}));')
        want.append(ctypes.sizeof(cls))
        for f, _ in cls._fields_:
            lines.append(f'  printf("%zu ", offsetof({c}, {f}));')
            want.append(getattr(cls, f).offset)
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True)
    assert [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()] == want


def _args(name):
    """Valid arguments of each entry point (addresses are never read: every test refuses the call)."""
    from dsca_moe_b200 import _lib as L

    a = getattr(L, STRUCTS[name + "_args"])()
    for f, t in a._fields_:
        if t is ctypes.c_void_p:
            setattr(a, f, 4096)
        elif f.startswith("ld_"):
            setattr(a, f, 128)
    a.rows, a.dtype = 4, L.BF16
    for f, v in dict(d=64, inter=96, k=64, n=48).items():
        if hasattr(a, f):
            setattr(a, f, v)
    if hasattr(a, "workspace_bytes"):
        a.workspace_bytes = 1 << 40
    return a


_COMMON = [dict(rows=-1), dict(dtype=2), dict(dtype=-1)]
_BAD = {
    "dsca_gated_ffn": _COMMON + [dict(x=None), dict(w_gate=None), dict(w_up=None), dict(w_down=None), dict(y=None),
                                 dict(h=None), dict(g=None), dict(u=None), dict(gu_exp=None), dict(h=4104), dict(x=4097), dict(d=0), dict(inter=0),
                                 dict(act=3), dict(ld_x=63), dict(ld_gate=63), dict(ld_up=0), dict(ld_down=95), dict(ld_y=1),
                                 dict(ld_h=95), dict(ld_h=97), dict(d=1 << 21), dict(ld_x=1 << 41)],
    "dsca_gated_ffn_backward": _COMMON + [dict(x=None), dict(dy=None), dict(g=None), dict(u=None), dict(gu_exp=None), dict(h=None), dict(dg=None),
                                          dict(du=None), dict(dx=4097), dict(d_gate=4097), dict(d=0), dict(inter=-2), dict(act=-1),
                                          dict(ld_dy=63), dict(ld_down=95), dict(ld_h=100)],
    "dsca_quantize_rows": _COMMON + [dict(x=None), dict(q=None), dict(scale=None), dict(q=4104), dict(scale=4098), dict(k=0),
                                     dict(ld_x=63), dict(ld_q=63), dict(ld_q=72), dict(x=4097)],
    "dsca_int8_linear": _COMMON + [dict(q=None), dict(scale=None), dict(w=None), dict(w_scale=None), dict(y=None), dict(w=4104),
                                   dict(q=4104), dict(k=0), dict(n=0), dict(ld_x=63), dict(ld_q=63), dict(ld_q=72), dict(ld_w=63),
                                   dict(ld_w=72), dict(ld_y=47), dict(bias=4097)],
    "dsca_gated_ffn_int8": _COMMON + [dict(x=None), dict(q=None), dict(scale=None), dict(w_gate=None), dict(w_up=None),
                                      dict(w_down=None), dict(gate_scale=None), dict(up_scale=None), dict(down_scale=None),
                                      dict(h=None), dict(hq=None), dict(h_scale=None), dict(y=None), dict(h=4100), dict(act=7),
                                      dict(ld_q=48), dict(ld_gate=72), dict(ld_down=80), dict(ld_h=98), dict(ld_hq=100),
                                      dict(ld_y=63), dict(w_up=4104)],
}


@pytest.mark.parametrize("name,change", [(n, c) for n, cs in _BAD.items() for c in cs])
def test_bad_arguments(lib, name, change):
    from dsca_moe_b200 import _lib as L

    a = _args(name)
    for k, v in change.items():
        setattr(a, k, v)
    assert getattr(lib, name)(ctypes.byref(a), None) == L.ERR_BAD_ARG
    if name != "dsca_quantize_rows":
        assert getattr(lib, name + "_workspace")(ctypes.byref(a)) == 0


@pytest.mark.parametrize("name", list(_BAD))
def test_limits_and_nothing_to_do(lib, name):
    from dsca_moe_b200 import _lib as L

    assert getattr(lib, name)(None, None) == L.ERR_BAD_ARG
    a = _args(name)
    a.rows = L.DENSE_MAX_ROWS + 1
    assert getattr(lib, name)(ctypes.byref(a), None) == L.ERR_CAPACITY
    if name in ("dsca_int8_linear", "dsca_gated_ffn_int8"):
        a = _args(name)
        setattr(a, "k" if name == "dsca_int8_linear" else "inter", 131073)
        assert getattr(lib, name)(ctypes.byref(a), None) == L.ERR_CAPACITY
    a = _args(name)
    a.rows, a.x = 0, None
    for f in ("d_gate", "d_up", "d_down"):
        if hasattr(a, f):
            setattr(a, f, None)
    assert getattr(lib, name)(ctypes.byref(a), None) == L.OK


def test_python_refusals(lib):
    from dsca_moe_b200 import (Int8Weight, gated_ffn, gated_ffn_int8, int8_linear, pack_int8, patch, quantize_rows)

    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    w = torch.zeros(96, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        gated_ffn(x, w, w, w.T.contiguous())
    with pytest.raises(ValueError, match="act"):
        gated_ffn(x, w, w, w.T.contiguous(), act="tanh")
    with pytest.raises(ValueError, match="dtype"):
        gated_ffn(x.half(), w, w, w.T.contiguous())
    q = Int8Weight(torch.zeros(96, 64, dtype=torch.int8), torch.ones(96))
    with pytest.raises(ValueError, match="GPU"):
        int8_linear(x, q)
    with pytest.raises(ValueError, match="x_scale"):
        int8_linear(x, q, x_scale=torch.ones(4))
    with pytest.raises(ValueError, match="x_scale"):
        int8_linear(x.to(torch.int8), q)
    with pytest.raises(ValueError, match="out_dtype"):
        int8_linear(x, q, out_dtype=torch.float32)
    with pytest.raises(ValueError, match="GPU"):
        gated_ffn_int8(x, q, q, q)
    with pytest.raises(ValueError, match="dtype"):
        quantize_rows(x.half())
    with pytest.raises(ValueError, match="GPU"):
        quantize_rows(x)
    with pytest.raises(ValueError, match="out, in"):
        pack_int8(x[0])
    with pytest.raises(ValueError, match="dense_ffn"):
        patch(None, 0, 1, dense_ffn="fp8")


def test_gated_module_refusals():
    from dsca_moe_b200 import GatedFFN

    class M(torch.nn.Module):
        def __init__(self, act, bias=False, up=True):
            super().__init__()
            self.gate_proj = torch.nn.Linear(8, 16, bias=bias)
            if up:
                self.up_proj = torch.nn.Linear(8, 16, bias=bias)
            self.down_proj = torch.nn.Linear(16, 8, bias=bias)
            self.act_fn = act

    with pytest.raises(ValueError, match="biases"):
        GatedFFN(M(torch.nn.SiLU(), bias=True))
    with pytest.raises(ValueError, match="neither"):
        GatedFFN(M(torch.nn.SiLU(), up=False))
    with pytest.raises(ValueError, match="not offered"):
        GatedFFN(M(torch.nn.GELU()))
    for act, name in ((torch.nn.SiLU(), "silu"), (torch.nn.ReLU(), "relu"), (torch.nn.GELU(approximate="tanh"), "gelu")):
        old = M(act)
        new = GatedFFN(old)
        assert new.act == name and new.state_dict().keys() == old.state_dict().keys()
        assert new.gate_proj.weight is old.gate_proj.weight


@pytest.mark.parametrize("act", R.ACTS)
def test_reference_gradients(act):
    """dense_ref's formulas against autograd and against differences."""
    g = torch.Generator().manual_seed(3)
    x, wg, wu, dy = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((5, 7), (9, 7), (9, 7), (5, 7)))
    wd = torch.randn(7, 9, generator=g, dtype=torch.float64)
    ref = R.ffn(x, wg, wu, wd, act, torch.float32, dy)
    p = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    fn = {"silu": torch.nn.functional.silu, "relu": torch.relu,
          "gelu": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[act]
    y = (fn(p[0] @ p[1].T) * (p[0] @ p[2].T)) @ p[3].T
    assert torch.allclose(y, ref["y"][0], rtol=1e-12, atol=1e-12)
    for got, name in zip(torch.autograd.grad(y, p, dy), ("dx", "d_gate", "d_up", "d_down")):
        assert torch.allclose(got, ref[name][0], rtol=1e-10, atol=1e-12), name
    step = 1e-6
    for i, name in enumerate(("dx", "d_gate", "d_up", "d_down")):
        args = [x, wg, wu, wd]
        v = torch.randn(args[i].shape, generator=g, dtype=torch.float64)
        lo, hi = list(args), list(args)
        lo[i], hi[i] = args[i] - step * v, args[i] + step * v
        diff = ((R.ffn(*hi, act, torch.float32)["y"][0] - R.ffn(*lo, act, torch.float32)["y"][0]) * dy).sum() / (2 * step)
        assert abs(float(diff - (ref[name][0] * v).sum())) <= 1e-6 * (1 + abs(float(diff)))


def test_reference_codes():
    v = torch.tensor([[1.0, 0.5, -0.5, 0.0], [0, 0, 0, 0], [254.0, 1.0, 3.0, -5.0]], dtype=torch.float64)
    q, s = R.codes(v)
    assert q.tolist() == [[127, 64, -64, 0], [0, 0, 0, 0], [127, 0, 2, -2]]
    assert s.tolist() == [1 / 127, 1.0, 2.0]
