"""include/dsca_b200_block.h without a GPU: every symbol exported, every argument struct mirrored with the
C compiler's offsets, and the calls that both entry points and their Python callers refuse."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"dsca_rms_norm_args": "RmsNormArgs", "dsca_few_args": "FewArgs"}


def _header():
    return open(os.path.join(ROOT, "include", "dsca_b200_block.h")).read()


def test_symbols_and_constants(lib):
    from dsca_moe_b200 import _lib as L

    src = re.sub(r"/\*.*?\*/", " ", _header(), flags=re.S)
    assert set(re.findall(r"\b(dsca_[a-z0-9_]+)\s*\(", src)) == set(L.EXPORTED_BLOCK)
    for name in L.EXPORTED_BLOCK:
        assert hasattr(lib, name), name
    for c, v in (("DSCA_NORM_MAX_D", L.NORM_MAX_D), ("DSCA_FEW_TOKENS", L.FEW_TOKENS),
                 ("DSCA_FEW_ZERO_BYTES", L.FEW_ZERO_BYTES)):
        assert int(re.search(rf"#define {c} (\d+)", src).group(1)) == v
    assert set(re.findall(r"\}\s*(dsca_[a-z0-9_]+)\s*;", src)) == set(STRUCTS)


def test_struct_layouts(tmp_path):
    from dsca_moe_b200 import _lib as L

    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "dsca_b200_block.h"', "int main(void) {"]
    want = []
    for c, py in STRUCTS.items():
        cls = getattr(L, py)
        lines.append(f'  printf("%zu ", sizeof({c}));')
        want.append(ctypes.sizeof(cls))
        for f, _ in cls._fields_:
            lines.append(f'  printf("%zu ", offsetof({c}, {f}));')
            want.append(getattr(cls, f).offset)
    lines += ["  return 0;", "}"]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True)
    assert [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()] == want


def _norm_args():
    from dsca_moe_b200 import _lib as L

    a = L.RmsNormArgs()
    a.x = a.residual = a.weight = a.y = a.residual_out = 4096
    a.rows, a.d, a.eps = 4, 64, 1e-6
    a.dtype = a.weight_dtype = L.BF16
    a.ld_x = a.ld_residual = a.ld_y = a.ld_residual_out = 64
    return a


@pytest.mark.parametrize("change", [
    dict(x=None), dict(weight=None), dict(y=None), dict(d=0), dict(rows=-1), dict(dtype=2), dict(weight_dtype=2),
    dict(quant=3), dict(quant=1), dict(quant=2, q=4096), dict(eps=-1.0), dict(eps=float("nan")), dict(ld_x=63),
    dict(ld_residual=63), dict(ld_y=0), dict(ld_residual_out=8), dict(x=4097), dict(scale=4098, quant=1, q=4096),
    dict(quant=2, q=4096, scale=4096, dtype=0, weight_dtype=0), dict(quant=2, q=4096, scale=4096, d=63),
    dict(dtype=0, weight_dtype=1)])
def test_norm_bad_arguments(lib, change):
    from dsca_moe_b200 import _lib as L

    a = _norm_args()
    for k, v in change.items():
        setattr(a, k, v)
    assert lib.dsca_rms_norm(ctypes.byref(a), None) == L.ERR_BAD_ARG


def test_norm_limits(lib):
    from dsca_moe_b200 import _lib as L

    assert lib.dsca_rms_norm(None, None) == L.ERR_BAD_ARG
    a = _norm_args()
    a.d = a.ld_x = a.ld_residual = a.ld_y = a.ld_residual_out = L.NORM_MAX_D + 1
    assert lib.dsca_rms_norm(ctypes.byref(a), None) == L.ERR_CAPACITY
    a = _norm_args()
    a.rows, a.x = 0, None  # nothing to do
    assert lib.dsca_rms_norm(ctypes.byref(a), None) == L.OK


def _few_args():
    from dsca_moe_b200 import _lib as L

    a = L.FewArgs()
    for f in ("x", "w_router", "w_shared_gate", "w1", "w2", "ws1", "ws2", "out", "logits", "topk_ids", "topk_w",
              "workspace"):
        setattr(a, f, 4096)
    a.T, a.d, a.E, a.top_k = 4, 64, 8, 2
    a.weights, a.mode, a.act = L.BF16, L.ROUTE_SOFTMAX_TOPK, L.ACT_SWIGLU
    a.inter, a.n1p, a.ip, a.dp = 100, 256, 128, 256
    a.shared_inter, a.shared_n1p, a.shared_ip = 128, 256, 128
    a.workspace_bytes = 1 << 30
    return a


@pytest.mark.parametrize("change", [
    dict(x=None), dict(w1=None), dict(out=None), dict(logits=None), dict(topk_w=None), dict(workspace=None),
    dict(T=-1), dict(d=0), dict(d=60), dict(E=0), dict(top_k=0), dict(top_k=9), dict(E=1), dict(weights=3), dict(mode=2),
    dict(act=2), dict(inter=0), dict(inter=129), dict(n1p=255), dict(ip=256), dict(dp=32), dict(shared_inter=0),
    dict(shared_inter=129), dict(shared_ip=64), dict(ws1=None), dict(x=4104), dict(workspace=4112),
    dict(weights=2), dict(weights=2, w1_scale=4096, w2_scale=4096),
    dict(weights=2, w1_scale=4096, w2_scale=4096, ws1_scale=4096, ws2_scale=4096, w1_max=-1.0),
    dict(weights=2, w1_scale=4096, w2_scale=4096, ws1_scale=4096, ws2_scale=4096, w1_max=float("inf")), dict(weights=2, d=72)])
def test_few_bad_arguments(lib, change):
    from dsca_moe_b200 import _lib as L

    a = _few_args()
    for k, v in change.items():
        setattr(a, k, v)
    assert lib.dsca_moe_few(ctypes.byref(a), None) == L.ERR_BAD_ARG


def test_few_limits(lib):
    from dsca_moe_b200 import _lib as L

    assert lib.dsca_moe_few(None, None) == L.ERR_BAD_ARG
    for change in (dict(T=33), dict(E=64), dict(workspace_bytes=1000)):
        a = _few_args()
        for k, v in change.items():
            setattr(a, k, v)
        assert lib.dsca_moe_few(ctypes.byref(a), None) == L.ERR_CAPACITY
    a = _few_args()
    a.T, a.x = 0, None
    assert lib.dsca_moe_few(ctypes.byref(a), None) == L.OK
    assert lib.dsca_few_workspace_bytes(33, 64, 4, 64, 0) == 0 and lib.dsca_few_workspace_bytes(4, 64, 9, 64, 0) == 0
    n = lib.dsca_few_workspace_bytes(32, 2048, 4, 1408, 5632)
    assert n >= 1024 + 4 * 32 * (4 * 1408 + 5632) and n % 256 == 0


def test_norm_python_refusals(lib):
    from dsca_moe_b200 import add_rms_norm

    w = torch.ones(64, dtype=torch.bfloat16)
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        add_rms_norm(x, w)
    with pytest.raises(ValueError, match="dtype"):
        add_rms_norm(x.half(), w.half())
    with pytest.raises(ValueError, match="quant"):
        add_rms_norm(x, w, quant="int8")
