"""Root-mean-square norm in front of an MoE block (dsca_rms_norm, include/dsca_b200_block.h).

add_rms_norm(x, weight, eps, residual, quant) adds the block's input to the residual stream,
normalises the sum and, on request, writes the normed rows in 8 bits as well: what a decoder layer
runs between its attention and its MoE block (Qwen2MoeDecoderLayer.post_attention_layernorm,
SwitchTransformersLayerFF.layer_norm).  MoEEngine.forward_normed runs it with the block behind it.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib as L

__all__ = ["RmsNormOutput", "add_rms_norm"]

_QUANT = {None: L.NORM_Q_NONE, "e4m3": L.NORM_Q_E4M3, "split": L.NORM_Q_SPLIT}
_DTYPES = {torch.bfloat16: L.BF16, torch.float32: L.F32}


class RmsNormOutput(NamedTuple):
    """y: the normed rows, shaped like x (None when not asked for); residual: the residual stream h
    (x itself without a residual); q, scale: the 8-bit rows [rows, ...] e4m3 and their fp32 scales
    [rows] (None without quant)."""
    y: torch.Tensor | None
    residual: torch.Tensor
    q: torch.Tensor | None
    scale: torch.Tensor | None


def _stride(t: torch.Tensor, name: str, d: int) -> int:
    """Distance of t's rows in elements: the leading dimensions must lie one stride apart."""
    if t.is_contiguous():
        return d
    if t.dim() > 2:
        try:
            t = t.view(-1, d)
        except RuntimeError:
            raise ValueError(f"{name}: the rows of {tuple(t.shape)} with strides {t.stride()} are not evenly "
                             "spaced (call contiguous())") from None
    if d > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    ld = t.stride(0) if t.dim() > 1 and t.shape[0] > 1 else d
    if ld < d:
        raise ValueError(f"{name}: rows overlap (stride {ld}, width {d})")
    return ld


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor | None = None,
                 quant: str | None = None, write_y: bool = True) -> RmsNormOutput:
    """h = x + residual (rounded to x's type), y = weight * h / sqrt(mean(h^2) + eps) over the last
    dimension, summed in fp32 and rounded once.

    x [..., d] bf16 or fp32 (rows may lie in a wider buffer), residual the same shape and type,
    weight [d] of x's type or fp32.  quant "e4m3": q [rows, d] with scale = max|y| / 448 a row, from
    the unrounded y (the row format of the fp8 expert weights); "split" (bf16, d % 8 == 0): q
    [rows, 2 * ceil(d / 128) * 128], the two-term rows of dsca_split_rows with scale = 1 / s, the layout in
    which the fp8-weight experts multiply tokens (MoEEngine takes y and splits it itself).  write_y=False leaves y out when only the 8-bit rows are
    wanted.  Runs on x's device, on its current stream.  Inference only: the results carry no
    gradient."""
    dtype, dev, shape = x.dtype, x.device, x.shape
    dt, q_mode = _DTYPES.get(dtype), _QUANT.get(quant)
    if dt is None:
        raise ValueError(f"unsupported dtype {dtype}")
    if q_mode is None:
        raise ValueError(f"quant must be None, 'e4m3' or 'split', not {quant!r}")
    if dev.type != "cuda":
        raise ValueError("x must be on a GPU")
    if not shape or shape[-1] == 0:
        raise ValueError(f"expected [..., d] rows, got {tuple(shape)}")
    d = shape[-1]
    w_dt = _DTYPES.get(weight.dtype)
    if weight.dim() != 1 or weight.shape[0] != d or (w_dt != dt and w_dt != L.F32) or weight.device != dev or not weight.is_contiguous():
        raise ValueError(f"weight must be a contiguous [{d}] tensor of x's type or float32 on x's device")
    if quant == "split" and (dt != L.BF16 or d % 8):
        raise ValueError("quant='split' takes bf16 rows with d % 8 == 0")
    if not write_y and quant is None:
        raise ValueError("write_y=False needs a quant")
    if d > L.NORM_MAX_D:
        raise ValueError(f"rows of {d} values exceed {L.NORM_MAX_D}")
    dense = x.is_contiguous()
    ld = d if dense else _stride(x, "x", d)
    rows = x.numel() // d
    if rows > 0x7FFFFFFF:
        raise ValueError(f"{rows} rows exceed 2^31 - 1")
    h, r_ptr, h_ptr, ld_r = x, None, None, 0
    if residual is not None:
        if residual.shape != shape or residual.dtype != dtype or residual.device != dev:
            raise ValueError("residual must have x's shape, type and device")
        ld_r = _stride(residual, "residual", d)
        h = torch.empty_like(x) if dense else x.new_empty(shape)
        r_ptr, h_ptr = residual.data_ptr(), h.data_ptr()
    y = q = scale = y_ptr = q_ptr = s_ptr = None
    if write_y:
        y = torch.empty_like(x) if dense else x.new_empty(shape)
        y_ptr = y.data_ptr()
    if quant is not None:
        width = d if quant == "e4m3" else 2 * ((d + 127) // 128 * 128)
        q = torch.empty_strided((rows, width), (width, 1), dtype=torch.float8_e4m3fn, device=dev)
        scale = torch.empty_strided((rows,), (1,), dtype=torch.float32, device=dev)
        q_ptr, s_ptr = q.data_ptr(), scale.data_ptr()
    if rows:
        a = L.RmsNormArgs(x.data_ptr(), r_ptr, weight.data_ptr(), rows, d, dt, w_dt, ld, ld_r, d, d, eps, q_mode, y_ptr,
                          h_ptr, q_ptr, s_ptr)
        L.call_on(dev, "dsca_rms_norm", ctypes.byref(a))
    return RmsNormOutput(y, h, q, scale)
