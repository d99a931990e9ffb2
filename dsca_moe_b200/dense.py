"""Dense gated feed-forward blocks and 8-bit integer products (include/dsca_b200_dense.h).

The dense layers between MoE blocks (Qwen2MoeMLP of `mlp_only_layers` and `decoder_sparse_step`, or a
shared expert on its own) are y = (act(x Wg^T) * (x Wu^T)) Wd^T:

  gated_ffn        the block in bf16 or fp32 on weights as Linear layers hold them, with its gradients
  gated_ffn_int8   the block on 8-bit integer weights (inference)
  int8_linear      one product with 8-bit integer weights, scales for each token and channel
  quantize_rows, pack_int8   rows and weights in 8-bit integers
  GatedFFN         the module that replace_dense_ffn and patch(dense_ffn=...) put into a model
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib as L
from .gradients import refuse_tangents, without_gradient
from .norm import _DTYPES, _stride

__all__ = ["GatedFFN", "Int8Weight", "check_dense", "gated_ffn", "gated_ffn_int8", "int8_linear", "pack_int8",
           "quantize_rows"]

_ACTS = {"silu": L.GATE_SILU, "gelu": L.GATE_GELU, "relu": L.GATE_RELU}
_ERR: dict = {}
_BF16 = torch.bfloat16


def _err(dev):
    """Address of the device's error word (a wait inside a kernel that ran out records there); None for calls captured
    before the first other call, whose graph's memory must not hold it."""
    e = _ERR.get(dev.index)
    if e is None:
        if torch.cuda.is_current_stream_capturing():
            return None
        t = torch.zeros(64, dtype=torch.int32, device=dev)
        torch.cuda.current_stream(dev).synchronize()  # once: a call on another stream may record before this one's zeros land
        e = _ERR[dev.index] = (t.data_ptr(), t)
    return e[0]


def check_dense(device=None):
    """Raise if a dense block or 8-bit product on `device` recorded an error since the last check, which
    it clears (synchronises the current stream)."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    e = _ERR.get(dev.index if dev.index is not None else torch.cuda.current_device())
    if e is not None:
        L.call_on(e[1].device, "dsca_check_error", e[0])


def _act(act: str) -> int:
    code = _ACTS.get(act)
    if code is None:
        raise ValueError(f"act must be 'silu', 'gelu' (tanh form) or 'relu', not {act!r}")
    return code


def _rows(x, name: str, width: int | None = None):
    """(rows, row stride) of x [..., width] on a GPU."""
    if not x.is_cuda:
        raise ValueError(f"{name} must be on a GPU")
    shape = x.shape
    if not shape or shape[-1] == 0 or (width is not None and shape[-1] != width):
        raise ValueError(f"{name}: expected [..., {'d' if width is None else width}] rows, got {tuple(shape)}")
    d = shape[-1]
    if d > L.DENSE_MAX_DIM:
        raise ValueError(f"{name}: rows of {d} values exceed {L.DENSE_MAX_DIM}")
    rows = x.numel() // d
    if rows > L.DENSE_MAX_ROWS:
        raise ValueError(f"{name}: {rows} rows exceed {L.DENSE_MAX_ROWS}")
    return rows, (d if x.is_contiguous() or rows == 0 else _stride(x, name, d))


def _weight(w, name: str, out: int, inp: int, x, dtype, index: int) -> int:
    """Row stride of a weight [out, inp] of x's type on x's device."""
    if w.is_contiguous() and w.shape == (out, inp) and w.dtype is dtype and w.get_device() == index:
        return inp
    if w.dim() != 2 or w.shape[0] != out or w.shape[1] != inp:
        raise ValueError(f"{name}: expected [{out}, {inp}], got {tuple(w.shape)}")
    if w.dtype != x.dtype or w.device != x.device:
        raise ValueError(f"{name} must have x's type and device")
    return inp if w.is_contiguous() else _stride(w, name, inp)


def _workspace(name: str, args, dev):
    """The call's workspace, allocated on the current stream, in args."""
    fn = getattr(L._LIB or L.load(), name)
    if dev.index == torch._C._cuda_getDevice():
        n = fn(ctypes.byref(args))
    else:
        with torch.cuda.device(dev):
            n = fn(ctypes.byref(args))
    if n == 0:
        return None
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    args.workspace, args.workspace_bytes = ws.data_ptr(), n
    return ws


def _forward(x, wg, wu, wd, act: int, shapes, save: bool):
    """(y, the buffer with h and, with `save`, g and u)."""
    dev, dtype = x.device, x.dtype
    rows, d, inter, ld_x, ld_g, ld_u, ld_d = shapes
    y = torch.empty(x.shape, dtype=dtype, device=dev)
    if rows == 0:
        return y, None
    ld_h, step, size = _saved(rows, inter, dtype)
    buf = torch.empty(size if save else step, dtype=torch.uint8, device=dev)
    h = buf.data_ptr()
    g, u, e = (h + step, h + 2 * step, h + 3 * step) if save else (None, None, None)
    a = L.GatedFfnArgs(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), y.data_ptr(), g, u, e, h, rows, d, inter,
                       _DTYPES[dtype], act, ld_x, ld_g, ld_u, ld_d, d, ld_h, None, 0, _err(dev))
    if rows > L.DENSE_FEW_TOKENS:  # others need none
        ws = _workspace("dsca_gated_ffn_workspace", a, dev)  # noqa: F841 - alive until the launch
    L.call_on(dev, "dsca_gated_ffn", ctypes.byref(a))
    return y, buf


def _saved(rows: int, inter: int, dtype):
    """(row stride, bytes of each of h, g and u, bytes in all with g's and u's exponents): rows on 32-byte sectors; g and u
    take what h takes (fp16 codes beside bf16, fp32 beside fp32)."""
    ld_h = (inter + 15) // 16 * 16
    step = rows * ld_h * (2 if dtype is _BF16 else 4)
    return ld_h, step, 3 * step + (8 * rows * ((inter + 31) // 32) if dtype is _BF16 else 0)


def _as_saved(t, name: str, shape, dtype, index: int):
    """(t, its row stride) of a tensor that the backward pass reads.  Saved-tensor hooks (offloading, for one) may return it
    in other strides than it was saved with, and a gradient comes in any (expanded, transposed)."""
    if t.shape != shape or t.dtype is not dtype or t.get_device() != index:
        raise RuntimeError(f"{name} came back as {t.dtype} {tuple(t.shape)} on {t.device}, not {dtype} {tuple(shape)} on GPU {index}")
    try:
        return t, _stride(t, name, shape[-1])
    except ValueError:
        return t.contiguous(), shape[-1]


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, wd, act, shapes):
        y, buf = _forward(x, wg, wu, wd, act, shapes, True)
        ctx.act, ctx.sizes, ctx.x_shape = act, shapes[:3], x.shape
        ctx.save_for_backward(x, wg, wu, wd, buf)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, wg, wu, wd, buf = ctx.saved_tensors
        rows, d, inter = ctx.sizes
        dev, dtype = dy.device, dy.dtype
        need = ctx.needs_input_grad
        dx = torch.empty(ctx.x_shape, dtype=dtype, device=dev) if need[0] else None
        dwg = torch.empty((inter, d), dtype=dtype, device=dev) if need[1] else None
        dwu = torch.empty((inter, d), dtype=dtype, device=dev) if need[2] else None
        dwd = torch.empty((d, inter), dtype=dtype, device=dev) if need[3] else None
        dx_p, dwg_p, dwu_p, dwd_p = [None if t is None else t.data_ptr() for t in (dx, dwg, dwu, dwd)]
        if rows:
            i, x_shape = dy.get_device(), ctx.x_shape
            ld_dy = d
            if not dy.is_contiguous():
                dy, ld_dy = _as_saved(dy, "dy", x_shape, dtype, i)
            # the usual case first: as they were saved
            ld_x = ld_g = ld_u = d
            ld_d, up = inter, (inter, d)
            if not (x.is_contiguous() and x.shape == x_shape and x.dtype is dtype and x.get_device() == i):
                x, ld_x = _as_saved(x, "x", x_shape, dtype, i)
            if not (wg.is_contiguous() and wg.shape == up and wg.dtype is dtype and wg.get_device() == i):
                wg, ld_g = _as_saved(wg, "w_gate", up, dtype, i)
            if not (wu.is_contiguous() and wu.shape == up and wu.dtype is dtype and wu.get_device() == i):
                wu, ld_u = _as_saved(wu, "w_up", up, dtype, i)
            if not (wd.is_contiguous() and wd.shape == (d, inter) and wd.dtype is dtype and wd.get_device() == i):
                wd, ld_d = _as_saved(wd, "w_down", (d, inter), dtype, i)
            ld_h, step, size = _saved(rows, inter, dtype)
            grads = torch.empty(2 * step, dtype=torch.uint8, device=dev)
            h, dg = buf.data_ptr(), grads.data_ptr()
            if buf.dtype is not torch.uint8 or buf.get_device() != i or buf.numel() != size or not buf.is_contiguous() or h % 16:
                raise RuntimeError("the saved intermediates came back otherwise than they were saved")
            a = L.GatedFfnBackwardArgs(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), dy.data_ptr(), h + step,
                                       h + 2 * step, h + 3 * step, h, dx_p, dwg_p, dwu_p, dwd_p, dg, dg + step, rows, d,
                                       inter, _DTYPES[dtype], ctx.act, ld_x, ld_g, ld_u, ld_d, ld_dy, ld_h, None, 0,
                                       _err(dev))
            ws = _workspace("dsca_gated_ffn_backward_workspace", a, dev)  # noqa: F841 - alive until the launch
        else:
            a = L.GatedFfnBackwardArgs()
            a.dx, a.d_gate, a.d_up, a.d_down = dx_p, dwg_p, dwu_p, dwd_p
            a.d, a.inter, a.dtype, a.act = d, inter, _DTYPES[dtype], ctx.act
        L.call_on(dev, "dsca_gated_ffn_backward", ctypes.byref(a))
        return dx, dwg, dwu, dwd, None, None


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
              act: str = "silu") -> torch.Tensor:
    """y = (act(x w_gate^T) * (x w_up^T)) w_down^T, with gradients for x and the three weights.

    x [..., d] bf16 or fp32 (rows may lie in a wider buffer), w_gate and w_up [inter, d], w_down
    [d, inter] of x's type, as Linear layers hold them.  act: "silu", "gelu" (tanh form) or "relu".
    Products are summed in fp32; the gated intermediate is rounded to x's type, and so are its two
    gradients in the backward pass.  Under autograd the call keeps the intermediate, the gate and the up
    values, each [rows, inter] (the latter two to 11 bits for bf16), for the backward pass; second derivatives and forward-mode
    ones are not offered.  Autocast does not apply (GatedFFN follows it).  Runs on x's device, on its current stream; check_dense() reports a wait that ran out."""
    code, dtype = _act(act), x.dtype
    if dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {dtype}")
    rows, ld_x = _rows(x, "x")
    d, i = x.shape[-1], x.get_device()
    if w_gate.dim() != 2 or w_gate.shape[0] == 0:
        raise ValueError(f"w_gate: expected [inter, {d}], got {tuple(w_gate.shape)}")
    inter = w_gate.shape[0]
    if inter > L.DENSE_MAX_DIM:
        raise ValueError(f"w_gate: {inter} rows exceed {L.DENSE_MAX_DIM}")
    shapes = (rows, d, inter, ld_x, _weight(w_gate, "w_gate", inter, d, x, dtype, i),
              _weight(w_up, "w_up", inter, d, x, dtype, i), _weight(w_down, "w_down", d, inter, x, dtype, i))
    refuse_tangents("gated_ffn", x, w_gate, w_up, w_down)
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad
                                    or w_down.requires_grad):
        return _GatedFFN.apply(x, w_gate, w_up, w_down, code, shapes)
    return _forward(x, w_gate, w_up, w_down, code, shapes, False)[0]


# ----------------------------------------------------------------------------- 8-bit integers
class Int8Weight(NamedTuple):
    """q [out, in] int8 codes (a view of rows padded with zeros to a multiple of 16), scale [out] fp32:
    the weight is q * scale[:, None]."""
    q: torch.Tensor
    scale: torch.Tensor

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        return (self.q.float() * self.scale[:, None]).to(dtype)


def _quantize(x):
    """(codes [rows, k rounded up to 16], scales) of x's rows."""
    refuse_tangents("quantize_rows", x)
    dt = _DTYPES.get(x.dtype)
    if dt is None:
        raise ValueError(f"unsupported dtype {x.dtype}")
    rows, ld_x = _rows(x, "x")
    k = x.shape[-1]
    ld_q = (k + 15) // 16 * 16
    q = torch.empty((rows, ld_q), dtype=torch.int8, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    if rows:
        a = L.QuantizeRowsArgs(x.data_ptr(), rows, k, dt, ld_x, q.data_ptr(), ld_q, scale.data_ptr())
        L.call_on(x.device, "dsca_quantize_rows", ctypes.byref(a))
    return q, without_gradient("quantize_rows", scale, x)


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(q [..., k] int8, scale [...] fp32) of x [..., k] bf16 or fp32: scale = max|x| / 127 a row (1 for a
    row of zeros), q the quotient 127 x / max|x| rounded to the nearest integer, ties to even,
    exactly.  q's rows lie a multiple of 16 bytes apart, the bytes between them zero.  A row with an
    infinity or a NaN has that as its scale.  Inference only: a backward pass that reaches the scale raises."""
    q, scale = _quantize(x)
    k = x.shape[-1]
    return q[:, :k] if x.dim() == 2 else q[:, :k].unflatten(0, x.shape[:-1]) if x.dim() > 2 else q[0, :k], scale


def pack_int8(weight: torch.Tensor) -> Int8Weight:
    """A Linear layer's weight [out, in] (bf16 or fp32, on a GPU) in 8-bit integers, one scale an output
    channel."""
    if weight.dim() != 2 or weight.shape[0] == 0:
        raise ValueError(f"weight: expected [out, in], got {tuple(weight.shape)}")
    return Int8Weight(*quantize_rows(weight.detach()))


def _int8_weight(w, name: str, dev, inp: int, out: int | None = None) -> int:
    """Row stride of an Int8Weight."""
    q, s = w
    shape = q.shape
    index = dev.index
    if q.dtype is torch.int8 and len(shape) == 2 and shape[1] == inp and (out is None or shape[0] == out) \
            and q.get_device() == index and s.get_device() == index and s.dtype is torch.float32 and s.shape == shape[:1] \
            and s.is_contiguous() and shape[0] > 1:
        ld, last = q.stride()
        if (last == 1 or inp == 1) and ld >= inp and ld % 16 == 0 and q.data_ptr() % 16 == 0:
            return ld
    if q.dtype != torch.int8 or q.dim() != 2 or q.shape[1] != inp or (out is not None and q.shape[0] != out):
        raise ValueError(f"{name}: expected an Int8Weight [{'out' if out is None else out}, {inp}], got "
                         f"{q.dtype} {tuple(q.shape)}")
    if q.device != dev or s.device != dev:
        raise ValueError(f"{name} must be on x's device")
    if s.dtype != torch.float32 or s.shape != (q.shape[0],) or not s.is_contiguous():
        raise ValueError(f"{name}: scale must be a contiguous float32 [{q.shape[0]}] tensor")
    ld = q.stride(0)
    if (inp > 1 and q.stride(1) != 1) or ld % 16 or ld < inp or q.data_ptr() % 16:
        raise ValueError(f"{name}: rows of codes must lie a multiple of 16 bytes apart (pack_int8 lays them out)")
    return ld


_INT8_MAX_K = 131072


def int8_linear(x: torch.Tensor, weight: Int8Weight, bias: torch.Tensor | None = None,
                x_scale: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y = x W^T (+ bias) with W in 8-bit integers (pack_int8) and x's rows quantised in the call.

    x [..., k] bf16 or fp32; or int8 codes of quantize_rows with their x_scale [...], out_dtype then
    chooses y's type (bf16 by default, otherwise x's type).  Codes lie in [-127, 127].  The products' sum
    is exact; its conversion to fp32, the products with the two scales and the addition of the bias round to
    fp32, the result to y's type.  bias [n] of y's type.  Inference only: a backward pass
    that reaches y raises."""
    refuse_tangents("int8_linear", x, bias, x_scale)
    given = x.dtype == torch.int8
    if given:
        if x_scale is None:
            raise ValueError("int8 codes need x_scale")
        dtype = torch.bfloat16 if out_dtype is None else out_dtype
    else:
        if x_scale is not None:
            raise ValueError("x_scale goes with int8 codes")
        dtype = x.dtype
        if out_dtype not in (None, dtype):
            raise ValueError("out_dtype goes with int8 codes (y has x's type otherwise)")
    dt = _DTYPES.get(dtype)
    if dt is None:
        raise ValueError(f"unsupported dtype {dtype}")
    rows, ld_x = _rows(x, "x")
    k, dev = x.shape[-1], x.device
    if k > _INT8_MAX_K:
        raise ValueError(f"sums of {k} products exceed {_INT8_MAX_K}")
    ld_w = _int8_weight(weight, "weight", dev, k)
    n = weight[0].shape[0]
    if bias is not None and (bias.dtype != dtype or bias.device != dev or tuple(bias.shape) != (n,)
                             or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous [{n}] tensor of y's type on x's device")
    if given:
        if x_scale.shape != x.shape[:-1] or x_scale.dtype != torch.float32 or x_scale.device != dev \
                or not x_scale.is_contiguous():
            raise ValueError("x_scale must be a contiguous float32 tensor, one value a row of x")
        if rows == 1:
            ld_x = (k + 15) // 16 * 16
        if rows and (ld_x % 16 or x.data_ptr() % 16):
            raise ValueError("rows of codes must lie a multiple of 16 bytes apart (quantize_rows lays them out)")
    y = torch.empty(x.shape[:-1] + (n,), dtype=dtype, device=dev)
    if rows == 0:
        return y
    if given:
        x_p, q_p, s_p, ld_q = None, x.data_ptr(), x_scale.data_ptr(), ld_x
    else:
        ld_q = (k + 15) // 16 * 16
        buf = torch.empty(rows * (ld_q + 4), dtype=torch.uint8, device=dev)
        x_p, q_p = x.data_ptr(), buf.data_ptr()
        s_p = q_p + rows * ld_q
    a = L.Int8LinearArgs(x_p, q_p, s_p, weight[0].data_ptr(), weight[1].data_ptr(),
                         None if bias is None else bias.data_ptr(), y.data_ptr(), rows, k, n, dt, ld_x, ld_q, ld_w, n,
                         None, 0, _err(dev))
    if rows > L.DENSE_FEW_TOKENS:
        ws = _workspace("dsca_int8_linear_workspace", a, dev)  # noqa: F841 - alive until the launch
    L.call_on(dev, "dsca_int8_linear", ctypes.byref(a))
    return without_gradient("int8_linear", y, x, bias, x_scale, weight[1])


def gated_ffn_int8(x: torch.Tensor, w_gate: Int8Weight, w_up: Int8Weight, w_down: Int8Weight,
                   act: str = "silu") -> torch.Tensor:
    """gated_ffn with its weights in 8-bit integers (pack_int8): x's rows are quantised, the gated
    intermediate is formed and its rows quantised in turn.  x [..., d] bf16 or fp32; y has its shape and
    type.  The intermediate is formed in fp32.  fp32 tokens: where that leaves a code open it is formed
    again in 64 bits, so that all codes are those of the definition.  bf16 tokens: a code next to a border may
    lie on its other side, which moves y by one code's worth of that channel.  Inference only: a
    backward pass that reaches y raises."""
    refuse_tangents("gated_ffn_int8", x)
    code = _act(act)
    dt = _DTYPES.get(x.dtype)
    if dt is None:
        raise ValueError(f"unsupported dtype {x.dtype}")
    rows, ld_x = _rows(x, "x")
    d, dev = x.shape[-1], x.device
    inter = w_gate[0].shape[0]
    if max(d, inter) > _INT8_MAX_K:
        raise ValueError(f"sums of {max(d, inter)} products exceed {_INT8_MAX_K}")
    ld_gate = _int8_weight(w_gate, "w_gate", dev, d)
    ld_up = _int8_weight(w_up, "w_up", dev, d, inter)
    ld_down = _int8_weight(w_down, "w_down", dev, inter, d)
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    if rows == 0:
        return y
    ld_q, ld_hq = (d + 15) // 16 * 16, (inter + 15) // 16 * 16
    # one buffer: h, the two sets of codes, the two sets of scales
    buf = torch.empty(rows * (5 * ld_hq + ld_q + 8), dtype=torch.uint8, device=dev)
    h = buf.data_ptr()
    hq = h + rows * 4 * ld_hq
    q = hq + rows * ld_hq
    scale = q + rows * ld_q
    a = L.GatedFfnInt8Args(x.data_ptr(), q, scale, w_gate[0].data_ptr(), w_up[0].data_ptr(), w_down[0].data_ptr(),
                           w_gate[1].data_ptr(), w_up[1].data_ptr(), w_down[1].data_ptr(), h, hq, scale + 4 * rows,
                           y.data_ptr(), rows, d, inter, dt, code, ld_x, ld_q, ld_gate, ld_up, ld_down, ld_hq, ld_hq, d,
                           None, 0, _err(dev))
    if rows > L.DENSE_FEW_TOKENS:
        ws = _workspace("dsca_gated_ffn_int8_workspace", a, dev)  # noqa: F841 - alive until the launch
    L.call_on(dev, "dsca_gated_ffn_int8", ctypes.byref(a))
    return without_gradient("gated_ffn_int8", y, x, w_gate[1], w_up[1], w_down[1])


# ----------------------------------------------------------------------------- module
_NAMES = (("gate_proj", "up_proj", "down_proj"), ("wi_0", "wi_1", "wo"))


def _act_name(mod) -> str:
    """The gate's name of a transformers MLP (its act_fn / act module)."""
    fn = getattr(mod, "act_fn", None)
    fn = getattr(mod, "act", None) if fn is None else fn
    name = type(fn).__name__
    if isinstance(fn, nn.SiLU) or name in ("SiLUActivation", "SiLU"):
        return "silu"
    if isinstance(fn, nn.ReLU):
        return "relu"
    if name in ("NewGELUActivation", "GELUTanh", "PytorchGELUTanh", "FastGELUActivation") \
            or (isinstance(fn, nn.GELU) and fn.approximate == "tanh"):
        return "gelu"
    raise ValueError(f"gate activation {name} is not offered (silu, tanh gelu, relu)")


def _bare(m: nn.Module) -> bool:
    """Whether nothing hangs on a module: no hook and no forward of its own."""
    return not (m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks
                or "forward" in m.__dict__)


def _plain(m: nn.Module) -> bool:
    """Whether a layer is its weight's product and nothing else: a Linear (adapters and parametrisations have types of their
    own) without bias and hooks, on an ordinary tensor."""
    return type(m) is nn.Linear and m.bias is None and type(m.weight) in (nn.Parameter, torch.Tensor) and _bare(m)


def _parts(old: nn.Module):
    """(names, Linear layers, gate, dropout or None) of a gated MLP; raises for one that is more than the block."""
    kind = type(old).__name__
    names = next((n for n in _NAMES if all(hasattr(old, m) for m in n)), None)
    if names is None:
        raise ValueError(f"{kind} has neither gate_proj / up_proj / down_proj nor wi_0 / wi_1 / wo")
    linears = [getattr(old, n) for n in names]
    if any(getattr(m, "bias", None) is not None for m in linears):
        raise ValueError("gated blocks with biases are not offered")
    act = _act_name(old)
    if not _bare(old) or not all(_plain(m) for m in linears):
        raise ValueError(f"{kind} has hooks, adapters or layers other than nn.Linear, which the block would leave out "
                         "(replace it first, then put them on)")
    dropout = getattr(old, "dropout", None)
    rest = sorted(set(dict(old.named_children())) - {*names, "act_fn", "act", "dropout"})
    if rest or not (dropout is None or type(dropout) is nn.Dropout):
        raise ValueError(f"{kind} has {', '.join(rest) or 'a dropout of its own'}, which the block would leave out")
    return names, linears, act, dropout


class GatedFFN(nn.Module):
    """A dense gated MLP (Qwen2MoeMLP's gate_proj / up_proj / down_proj, or wi_0 / wi_1 / wo) on gated_ffn.

    Keeps the old module's Linear layers under their names, so that its parameters, their gradients and
    state_dict stay what they were.  The layers run one by one, as in the old module, where the block is not the whole
    of it: with a dropout in training mode, with an adapter or a hook that was put on a layer since, with weights of another type than x
    (a `wo` kept in fp32), under fp16 autocast.  bf16 autocast runs the block in bf16.  Modules that already have hooks, adapters or other
    parts are refused.  int8=True packs the weights in 8-bit integers instead (buffers; inference only) and
    lets the Linear layers go."""

    def __init__(self, old: nn.Module, int8: bool = False):
        super().__init__()
        names, linears, act, dropout = _parts(old)
        self.names, self.act, self.int8 = names, act, bool(int8)
        self.act_fn = old.act_fn if getattr(old, "act_fn", None) is not None else old.act
        self.dropout = dropout
        self.training = old.training
        if not int8:
            for n, m in zip(names, linears):
                setattr(self, n, m)
            return
        self.widths = tuple(m.weight.shape[1] for m in linears)
        for n, m in zip(names, linears):
            q, scale = _quantize(m.weight.detach())
            self.register_buffer(n + "_q", q)  # whole padded rows, so that a copy keeps their layout
            self.register_buffer(n + "_scale", scale)

    def _apply(self, fn, recurse=True):
        """The scales of 8-bit weights stay fp32 when the model changes its type."""
        scales = {n: b for n, b in self._buffers.items() if n.endswith("_scale")}
        super()._apply(fn, recurse)
        for n, b in scales.items():
            if self._buffers[n].dtype != b.dtype:
                self._buffers[n] = b.to(self._buffers[n].device)
        return self

    def _layers(self, x: torch.Tensor) -> torch.Tensor:
        """The old module's forward."""
        gate, up, down = (getattr(self, n) for n in self.names)
        h = self.act_fn(gate(x)) * up(x)
        if self.dropout is not None:
            h = self.dropout(h)
        w = getattr(down, "weight", None)
        if self.names[2] == "wo" and isinstance(w, torch.Tensor) and w.is_floating_point() and h.dtype != w.dtype:
            h = h.to(w.dtype)
        return down(h)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        drop = self.dropout is not None and (type(self.dropout) is not nn.Dropout or not _bare(self.dropout)
                                             or (self.dropout.training and self.dropout.p > 0))
        amp = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else None
        if amp is not None and not (amp in _DTYPES and x.is_floating_point() and x.dtype != torch.float64):
            amp = None if self.int8 else False
        if self.int8:
            if drop:
                raise RuntimeError("a dropout is not offered on 8-bit weights (call eval())")
            return gated_ffn_int8(x if amp is None else x.to(amp),
                                  *(Int8Weight(getattr(self, n + "_q")[:, :k], getattr(self, n + "_scale"))
                                    for n, k in zip(self.names, self.widths)), act=self.act)
        linears = [getattr(self, n) for n in self.names]
        if drop or amp is False or not all(_plain(m) for m in linears):
            return self._layers(x)
        weights = [m.weight for m in linears]
        if amp is not None:  # what autocast does at each layer
            x, weights = x.to(amp), [w.to(amp) for w in weights]
        if any(w.dtype is not x.dtype for w in weights):
            return self._layers(x)
        return gated_ffn(x, *weights, act=self.act)
