"""What the dense gated feed-forward block and the 8-bit integer product are measured on.

Four operators that a program around an MoE block runs on its dense layers:

  ffn    the gated feed-forward block y = (act(x Wg^T) * (x Wu^T)) Wd^T, in 16 or 32 bits
  train  the same with its backward pass: y, dx, dWg, dWu, dWd for a given dy
  int8   y = x W^T with x and W in 8-bit integers, one scale a token and one an output channel; the
         token's scale and codes are made within the call
  ffn8   the gated block with its three weights in 8-bit integers, the intermediate rows quantised
         like the tokens

A row's scale is max|x| / 127 (1 for a row of zeros), its codes those of the quotient 127 x / max|x|,
ties to even.  With `own` false, run() computes the operators from elementary torch operations in 32
bits (the codes in 64, since they hang on a border); with `own` true it makes the calls a user makes
of this package.
"""
import math

import torch

own = False


def _case(name, kind, **kw):
    return dict(name=name, kind=kind, **kw)


def _ffn(name, T, d, inter, kind="ffn", dtype="bf16", act="silu"):
    return _case(name, kind, T=T, d=d, inter=inter, dtype=dtype, act=act)


def _int8(name, T, k, n, dtype="bf16", bias=False):
    return _case(name, "int8", T=T, k=k, n=n, dtype=dtype, bias=bias)


def listed():
    return [
        # one decode token through a dense block of the shared expert's size: only the weights' stream counts
        _ffn("ffn-1-qwen", 1, 2048, 5632),
        # a prefill batch of 16 x 256 tokens
        _ffn("ffn-4096-qwen", 4096, 2048, 5632),
        # odd sizes in fp32, gelu gate
        _ffn("ffn-100-f32", 100, 712, 1021, dtype="f32", act="gelu"),
        # a fine-tuning step on a small batch of a narrow model
        _ffn("train-640-narrow", 640, 768, 2048, kind="train", act="gelu"),
        # rows that no 16-byte vector fits, in both widths, relu gate
        _ffn("train-333-odd", 333, 1021, 901, kind="train", act="relu"),
        # fp32 training of a small block
        _ffn("train-256-f32", 256, 712, 1408, kind="train", dtype="f32"),
        # a large fine-tuning batch: 32 x 256 tokens
        _ffn("train-8192-qwen", 8192, 2048, 5632, kind="train"),
        # the vocabulary's projection of a decode batch
        _int8("int8-32-head", 32, 2048, 151936),
        # odd sizes, fp32 tokens, with a bias
        _int8("int8-777-odd", 777, 1021, 1363, dtype="f32", bias=True),
        # the down projection of a large prefill batch
        _int8("int8-16384-down", 16384, 5632, 2048),
        # one decode token through the block with 8-bit weights, and a prefill batch
        _ffn("ffn8-1-qwen", 1, 2048, 5632, kind="ffn8"),
        _ffn("ffn8-4096-qwen", 4096, 2048, 5632, kind="ffn8"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A row's width: a multiple of eight more often than not."""
    v = _log_int(rng, lo, hi)
    return max(8, v // 8 * 8) if rng.random() < 0.6 else v


def draw(rng):
    kind = rng.choice(("ffn", "train", "int8", "ffn8"))
    dtype = "f32" if rng.random() < 0.25 else "bf16"
    if kind == "int8":
        k, n = _width(rng, 48, 8192), _width(rng, 48, 65536)
        T = min(_log_int(rng, 1, 16384), max(1, 16384 * 5632 * 2048 // (k * n)))
        return dict(kind=kind, T=T, k=k, n=n, dtype=dtype, bias=rng.random() < 0.3)
    d, inter = _width(rng, 48, 4096), _width(rng, 48, 6144)
    most = 8192 * 2048 * 5632 // (20 if dtype == "f32" else 1)
    T = min(_log_int(rng, 1, 16384), max(1, most // (d * inter)))
    return dict(kind=kind, T=T, d=d, inter=inter, dtype=dtype, act=rng.choice(("silu", "gelu", "relu")))


# ----------------------------------------------------------------------------- inputs
def _dtype(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def _codes(x):
    """(codes as whole numbers in fp32, scale) of x's rows."""
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True)
    scale = torch.where(amax > 0, amax / 127.0, torch.ones_like(amax))
    q = x.double() * 127.0 / torch.where(amax > 0, amax, torch.ones_like(amax)).double()
    return torch.round(q).float(), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = _dtype(case["dtype"])

    def n(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dt)

    def tokens(T, d):
        # normed hidden states of a model: tokens of somewhat different magnitude
        return (torch.randn(T, d, generator=g, device="cuda")
                * torch.exp(0.3 * torch.randn(T, 1, generator=g, device="cuda"))).to(dt)

    s = dict(case=case)
    if case["kind"] == "int8":
        s["x"] = tokens(case["T"], case["k"])
        w = {"w": n(case["n"], case["k"], std=case["k"] ** -0.5)}
        s["bias"] = n(case["n"]) if case["bias"] else None
    else:
        T, d, I = case["T"], case["d"], case["inter"]
        s["x"] = tokens(T, d)
        w = dict(gate=n(I, d, std=d ** -0.5), up=n(I, d, std=d ** -0.5), down=n(d, I, std=I ** -0.5))
        if case["kind"] == "train":
            s["dy"] = n(T, d, std=0.1)
    if case["kind"] in ("int8", "ffn8"):
        if own:
            from dsca_moe_b200 import Int8Weight, pack_int8

            # a serving program's weights, with the scales that the plain form has: _codes divides on the GPU, where torch
            # multiplies by 1 / 127, so that they may be a step from pack_int8's, and a code of the intermediate
            # next to a border hangs on it
            s["w"] = {key: Int8Weight(pack_int8(v).q, _packed(v)[1]) for key, v in w.items()}
        else:
            s["w"] = {key: _packed(v) for key, v in w.items()}
        return s
    if own and case["kind"] == "train":
        s["x"].requires_grad_()
        for v in w.values():
            v.requires_grad_()
    s["w"] = w
    return s


def _packed(w):
    q, scale = _codes(w)
    return q.to(torch.int8), scale[:, 0]


# ----------------------------------------------------------------------------- one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        return _OWN[kind](state)
    return _PLAIN[kind](state)


def _act(g, act):
    if act == "silu":
        return g * torch.sigmoid(g)
    if act == "relu":
        return torch.relu(g)
    return 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g)))


def _act_grad(g, act):
    if act == "silu":
        s = torch.sigmoid(g)
        return s * (1.0 + g * (1.0 - s))
    if act == "relu":
        return (g > 0).to(g.dtype)
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * g * g)


def _run_ffn(s):
    x, w, act = s["x"].float(), s["w"], s["case"]["act"]
    h = _act(x @ w["gate"].float().T, act) * (x @ w["up"].float().T)
    return {"y": (h @ w["down"].float().T).to(s["x"].dtype)}


def _run_train(s):
    dt, act = s["x"].dtype, s["case"]["act"]
    x, dy = s["x"].float(), s["dy"].float()
    wg, wu, wd = (s["w"][n].float() for n in ("gate", "up", "down"))
    g, u = x @ wg.T, x @ wu.T
    a = _act(g, act)
    h = a * u
    dh = dy @ wd
    dg, du = dh * u * _act_grad(g, act), dh * a
    out = {"y": h @ wd.T, "dx": dg @ wg + du @ wu, "dgate": dg.T @ x, "dup": du.T @ x, "ddown": dy.T @ h}
    return {k: v.to(dt) for k, v in out.items()}


def _product(q, scale, w):
    return (q @ w[0].float().T) * scale * w[1]


def _run_int8(s):
    q, scale = _codes(s["x"])
    y = _product(q, scale, s["w"]["w"])
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return {"y": y.to(s["x"].dtype)}


def _run_ffn8(s):
    w = s["w"]
    q, scale = _codes(s["x"])
    h = _act(_product(q, scale, w["gate"]), s["case"]["act"]) * _product(q, scale, w["up"])
    q, scale = _codes(h)
    return {"y": _product(q, scale, w["down"]).to(s["x"].dtype)}


def _own_ffn(s):
    from dsca_moe_b200 import gated_ffn

    w = s["w"]
    return {"y": gated_ffn(s["x"], w["gate"], w["up"], w["down"], act=s["case"]["act"])}


def _own_train(s):
    from dsca_moe_b200 import gated_ffn

    w = s["w"]
    y = gated_ffn(s["x"], w["gate"], w["up"], w["down"], act=s["case"]["act"])
    dx, dgate, dup, ddown = torch.autograd.grad(y, (s["x"], w["gate"], w["up"], w["down"]), s["dy"])
    return {"y": y.detach(), "dx": dx, "dgate": dgate, "dup": dup, "ddown": ddown}


def _own_int8(s):
    from dsca_moe_b200 import int8_linear

    return {"y": int8_linear(s["x"], s["w"]["w"], bias=s["bias"])}


def _own_ffn8(s):
    from dsca_moe_b200 import gated_ffn_int8

    w = s["w"]
    return {"y": gated_ffn_int8(s["x"], w["gate"], w["up"], w["down"], act=s["case"]["act"])}


_PLAIN = dict(ffn=_run_ffn, train=_run_train, int8=_run_int8, ffn8=_run_ffn8)
_OWN = dict(ffn=_own_ffn, train=_own_train, int8=_own_int8, ffn8=_own_ffn8)


# ----------------------------------------------------------------------------- floors
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    T = case["T"]
    if case["kind"] == "int8":
        k, n = case["k"], case["n"]
        nbytes = e * T * (k + n) + n * (k + 4) + (e * n if case["bias"] else 0)
        return {"bytes": nbytes, "flops": 2.0 * T * k * n}
    d, I = case["d"], case["inter"]
    if case["kind"] == "ffn":
        return {"bytes": e * (2 * T * d + 3 * I * d), "flops": 6.0 * T * d * I}
    if case["kind"] == "ffn8":
        return {"bytes": e * 2 * T * d + 3 * I * d + 4 * (2 * I + d), "flops": 6.0 * T * d * I}
    # x and dy read, y and dx written; the weights read, their gradients written
    return {"bytes": e * (4 * T * d + 6 * I * d), "flops": 18.0 * T * d * I}


# ----------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    x = s["x"].double()
    if case["kind"] == "int8":
        q, sc = _exact_rows(x)
        w, ws = s["w"]["w"]
        y = torch.einsum("tk,nk->tn", q, w.double()) * sc.unsqueeze(1) * ws.double().unsqueeze(0)
        return {"y": y if s["bias"] is None else y + s["bias"].double()}
    if case["kind"] == "ffn8":
        q, sc = _exact_rows(x)
        (wg, sg), (wu, su), (wd, sd) = (s["w"][n] for n in ("gate", "up", "down"))
        g = torch.einsum("td,id->ti", q, wg.double()) * sc.unsqueeze(1) * sg.double()
        u = torch.einsum("td,id->ti", q, wu.double()) * sc.unsqueeze(1) * su.double()
        q, sc = _exact_rows(_exact_gate(g, case["act"])[0] * u)
        return {"y": torch.einsum("ti,di->td", q, wd.double()) * sc.unsqueeze(1) * sd.double()}
    wg, wu, wd = (s["w"][n].double() for n in ("gate", "up", "down"))
    g, u = torch.einsum("td,id->ti", x, wg), torch.einsum("td,id->ti", x, wu)
    a, da = _exact_gate(g, case["act"])
    out = {"y": torch.einsum("ti,di->td", a * u, wd)}
    if case["kind"] == "ffn":
        return out
    dy = s["dy"].double()
    dh = torch.einsum("td,di->ti", dy, wd)
    dg, du = dh * u * da, dh * a
    out["dx"] = torch.einsum("ti,id->td", dg, wg) + torch.einsum("ti,id->td", du, wu)
    out["dgate"] = torch.einsum("ti,td->id", dg, x)
    out["dup"] = torch.einsum("ti,td->id", du, x)
    out["ddown"] = torch.einsum("td,ti->di", dy, a * u)
    return out


def _exact_rows(v):
    """(codes, scale) of the rows of v in 64 bits."""
    m = v.abs().max(dim=1).values
    m = torch.where(m == 0, torch.full_like(m, 127.0), m)
    return torch.round(127.0 * v / m.unsqueeze(1)), m / 127.0


def _exact_gate(g, act):
    """The gate's value and derivative in 64 bits."""
    if act == "relu":
        return g.clamp_min(0.0), (g > 0).double()
    if act == "silu":
        e = torch.exp(-g.abs())
        s = torch.where(g >= 0, 1.0 / (1.0 + e), e / (1.0 + e))
        return g * s, s + g * s * (1.0 - s)
    c = (2.0 / math.pi) ** 0.5
    z = c * (g + 0.044715 * g ** 3)
    p = 1.0 / (1.0 + torch.exp(-2.0 * z))  # (1 + tanh z) / 2
    return g * p, p + g * 2.0 * p * (1.0 - p) * c * (1.0 + 0.134145 * g ** 2)
