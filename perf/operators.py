"""What the operators around a decode step's MoE block are measured on.

Two operators that follow one another in a decoder layer:

  norm   h = x + residual, y = w * h / sqrt(mean(h^2) + eps), with the residual stream h as an
         output of its own and, on request, y in 8 bits with one scale a row: quant "e4m3" (one e4m3
         term, scale = max|y| / 448) or "split" (two e4m3 terms and a power-of-two scale, the token
         operand of the fp8-weight expert products)
  moe    the whole mixture-of-experts block for a few tokens: router, softmax, top-k, the chosen
         experts' FFNs (SwiGLU, or ReLU behind a top-1 router), the gated shared expert, and the
         weighted sum

With `own` false, run() computes them from elementary torch operations in 32 bits (the router's
products in 64, since a choice of experts hangs on the logits' last bits); with `own` true it makes
the calls a user makes of this package.
"""
import math

import torch

own = False

EPS = 1e-6


def _case(name, kind, **kw):
    return dict(name=name, kind=kind, **kw)


def _norm(name, rows, d, dtype="bf16", residual=True, quant="none", gap=0):
    return _case(name, "norm", rows=rows, d=d, dtype=dtype, residual=residual, quant=quant, gap=gap)


def _moe(name, T, d, E, k, inter, shared, weights="bf16", act="swiglu", norm_topk=False):
    return _case(name, "moe", T=T, d=d, E=E, k=k, inter=inter, shared=shared, weights=weights, act=act,
                 norm_topk=norm_topk)


def listed():
    return [
        # one decode token of a 2048-wide model: only latency counts
        _norm("norm-1x2048", 1, 2048),
        # a decode batch in front of an fp8-weight block, two-term rows written along
        _norm("norm-32x2048-split", 32, 2048, quant="split"),
        # the first norm of a model: nothing to add yet, odd width, fp32, rows cut out of a wider buffer
        _norm("norm-777x1021-f32", 777, 1021, dtype="f32", residual=False, gap=3),
        # one prefill batch of 16 x 256 tokens, 8-bit rows for storage or exchange
        _norm("norm-4096x2048-e4m3", 4096, 2048, quant="e4m3"),
        # the largest prefill batch of one GPU
        _norm("norm-16384x2048", 16384, 2048),
        # a narrow model's batch with two-term rows
        _norm("norm-20000x768-split", 20000, 768, quant="split"),
        # one token through a Qwen-shaped block (60 experts, top-4, shared expert): single-stream decoding
        _moe("moe-1-qwen", 1, 2048, 60, 4, 1408, 5632),
        # the same with fp8 weights
        _moe("moe-1-qwen-fp8", 1, 2048, 60, 4, 1408, 5632, weights="fp8"),
        # a small decode batch, and the largest one
        _moe("moe-8-qwen", 8, 2048, 60, 4, 1408, 5632),
        _moe("moe-32-qwen-fp8", 32, 2048, 60, 4, 1408, 5632, weights="fp8"),
        # a Switch-style layer: top-1, ReLU experts, no shared expert
        _moe("moe-16-switch", 16, 768, 64, 1, 2048, 0, act="relu"),
        # odd sizes in fp32: few experts, weights of the chosen ones normalised
        _moe("moe-5-f32", 5, 712, 13, 3, 333, 901, weights="f32", norm_topk=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        dtype = "bf16" if rng.random() < 0.7 else "f32"
        quant = rng.choice(("none", "none", "e4m3", "split"))
        d = _log_int(rng, 64, 8192)
        if rng.random() < 0.6 or quant == "split":
            d = max(64, d // 8 * 8)
        if quant == "split":
            dtype = "bf16"
        rows = _log_int(rng, 1, min(32768, 16384 * 2048 // d // (1 if dtype == "bf16" else 2)))
        return dict(kind="norm", rows=rows, d=d, dtype=dtype, residual=rng.random() < 0.7, quant=quant,
                    gap=rng.choice((0, 0, 8, 5)))
    weights = rng.choice(("bf16", "bf16", "fp8", "f32"))
    act = "swiglu" if rng.random() < 0.7 else "relu"
    E = rng.randint(4, 63)
    k = rng.randint(1, min(8, E)) if act == "swiglu" else 1
    T = _log_int(rng, 1, 32)
    d = _log_int(rng, 128, 2560) // 16 * 16
    inter = _log_int(rng, 48, 2048)
    if weights == "f32":  # as many bytes as the other types' cases
        inter = max(48, inter // 2)
    # no more expert rows gathered than the largest listed case has
    T = max(1, min(T, 32 * 4 * 1408 * 2048 // (k * inter * d)))
    shared = _log_int(rng, 64, 5632) if act == "swiglu" and rng.random() < 0.6 else 0
    return dict(kind="moe", T=T, d=d, E=E, k=k, inter=inter, shared=shared, weights=weights, act=act,
                norm_topk=rng.random() < 0.3)


# ----------------------------------------------------------------------------- inputs
def _dtype(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def _quantised(w):
    """Rows of w as e4m3 with one fp32 scale a row (largest magnitude to 448)."""
    w = w.float()
    amax = w.abs().amax(-1, keepdim=True)
    scale = torch.where(amax > 0, amax / 448.0, torch.ones_like(amax))
    return (w / scale).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def n(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    if case["kind"] == "norm":
        dt, rows, d = _dtype(case["dtype"]), case["rows"], case["d"]
        # a block's output, and a residual stream that has grown over the layers, tokens of
        # different magnitude; the rows may lie in a wider buffer
        x = n(rows, d + case["gap"], dtype=dt)[:, :d]
        residual = (n(rows, d) * torch.exp(n(rows, 1, std=0.7)) * 3.0).to(dt) if case["residual"] else None
        return dict(case=case, x=x, residual=residual, weight=(1.0 + n(d, std=0.2)).to(dt))
    dt = torch.float32 if case["weights"] == "f32" else torch.bfloat16
    T, d, E, I, Is = case["T"], case["d"], case["E"], case["inter"], case["shared"]
    s = dict(case=case, x=n(T, d, dtype=dt), router=n(E, d, std=d ** -0.5, dtype=dt), gate=None)
    if case["act"] == "swiglu":
        w = dict(gate=n(E, I, d, std=0.02, dtype=dt), up=n(E, I, d, std=0.02, dtype=dt),
                 down=n(E, d, I, std=0.02, dtype=dt))
    else:
        w = dict(wi=n(E, I, d, std=0.02, dtype=dt), wo=n(E, d, I, std=0.02, dtype=dt))
    if Is:
        w.update(s_gate=n(Is, d, std=0.02, dtype=dt), s_up=n(Is, d, std=0.02, dtype=dt),
                 s_down=n(d, Is, std=0.02, dtype=dt))
        s["gate"] = n(d, std=d ** -0.5, dtype=dt)
    if own:
        s["engine"] = _engine(case, s, w)
        return s
    s["w"] = {key: _quantised(v) for key, v in w.items()} if case["weights"] == "fp8" else {
        key: (v, None) for key, v in w.items()}
    return s


def _engine(case, s, w):
    """The handle a serving program keeps for a block: its packed weights and workspaces."""
    from dsca_moe_b200 import MoEEngine, pack_relu, pack_swiglu
    from dsca_moe_b200 import _lib as L
    from dsca_moe_b200.engine import quantize_fp8

    dt = s["x"].dtype
    if case["act"] == "swiglu":
        shared = (w["s_gate"], w["s_up"], w["s_down"]) if case["shared"] else None
        packed = pack_swiglu(w["gate"], w["up"], w["down"], shared=shared, dtype=dt)
    else:
        packed = pack_relu(w["wi"], w["wo"], dtype=dt)
    if case["weights"] == "fp8":
        packed = quantize_fp8(packed)
    mode = L.ROUTE_SOFTMAX_TOPK if case["act"] == "swiglu" else L.ROUTE_SWITCH_TOP1
    return MoEEngine(s["router"], packed, top_k=case["k"], route_mode=mode, norm_topk=case["norm_topk"],
                     shared_gate_weight=s["gate"])


# ----------------------------------------------------------------------------- one pass
def run(state):
    if state["case"]["kind"] == "norm":
        return _run_norm_own(state) if own else _run_norm(state)
    return _run_moe_own(state) if own else _run_moe(state)


def _run_norm_own(s):
    from dsca_moe_b200 import add_rms_norm

    quant = s["case"]["quant"]
    r = add_rms_norm(s["x"], s["weight"], eps=EPS, residual=s["residual"], quant=None if quant == "none" else quant)
    return _norm_outputs(r.y, r.residual if s["residual"] is not None else None, r.q, r.scale)


def _norm_outputs(y, residual, q, scale):
    out = {"y": y}
    if residual is not None:
        out["residual"] = residual
    if q is not None:
        out["q"], out["scale"] = q, scale
    return out


def _run_norm(s):
    dt, quant = s["x"].dtype, s["case"]["quant"]
    h = s["x"].float()
    residual = None
    if s["residual"] is not None:
        # the stream is held in its own type, and the norm is of what is held
        residual = (h + s["residual"].float()).to(dt)
        h = residual.float()
    d = h.shape[1]
    inv = torch.rsqrt((h * h).sum(-1, keepdim=True) / d + EPS)
    yf = h * inv * s["weight"].float()
    y = yf.to(dt)
    if quant == "e4m3":
        amax = yf.abs().amax(-1, keepdim=True)
        scale = torch.where(amax > 0, amax / 448.0, torch.ones_like(amax))
        return _norm_outputs(y, residual, (yf / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), scale[:, 0])
    if quant == "split":
        v = y.float()  # the two terms stand for the rounded row
        e = torch.frexp(v.abs().amax(-1, keepdim=True))[1] - 1
        e = torch.where(v.abs().amax(-1, keepdim=True) > 0, e, torch.full_like(e, -127)).clamp(-119, 127)
        v = torch.ldexp(v, 7 - e)
        hi = v.to(torch.float8_e4m3fn)
        lo = (v - hi.float()).to(torch.float8_e4m3fn)
        pad = (0, -d % 128)
        q = torch.cat([torch.nn.functional.pad(hi.view(torch.uint8), pad),
                       torch.nn.functional.pad(lo.view(torch.uint8), pad)], 1).view(torch.float8_e4m3fn)
        return _norm_outputs(y, residual, q, torch.ldexp(torch.ones_like(v[:, 0]), e[:, 0] - 7))
    return _norm_outputs(y, residual, None, None)


def _run_moe_own(s):
    r = s["engine"].forward_few(s["x"])
    return {"out": r["out"], "logits": r["logits"], "topk_ids": r["topk_ids"], "topk_w": r["topk_w"]}


def _rows(w, ids=None):
    """Weight rows in 32 bits, those of the experts `ids` (all without)."""
    v, scale = w
    if ids is not None:
        v = v.view(torch.uint8)[ids].view(v.dtype) if scale is not None else v[ids]
    return v.float() if scale is None else v.float() * (scale if ids is None else scale[ids])


def _route(x, router, case):
    """(logits in the router's type, ids, weights): softmax in 32 bits, the k largest, the lowest id
    first among equals; a top-1 router holds its probabilities in its own type."""
    logits = (x.double() @ router.double().T).to(x.dtype)
    p = torch.softmax(logits.float(), -1)
    if case["act"] == "relu":
        p = p.to(x.dtype).float()
    p, ids = torch.sort(p, dim=-1, descending=True, stable=True)
    p, ids = p[:, :case["k"]], ids[:, :case["k"]]
    if case["act"] == "swiglu":
        if case["norm_topk"]:
            p = p / p.sum(-1, keepdim=True)
        p = p.to(x.dtype).float()
    return logits, ids, p


def _run_moe(s):
    case, x, w = s["case"], s["x"], s["w"]
    T, d, k = case["T"], case["d"], case["k"]
    logits, ids, p = _route(x, s["router"], case)
    a = ids.reshape(-1)
    xa = x.float().repeat_interleave(k, 0).unsqueeze(-1)  # one column for each (token, choice)
    if case["act"] == "swiglu":
        g, u = _rows(w["gate"], a) @ xa, _rows(w["up"], a) @ xa
        y = _rows(w["down"], a) @ (g * torch.sigmoid(g) * u)
    else:
        y = _rows(w["wo"], a) @ torch.relu(_rows(w["wi"], a) @ xa)
    out = (y.view(T, k, d) * p.unsqueeze(-1)).sum(1)
    if case["shared"]:
        xf = x.float()
        g, u = xf @ _rows(w["s_gate"]).T, xf @ _rows(w["s_up"]).T
        ys = (g * torch.sigmoid(g) * u) @ _rows(w["s_down"]).T
        z = (x.double() @ s["gate"].double()).to(x.dtype).float()
        out = out + torch.sigmoid(z).unsqueeze(-1) * ys
    return {"out": out.to(x.dtype), "logits": logits, "topk_ids": ids.to(torch.int32), "topk_w": p}


# ----------------------------------------------------------------------------- floors
def work(case):
    if case["kind"] == "norm":
        rows, d = case["rows"], case["d"]
        e = 4 if case["dtype"] == "f32" else 2
        nbytes = rows * d * e * (4 if case["residual"] else 2) + d * e
        if case["quant"] == "e4m3":
            nbytes += rows * d + 4 * rows
        elif case["quant"] == "split":
            nbytes += rows * 2 * (-(-d // 128) * 128) + 4 * rows
        return {"bytes": nbytes, "flops": 5 * rows * d}
    T, d, E, k, I, Is = (case[n] for n in ("T", "d", "E", "k", "inter", "shared"))
    e = {"bf16": 2, "fp8": 1, "f32": 4}[case["weights"]]
    xe = 4 if case["weights"] == "f32" else 2
    mats = 3 if case["act"] == "swiglu" else 2
    # experts that at least one of T tokens chooses, the choices spread evenly
    active = E * (1.0 - (1.0 - k / E) ** T)
    nbytes = (active * mats * I * d + 3 * Is * d) * e + (E + (1 if Is else 0)) * d * xe + 2 * T * d * xe + T * E * xe
    if case["weights"] == "fp8":
        nbytes += 4 * (active * ((mats - 1) * I + d) + ((2 * Is + d) if Is else 0))
    return {"bytes": nbytes, "flops": 2.0 * T * d * (k * mats * I + 3 * Is + E)}


# ----------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return _exact_norm(s) if case["kind"] == "norm" else _exact_moe(s)


def _exact_norm(s):
    case, dt = s["case"], s["x"].dtype
    h = s["x"].double()
    out = {}
    if s["residual"] is not None:
        t = h + s["residual"].double()
        out["residual"] = t
        h = t.to(dt).double()  # the definition: the norm of the stream as it is held
    y = s["weight"].double() * h / torch.sqrt(torch.mean(h * h, dim=1, keepdim=True) + EPS)
    out["y"] = y
    if case["quant"] == "e4m3":
        m = y.abs().max(dim=1, keepdim=True).values
        sc = torch.where(m == 0, torch.ones_like(m), m / 448)
        out["q"], out["scale"] = y / sc, sc.squeeze(1)
    elif case["quant"] == "split":
        v = y.to(dt).double()
        m = v.abs().max(dim=1).values.clamp_min(2.0 ** -119)
        inv = torch.pow(2.0, torch.floor(torch.log2(m)) - 7)
        v = v / inv.unsqueeze(1)
        hi = v.to(torch.float8_e4m3fn).double()
        kp = -(-case["d"] // 128) * 128
        q = torch.zeros(v.shape[0], 2 * kp, dtype=torch.float64, device=v.device)
        q[:, :case["d"]] = hi
        q[:, kp:kp + case["d"]] = v - hi
        out["q"], out["scale"] = q, inv
    return out


def _exact_moe(s):
    case, dt = s["case"], s["x"].dtype
    x = s["x"].double()

    def full(name, i=None):
        v, scale = s["w"][name]
        v = v if i is None else v[i]
        return v.double() if scale is None else v.double() * (scale if i is None else scale[i]).double()

    lg = x @ s["router"].double().T
    held = lg.to(dt).double()
    ex = torch.exp(held - held.max(dim=1, keepdim=True).values)
    prob = ex / ex.sum(dim=1, keepdim=True)
    if case["act"] == "relu":
        prob = prob.to(dt).double()
    out = torch.zeros_like(x)
    weights = torch.zeros(case["T"], case["k"], dtype=torch.float64, device=x.device)
    left = prob.clone()
    chosen = []
    for j in range(case["k"]):
        best = left.max(dim=1, keepdim=True).values
        first = torch.argmax((left == best).int(), dim=1)
        chosen.append(first)
        weights[:, j] = best[:, 0]
        left.scatter_(1, first.unsqueeze(1), -1.0)
    if case["act"] == "swiglu":
        if case["norm_topk"]:
            weights = weights / weights.sum(dim=1, keepdim=True)
        weights = weights.to(dt).double()
    ids = torch.stack(chosen, 1)
    for e in range(case["E"]):
        t, j = (ids == e).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        if case["act"] == "swiglu":
            g = x[t] @ full("gate", e).T
            mid = g / (1 + torch.exp(-g)) * (x[t] @ full("up", e).T)
            y = mid @ full("down", e).T
        else:
            y = (x[t] @ full("wi", e).T).clamp_min(0) @ full("wo", e).T
        out.index_add_(0, t, weights[t, j].unsqueeze(1) * y)
    if case["shared"]:
        g = x @ full("s_gate").T
        ys = (g / (1 + torch.exp(-g)) * (x @ full("s_up").T)) @ full("s_down").T
        z = (x @ s["gate"].double()).to(dt).double()
        out = out + ys / (1 + torch.exp(-z)).unsqueeze(1)
    return {"out": out, "logits": lg, "topk_ids": None, "topk_w": weights}
