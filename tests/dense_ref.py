"""The dense gated block and the 8-bit products in 64 bits, with bounds for every value.

Bounds.  A sum of k products in fp32, in any order and with truncating additions, is off by at most
(k + 8) 2^-23 of the sum of the products' magnitudes (`acc`).  Each rounding to the type is off by
half a step, eps / 2 (`half`).  The gates' exponentials and divisions are good to 2^-18 of their value
for 16-bit and 8-bit operands (the hardware's exponential: 2^-22, and 2^-24 |g| / ln 2 from its argument; where that
passes 2^-18, |g| > 45, the value is below e^-45), 2^-21 for 32-bit ones (`fast`).  |act'| <= 1.13 for all gates, |act''| <= 0.8 (relu: act' may be
anything in [0, 1] where g's own error reaches 0).  Errors of factors are carried through each
product at first order with both factors' magnitudes enlarged by their errors."""
import math

import torch

ACTS = ("silu", "gelu", "relu")


def act(g, name):
    """(act, act') in 64 bits."""
    if name == "relu":
        return g.clamp_min(0), (g > 0).double()
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    # (1 + tanh z) / 2 = sigmoid(2 z), which does not cancel where tanh z is near -1
    c = math.sqrt(2 / math.pi)
    p = torch.sigmoid(2 * c * (g + 0.044715 * g ** 3))
    return g * p, p + 2 * g * p * (1 - p) * c * (1 + 0.134145 * g * g)


def _acc(k):
    return (k + 8) * 2.0 ** -23


def _mul(a, da, b, db):
    """Error bound of a product of factors with errors da, db."""
    return da * b.abs() + a.abs() * db + da * db


def ffn(x, wg, wu, wd, name, dtype, dy=None):
    """{output: (value, bound)} for inputs of `dtype`."""
    half, fast = torch.finfo(dtype).eps / 2, 2.0 ** -18 if dtype == torch.bfloat16 else 2.0 ** -21
    x, wg, wu, wd = (t.double() for t in (x, wg, wu, wd))
    T, d = x.shape
    I = wg.shape[0]
    g, u = x @ wg.T, x @ wu.T
    eg, eu = _acc(d) * (x.abs() @ wg.abs().T), _acc(d) * (x.abs() @ wu.abs().T)
    a, da = act(g, name)
    ea = 1.13 * eg + fast * a.abs()
    h = a * u
    eh = _mul(a, ea, u, eu)
    eh = eh + half * (h.abs() + eh)
    y = h @ wd.T
    ey = eh @ wd.abs().T + _acc(I) * ((h.abs() + eh) @ wd.abs().T)
    out = {"y": (y, ey + half * (y.abs() + ey))}
    if dy is None:
        return out
    dy = dy.double()
    if dtype == torch.bfloat16:
        # the backward pass reads g and u as fp16: off by 2^-11 (half a step of 11 bits), or by half of 2^-24 of the
        # scaled range (2^-38 of the largest of a token's 32 channels)
        def held(v, e):
            big = torch.nn.functional.pad(v.abs() + e, (0, -I % 32)).view(T, -1, 32).amax(2)
            return e + 2.0 ** -11 * (v.abs() + e) + 2.0 ** -38 * big.repeat_interleave(32, 1)[:, :I]
        eg, eu = held(g, eg), held(u, eu)
    ea = 1.13 * eg + fast * (a.abs() + 1.13 * eg)
    eda = (g.abs() <= eg).double() if name == "relu" else 0.8 * eg + fast * (da.abs() + g.abs() * 0.5)
    dh = dy @ wd
    edh = _acc(d) * (dy.abs() @ wd.abs())
    t, et = dh * u, _mul(dh, edh, u, eu)
    dg, edg = t * da, _mul(t, et, da, eda)
    du, edu = dh * a, _mul(dh, edh, a, ea)
    edg, edu = edg + half * (dg.abs() + edg), edu + half * (du.abs() + edu)
    def dot(p, ep, q, eq, k):  # sums over the first index
        e = ep.T @ q.abs() + (p.abs() + ep).T @ eq if eq is not None else ep.T @ q.abs()
        return p.T @ q, e + _acc(k) * ((p.abs() + ep).T @ (q.abs() if eq is None else q.abs() + eq))
    vals = {}
    v1, e1 = dg @ wg, edg @ wg.abs()
    v2, e2 = du @ wu, edu @ wu.abs()
    vals["dx"] = (v1 + v2, e1 + e2 + _acc(2 * I) * ((dg.abs() + edg) @ wg.abs() + (du.abs() + edu) @ wu.abs()))
    vals["d_gate"] = dot(dg, edg, x, None, T)
    vals["d_up"] = dot(du, edu, x, None, T)
    v, e = dot(h, eh, dy, None, T)
    vals["d_down"] = (v.T, e.T)
    out.update({k: (v, e + half * (v.abs() + e)) for k, (v, e) in vals.items()})
    return out


def codes(v):
    """(codes, scale) of v's rows: ties to even; 1 for a row of zeros."""
    m = v.abs().amax(-1, keepdim=True)
    m1 = torch.where(m > 0, m, torch.full_like(m, 127.0))
    return torch.round(127 * v / m1), (m1 / 127)[..., 0]


def int8_linear(q, s, w, ws, dtype, bias=None):
    """(value, bound): the sum is exact; converting it, two scales' products and the bias round five
    times (2^-24 each, scales as given), the result once more."""
    y = (q.double() @ w.double().T) * s.double()[:, None] * ws.double()
    e = 5 * 2.0 ** -24 * y.abs()
    if bias is not None:
        y = y + bias.double()
        e = e + 2.0 ** -24 * y.abs()
    return y, e * 1.01 + torch.finfo(dtype).eps / 2 * (y.abs() + e)


def ffn_int8(x, wg, wu, wd, name, dtype):
    """(value, bound); weights as (codes, scale).  h's error may move a code by one where its quotient lies
    within that error of a tie."""
    q, s = codes(x.double())
    s = s.float().double()  # as the rows hold it
    def prod(w):
        v = (q @ w[0].double().T) * s[:, None] * w[1].double()
        return v, 4 * 2.0 ** -24 * v.abs()
    (g, eg), (u, eu) = prod(wg), prod(wu)
    a, _ = act(g, name)
    ea = 1.13 * eg + 2.0 ** -18 * a.abs()
    h = a * u
    eh = _mul(a, ea, u, eu) * 1.01 + 2.0 ** -24 * h.abs()
    m = h.abs().amax(-1, keepdim=True)
    em = eh.amax(-1, keepdim=True)  # the largest of rows that differ by at most this
    m1 = torch.where(m > 0, m, torch.full_like(m, 127.0))
    quo = 127 * h / m1
    equo = (127 * eh + quo.abs() * em) / (m1 - em).clamp_min(1e-300)
    hq = torch.round(quo)
    near = ((quo - torch.floor(quo) - 0.5).abs() <= equo + 1e-9).double()
    wdq, wds = wd[0].double(), wd[1].double()
    y = (hq @ wdq.T) * (m1 / 127) * wds
    e = (near @ wdq.abs().T) * (m1 / 127) * wds + y.abs() * (em / m1 + 6 * 2.0 ** -24)
    return y, e * 1.01 + torch.finfo(dtype).eps / 2 * (y.abs() + e)


def close(got, ref, what=""):
    v, e = ref
    assert tuple(got.shape) == tuple(v.shape), what
    bad = ~((got.double() - v).abs() <= e + 1e-37)
    assert not bad.any(), (what, int(bad.sum()), float(((got.double() - v).abs() / (e + 1e-37)).max()))
