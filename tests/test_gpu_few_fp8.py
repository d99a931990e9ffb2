"""forward_few with fp8 weights whose magnitudes differ between rows, experts and the shared expert.

The tolerance is that of the other tests of this block with what the interface states for these weights: a value of
the intermediate is held to 11 significant bits (off by 2^-11 of itself at most), or to 2^-16 of the largest value of
its token's row in that expert (half the spacing of f16's smallest numbers, 2^-25, where that largest value is at
least 2^-9)."""
import pytest
import torch

from oracle import oracle as O
from test_gpu_few import _route, _run, _weights

pytestmark = pytest.mark.gpu

EPS = torch.finfo(torch.float16).eps / 2
FLOOR = 2.0 ** -16


def dequantised(w):
    amax = w.float().abs().amax(-1, keepdim=True)
    s = torch.where(amax > 0, amax / 448.0, torch.ones_like(amax))
    return (w.float() / s).to(torch.float8_e4m3fn).double() * s.double()


def block(dev, d, E, k, I, Is=0, act="swiglu", seed=1, change=None):
    """(engine, its weights in fp64, router, gate, random numbers); change(w) edits the weights first."""
    from dsca_moe_b200 import _lib as L
    from dsca_moe_b200.engine import MoEEngine, pack_relu, pack_swiglu, quantize_fp8

    w, router, gate, n = _weights(dev, d, E, I, Is, act, torch.bfloat16, seed)
    if change is not None:
        change(w)
    if act == "swiglu":
        pe = pack_swiglu(w["gate"], w["up"], w["down"], shared=(w["s_gate"], w["s_up"], w["s_down"]) if Is else None, device=dev)
    else:
        pe = pack_relu(w["gate"], w["down"], device=dev)
    eng = MoEEngine(router, quantize_fp8(pe), top_k=k, shared_gate_weight=gate,
                    route_mode=L.ROUTE_SOFTMAX_TOPK if act == "swiglu" else L.ROUTE_SWITCH_TOP1)
    return eng, {key: dequantised(v) for key, v in w.items()}, router, gate, n


def ffn(x, gate, up, down, floor=FLOOR):
    """(result, bound of its error before the last rounding) of one expert in 64 bits."""
    d, I = gate.shape[1], gate.shape[0]
    c1, c2 = (d / 8 + 32) * 2.0 ** -23, (I / 8 + 32) * 2.0 ** -23
    g, eg = x @ gate.T, c1 * (x.abs() @ gate.abs().T)
    if up is None:
        h, eh = g.clamp_min(0), eg
    else:
        u, eu = x @ up.T, c1 * (x.abs() @ up.abs().T)
        s = g * torch.sigmoid(g)
        h, eh = s * u, 1.1 * eg * (u.abs() + eu) + s.abs() * eu
    eh = eh + torch.maximum(EPS * h.abs(), floor * (h.abs() + eh).amax(-1, keepdim=True))
    return h @ down.T, eh @ down.abs().T + c2 * ((h.abs() + eh) @ down.abs().T)


def check(r, x, w, router, gate, k, top1=False):
    lg, ids, p = _route(x, router, k, top1, False)
    assert torch.equal(r["logits"], lg) and torch.equal(r["topk_ids"].long(), ids) and torch.equal(r["topk_w"], p)
    xd, p = x.double(), p.double()
    y, err = torch.zeros_like(xd), torch.zeros_like(xd)
    for e in ids.unique().tolist():
        t, j = (ids == e).nonzero(as_tuple=True)
        o, eo = ffn(xd[t], w["gate"][e], w["up"][e] if "up" in w else None, w["down"][e])
        y.index_add_(0, t, p[t, j, None] * o)
        err.index_add_(0, t, p[t, j, None] * (eo + 2.0 ** -19 * o.abs()))
    if gate is not None:
        sg = torch.sigmoid((xd @ gate.double()).to(x.dtype).double())[:, None]
        o, eo = ffn(xd, w["s_gate"], w["s_up"], w["s_down"])
        y += sg * o
        err += sg * (eo + 2.0 ** -19 * o.abs())
    tol = torch.finfo(x.dtype).eps / 2 * (y.abs() + err) + err + 1e-30
    off = (r["out"].double() - y).abs()
    assert (off <= tol).all(), float((off / tol).max())
    # and as a whole: bf16's own rounding is 2^-9 of a row in the mean square
    rel = (r["out"].double() - y).norm(dim=-1) / y.norm(dim=-1)
    assert (rel <= 2.0 ** -8).all(), float(rel.max())


def scaled(**factor):
    """Multiplies weights: name=(index, factor)."""
    def change(w):
        for key, (at, f) in factor.items():
            w[key][at] *= f
    return change


# d, weights changed
CHANGES = {
    "expert": scaled(gate=(3, 256.0), up=(3, 256.0)),
    "expert_1024": scaled(gate=(3, 1024.0), up=(3, 1024.0)),
    "small_expert": scaled(gate=(2, 2.0 ** -9), up=(2, 2.0 ** -9)),
    "gate_row": scaled(gate=((1, 17), 1024.0)),
    "row_pair": scaled(gate=((1, 17), 256.0), up=((1, 17), 256.0)),
    "rows_apart": scaled(gate=((1, 17), 500.0), up=((1, 40), 500.0)),
    "single_weights": scaled(gate=((4, 5, 7), 1000.0), up=((4, 5, 9), 50.0), s_gate=((3, 11), 1000.0), s_up=((3, 12), 1000.0)),
    "shared": scaled(s_gate=(slice(None), 256.0), s_up=(slice(None), 256.0)),
    "pruned": scaled(gate=((slice(None), slice(10, 20)), 0.0), up=((slice(None), slice(10, 20)), 0.0),
                     s_gate=(slice(0, 5), 0.0), s_up=(slice(0, 5), 0.0)),
}


@pytest.mark.parametrize("T", [1, 8, 24])
@pytest.mark.parametrize("d", [2048, 8192])
@pytest.mark.parametrize("change", list(CHANGES))
def test_weights_of_different_magnitudes(cuda, change, d, T):
    eng, w, router, gate, n = block(cuda, d, 6, 4, 200, 136, seed=d + T, change=CHANGES[change])
    x = n(T, d, std=1.0)
    check(_run(eng, x), x, w, router, gate, 4)


@pytest.mark.parametrize("T", [3, 16])
@pytest.mark.parametrize("factor", [2.0 ** -12, 4096.0])
def test_relu_expert_of_another_magnitude(cuda, factor, T):
    eng, w, router, gate, n = block(cuda, 768, 6, 1, 300, act="relu", seed=41, change=scaled(gate=(2, factor)))
    x = n(T, 768, std=1.0)
    check(_run(eng, x), x, w, router, gate, 1, top1=True)


@pytest.mark.parametrize("T", [2, 8, 31])
def test_one_large_channel_that_the_activation_silences(cuda, T):
    """A channel whose gate is strongly negative for every token leaves the row without its largest weights: the
    other channels keep their bits."""
    def change(w):
        w["gate"][:, 30] = -w["gate"][:, 30].abs() * 512
        w["up"][:, 30] *= 512

    eng, w, router, gate, n = block(cuda, 2048, 6, 4, 200, 136, seed=43, change=change)
    x = n(T, 2048, std=1.0).abs()
    check(_run(eng, x), x, w, router, gate, 4)


@pytest.mark.parametrize("T", [3, 12])
def test_scales_changed_in_place(cuda, T):
    """The bounds go with what the scales hold at the call, in a captured call too."""
    eng, w, router, gate, n = block(cuda, 512, 6, 2, 200, 136, seed=45)
    x = n(T, 512, std=1.0)
    check(_run(eng, x), x, w, router, gate, 2)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = eng.forward_few(x)
    for factor in (2.0 ** 14, 2.0 ** -28):
        eng.experts.w1_scale.mul_(factor)
        eng.experts.ws1_scale.mul_(factor)
        for key in ("gate", "up", "s_gate", "s_up"):
            w[key] = w[key] * factor
        check(_run(eng, x), x, w, router, gate, 2)
        g.replay()
        torch.cuda.synchronize()
        check(r, x, w, router, gate, 2)


@pytest.mark.parametrize("T", [3, 16])
@pytest.mark.parametrize("what", ["weight", "scale", "infinite_scale"])
def test_bad_weights_spoil_their_expert_alone(cuda, what, T):
    from dsca_moe_b200 import _lib as L
    from dsca_moe_b200.engine import MoEEngine

    eng, w, router, gate, n = block(cuda, 256, 12, 2, 100, 72, seed=46)
    x = n(T, 256, std=1.0)
    want = _run(eng, x)
    e = int(want["topk_ids"][0, 0])
    if what == "weight":
        eng.experts.w1.view(torch.uint8)[e, 3, 5] = 0x7F
    else:
        eng.experts.w1_scale[e, 3] = float("nan" if what == "scale" else "inf")
    eng = MoEEngine(router, eng.experts, top_k=2, route_mode=L.ROUTE_SOFTMAX_TOPK, shared_gate_weight=gate)
    r = _run(eng, x)
    hit = (want["topk_ids"] == e).any(-1)
    assert hit.any() and not hit.all()
    assert torch.equal(r["out"][~hit], want["out"][~hit])
    assert torch.isnan(r["out"][hit]).all(-1).all() or what == "infinite_scale"
    assert not torch.isfinite(r["out"][hit]).all(-1).any()
    eng.few_tokens = 32
    assert torch.equal(eng.forward(x)["out"][~hit], want["out"][~hit])


def test_an_engine_makes_no_copy_of_its_weights(cuda):
    from dsca_moe_b200 import _lib as L
    from dsca_moe_b200.engine import MoEEngine, pack_swiglu, quantize_fp8

    w, router, gate, n = _weights(cuda, 1024, 16, 512, 0, "swiglu", torch.bfloat16, 47)
    pe = quantize_fp8(pack_swiglu(w["gate"], w["up"], w["down"], device=cuda))
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    eng = MoEEngine(router, pe, top_k=2, route_mode=L.ROUTE_SOFTMAX_TOPK)
    assert torch.cuda.max_memory_allocated() - before < pe.w1.numel() // 8
    eng.forward_few(n(2, 1024))
    eng.check()


@pytest.mark.parametrize("T", [1, 5, 12, 32])
def test_tokens_of_zeros(cuda, T):
    """Rows that no value of the intermediate ever reaches any size in, alone and between others (a padded batch)."""
    eng, w, router, gate, n = block(cuda, 512, 12, 3, 200, 136, seed=48)
    x = n(T, 512, std=1.0)
    want = _run(eng, x)["out"].clone()
    x[T // 2:] = 0
    r = _run(eng, x)
    lg, ids, p = _route(x, router, 3, False, False)
    assert torch.equal(r["topk_ids"].long(), ids) and torch.equal(r["topk_w"], p)
    assert torch.equal(r["out"][:T // 2], want[:T // 2])
    assert (r["out"][T // 2:] == 0).all()
