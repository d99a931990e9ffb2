"""MoEEngine.forward_few (dsca_moe_few) against the block's definition in 64 bits.

Logits, expert ids and weights are compared bit for bit: the kernel sums the router's products in 64 bits,
and its softmax, ties and weights are those of the block's routing oracle.  Tolerance of out, propagated from the inputs' magnitudes: a product sum of K terms is off by at most
c * sum|terms|, c = (K / 8 + 32) * 2^-23 (a warp's chain is K / 8 / 16 tensor-core steps or K / 32 fused
multiply-adds, then 8 partial sums and the activation's few operations; 2^-23 a step covers an
accumulator that truncates).  The intermediate is held to 2^-17 of itself (two bf16
terms, 2^-9 * 2^-9 and the first's sign; with fp8 weights one f16 term: half a step of 11 significant bits is
2^-11 of the value), |silu'| <= 1.1, the gate and the weighted products are off by 2^-19, and out is
rounded once: eps / 2 of its type, relative."""
import pytest
import torch

from oracle import oracle as O

pytestmark = pytest.mark.gpu

H_EPS = {"bf16": 2.0 ** -17, "f32": 2.0 ** -17, "fp8": torch.finfo(torch.float16).eps / 2}


def _weights(dev, d, E, I, Is, act, dtype, seed, std=0.03):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def n(*s, std=std):
        return (torch.randn(*s, generator=g, device=dev) * std).to(dtype)

    if act == "swiglu":
        w = dict(gate=n(E, I, d), up=n(E, I, d), down=n(E, d, I))
    else:
        w = dict(gate=n(E, I, d), down=n(E, d, I))
    if Is:
        w.update(s_gate=n(Is, d), s_up=n(Is, d), s_down=n(d, Is))
    return w, n(E, d, std=d ** -0.5), n(d, std=d ** -0.5) if Is else None, n


def _engine(dev, d, E, k, I, Is=0, act="swiglu", kind="bf16", norm=False, seed=1):
    """(engine, the weights it computes with in fp64, router rows, gate row, generator)."""
    from dsca_moe_b200 import _lib as L
    from dsca_moe_b200.engine import MoEEngine, pack_relu, pack_swiglu, quantize_fp8

    dtype = torch.float32 if kind == "f32" else torch.bfloat16
    w, router, gate, n = _weights(dev, d, E, I, Is, act, dtype, seed)
    if act == "swiglu":
        pe = pack_swiglu(w["gate"], w["up"], w["down"], shared=(w["s_gate"], w["s_up"], w["s_down"]) if Is else None,
                         dtype=dtype, device=dev)
    else:
        pe = pack_relu(w["gate"], w["down"], dtype=dtype, device=dev)
    w64 = {key: v.double() for key, v in w.items()}
    w64["h_eps"] = H_EPS[kind]
    if kind == "fp8":
        pe = quantize_fp8(pe)
        for key, v in w.items():
            amax = v.float().abs().amax(-1, keepdim=True)
            s = torch.where(amax > 0, amax / 448.0, torch.ones_like(amax))
            w64[key] = (v.float() / s).to(torch.float8_e4m3fn).double() * s.double()
    eng = MoEEngine(router, pe, top_k=k, route_mode=L.ROUTE_SOFTMAX_TOPK if act == "swiglu" else L.ROUTE_SWITCH_TOP1,
                    norm_topk=norm, shared_gate_weight=gate)
    return eng, w64, router, gate, n


def _route(x, router, k, top1, norm):
    """Logits rounded from their 64-bit sums; the choice and the weights by the oracle, bit for bit."""
    lg = (x.double() @ router.double().T).to(x.dtype)
    act, host = "bf16" if x.dtype == torch.bfloat16 else "f32", lg.float().cpu().numpy()
    if top1:
        ids, p = O.route_top1(host, act)
        ids, p = ids[:, None], p[:, None]
    else:
        ids, p = O.route_topk(host, k, norm, act)
    return lg, torch.from_numpy(ids).long().to(x.device), torch.from_numpy(p).to(x.device)


def _ffn(x, gate, up, down, h_eps):
    """(result, its error bound before the last rounding) of one expert on rows x, in 64 bits."""
    d, I = gate.shape[1], gate.shape[0]
    c1, c2 = (d / 8 + 32) * 2.0 ** -23, (I / 8 + 32) * 2.0 ** -23
    g, eg = x @ gate.T, c1 * (x.abs() @ gate.abs().T)
    if up is None:
        h, eh = g.clamp_min(0), eg
    else:
        u, eu = x @ up.T, c1 * (x.abs() @ up.abs().T)
        s = g * torch.sigmoid(g)
        h, eh = s * u, 1.1 * eg * (u.abs() + eu) + s.abs() * eu
    eh = eh + h_eps * h.abs()
    return h @ down.T, eh @ down.abs().T + c2 * (h.abs() @ down.abs().T)


def _check(r, x, w, router, gate, k, top1=False, norm=False):
    lg, ids, p = _route(x, router, k, top1, norm)
    assert torch.equal(r["logits"], lg)
    assert torch.equal(r["topk_ids"].long(), ids)
    assert torch.equal(r["expert_index"], ids[:, 0])
    assert torch.equal(r["topk_w"], p)
    xd, p = x.double(), p.double()
    y, err = torch.zeros_like(xd), torch.zeros_like(xd)
    for e in ids.unique().tolist():
        t, j = (ids == e).nonzero(as_tuple=True)
        o, eo = _ffn(xd[t], w["gate"][e], w["up"][e] if "up" in w else None, w["down"][e], w["h_eps"])
        y.index_add_(0, t, p[t, j, None] * o)
        err.index_add_(0, t, p[t, j, None] * (eo + 2.0 ** -19 * o.abs()))
    if gate is not None:
        sg = torch.sigmoid((xd @ gate.double()).to(x.dtype).double())[:, None]
        o, eo = _ffn(xd, w["s_gate"], w["s_up"], w["s_down"], w["h_eps"])
        y += sg * o
        err += sg * (eo + 2.0 ** -19 * o.abs())
    tol = torch.finfo(x.dtype).eps / 2 * (y.abs() + err) + err + 1e-30
    off = (r["out"].double() - y).abs()
    assert (off <= tol).all(), float((off / tol).max())


def _run(eng, x):
    r = eng.forward_few(x)
    torch.cuda.synchronize()
    eng.check()
    return r


@pytest.mark.parametrize("kind", ["bf16", "fp8", "f32"])
@pytest.mark.parametrize("T,d,E,k,I,Is", [(1, 64, 4, 2, 32, 64), (1, 2048, 16, 4, 136, 520), (2, 16, 5, 1, 1, 0),
                                          (7, 208, 60, 4, 101, 77), (8, 512, 63, 8, 64, 8), (9, 320, 64, 8, 250, 0),
                                          (16, 768, 13, 3, 333, 901), (17, 1040, 60, 4, 96, 129), (31, 128, 8, 8, 40, 40),
                                          (32, 2560, 30, 4, 200, 300), (5, 4096, 6, 2, 72, 0), (3, 48, 2, 2, 700, 15)])
def test_swiglu(cuda, T, d, E, k, I, Is, kind):
    norm = (T + k) % 2 == 0
    eng, w, router, gate, n = _engine(cuda, d, E, k, I, Is, kind=kind, norm=norm, seed=T + d)
    x = n(T, d, std=1.0)
    _check(_run(eng, x), x, w, router, gate, k, norm=norm)


@pytest.mark.parametrize("kind", ["bf16", "fp8", "f32"])
@pytest.mark.parametrize("T,d,E,k,I,Is", [(3, 5120, 6, 2, 72, 40), (12, 5120, 6, 2, 72, 40), (24, 8192, 4, 2, 40, 16),
                                          (16, 256, 2, 1, 4096, 0), (32, 512, 3, 2, 3000, 1000), (20, 1152, 40, 3, 500, 0), (9, 2304, 5, 2, 300, 100),
                                          (32, 1200, 2, 1, 900, 300), (28, 4096, 12, 4, 150, 70),
                                          (2, 16384, 3, 2, 24, 8), (11, 16384, 3, 1, 24, 0), (4, 64, 4, 2, 20000, 9000)])
def test_swiglu_long_rows_and_many_units(cuda, T, d, E, k, I, Is, kind):
    """Rows of more boxes than a warp keeps values of; consecutive units of one expert, with at most eight
    tokens and with more, and of the next one."""
    eng, w, router, gate, n = _engine(cuda, d, E, k, I, Is, kind=kind, seed=T + d)
    x = n(T, d, std=1.0)
    _check(_run(eng, x), x, w, router, gate, k)


@pytest.mark.parametrize("kind", ["bf16", "fp8", "f32"])
@pytest.mark.parametrize("T,d,E,F", [(1, 768, 64, 512), (6, 64, 3, 17), (16, 768, 64, 1000), (32, 272, 10, 2048)])
def test_switch(cuda, T, d, E, F, kind):
    eng, w, router, gate, n = _engine(cuda, d, E, 1, F, act="relu", kind=kind, seed=T + d)
    x = n(T, d, std=1.0)
    _check(_run(eng, x), x, w, router, gate, 1, top1=True)


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("T", [1, 4, 20])
def test_qwen_block(cuda, T, kind):
    """The full-size block, several calls on one workspace."""
    d, E, k, I, Is = 2048, 60, 4, 1408, 5632
    eng, w, router, gate, n = _engine(cuda, d, E, k, I, Is, kind=kind, seed=T)
    for _ in range(3):
        x = n(T, d, std=1.0)
        _check(_run(eng, x), x, w, router, gate, k)


@pytest.mark.parametrize("T", [8, 32])
def test_all_tokens_on_the_same_experts(cuda, T):
    eng, w, router, gate, n = _engine(cuda, 256, 20, 3, 120, 64, seed=3)
    x = n(1, 256, std=1.0).expand(T, 256).contiguous()
    r = _run(eng, x)
    _check(r, x, w, router, gate, 3)
    assert (r["out"] == r["out"][0]).all()


def test_ties_take_the_lowest_ids(cuda):
    eng, w, router, gate, n = _engine(cuda, 128, 40, 4, 64, seed=4)
    for x in (torch.zeros(3, 128, dtype=torch.bfloat16, device=cuda), n(3, 128, std=1.0)):
        eng.router_weight[7] = eng.router_weight[3]
        eng.router_weight[33] = eng.router_weight[3]
        _check(_run(eng, x), x, w, eng.router_weight, gate, 4)


@pytest.mark.parametrize("kind", ["bf16", "fp8", "f32"])
@pytest.mark.parametrize("T", [6, 18])
def test_bad_values_stay_in_their_row(cuda, kind, T):
    eng, w, router, gate, n = _engine(cuda, 256, 12, 2, 100, 72, kind=kind, seed=5)
    x = n(T, 256, std=1.0)
    want = _run(eng, x)["out"].clone()
    x[1, 3], x[4, 200] = float("nan"), float("inf")
    r = _run(eng, x)
    keep = [0, 2, 3, 5] + list(range(6, T))
    assert torch.equal(r["out"][keep], want[keep])
    assert not torch.isfinite(r["out"][[1, 4]]).all(-1).any()
    assert ((r["topk_ids"] >= 0) & (r["topk_ids"] < 12)).all()


@pytest.mark.parametrize("kind", ["bf16", "fp8", "f32"])
@pytest.mark.parametrize("T", [8, 24])
def test_large_and_small_magnitudes(cuda, kind, T):
    """Rows from 2^-30 to 2^30: each is held to its own size."""
    eng, w, router, gate, n = _engine(cuda, 256, 12, 2, 100, 72, kind=kind, seed=6)
    x = n(T, 256, std=1.0) * torch.exp2(torch.arange(-30, 31, 8, device=cuda).float()).repeat(3)[:T, None]
    x = x.to(eng.dtype)
    _check(_run(eng, x), x, w, router, gate, 2)


@pytest.mark.parametrize("kind", ["bf16", "fp8", "f32"])
def test_agrees_with_forward_and_is_repeatable(cuda, kind):
    """The same routing as the block's other path where the logits are not on a rounding border, outputs
    within the bf16 tolerance of the block's other tests; bit-equal from call to call."""
    eng, w, router, gate, n = _engine(cuda, 512, 60, 4, 384, 768, kind=kind, seed=7)
    x = n(32, 512, std=1.0)
    a, b = _run(eng, x), eng.forward(x)
    same = (a["topk_ids"] == b["topk_ids"]).all(-1)
    assert same.sum() >= 31
    ao, bo = a["out"][same].float(), b["out"][same].float()
    assert ((ao - bo).abs().max() / bo.abs().max()) < 2e-2
    c = _run(eng, x)
    for key in ("out", "topk_w", "topk_ids", "logits"):
        assert torch.equal(c[key], a[key])
    # the choice of experts does not depend on how many tokens a call has, nor a token's result on the
    # others' values
    for T in (9, 1):
        c = _run(eng, x[:T])
        _check(c, x[:T], w, router, gate, 4)
        for key in ("topk_w", "topk_ids", "logits"):
            assert torch.equal(c[key], a[key][:T])
    y = n(32, 512, std=1.0)
    y[5] = x[5]
    assert torch.equal(_run(eng, y)["out"][5], a["out"][5])


def test_input_forms(cuda):
    """Strided, unaligned and fp32 inputs, and no token at all."""
    eng, w, router, gate, n = _engine(cuda, 256, 12, 2, 100, 72, seed=8)
    x = n(6, 256, std=1.0)
    want = _run(eng, x)
    wide = torch.zeros(6, 300, dtype=torch.bfloat16, device=cuda)
    wide[:, 1:257] = x
    for y in (wide[:, 1:257], x.t().contiguous().t(), x.float(), wide.view(-1)[1:257][None]):
        r = _run(eng, y)
        assert torch.equal(r["out"], want["out"][:y.shape[0]]) and torch.equal(r["topk_ids"], want["topk_ids"][:y.shape[0]])
    e = eng.forward_few(x[:0])
    assert e["out"].shape == (0, 256) and e["topk_ids"].shape == (0, 2)


def test_refusals(cuda):
    from dsca_moe_b200 import _lib as L
    from dsca_moe_b200.engine import MoEEngine, pack_swiglu, quantize_fp8

    eng, w, router, gate, n = _engine(cuda, 64, 4, 2, 32, seed=9)
    for bad in (n(33, 64), n(4, 56), n(4, 64)[None], n(4, 64).cpu()):
        with pytest.raises(ValueError):
            eng.forward_few(bad)
    pe = quantize_fp8(pack_swiglu(n(4, 32, 72), n(4, 32, 72), n(4, 72, 32), device=cuda))
    odd = MoEEngine(n(4, 72), pe, top_k=2, route_mode=L.ROUTE_SOFTMAX_TOPK)
    with pytest.raises(ValueError, match="16 bytes"):
        odd.forward_few(n(4, 72))
    host = MoEEngine(n(4, 64), pack_swiglu(n(4, 32, 64), n(4, 32, 64), n(4, 64, 32), device="cpu"), top_k=2,
                     route_mode=L.ROUTE_SOFTMAX_TOPK, cache_slots=2, device=cuda)
    with pytest.raises(ValueError, match="resident"):
        host.forward_few(n(4, 64))


def test_streams_and_graphs(cuda):
    """Calls on two streams at once (a workspace each), and two captured graphs replayed on two streams
    at once, against the same calls one after the other."""
    eng, w, router, gate, n = _engine(cuda, 1024, 60, 4, 512, 1024, seed=10)
    xs = [n(T, 1024, std=1.0) for T in (3, 12)]
    want = [_run(eng, x)["out"].clone() for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (s, x) in enumerate(zip(streams, xs)):
            with torch.cuda.stream(s):
                got[i].append(eng.forward_few(x)["out"])
    torch.cuda.synchronize()
    eng.check()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])
    graphs, outs, ins = [], [], [torch.zeros_like(x) for x in xs]
    for x in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(eng.forward_few(x)["out"])
            outs[-1] = eng.forward_few(x)["out"]
        graphs.append(g)
    for x, b in zip(xs, ins):
        b.copy_(x)
    torch.cuda.synchronize()
    for _ in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        eng.check()
        assert all(torch.equal(o, v) for o, v in zip(outs, want))


def test_64_experts_and_a_shared_one_are_refused(cuda):
    """One logit more than the router holds."""
    eng, w, router, gate, n = _engine(cuda, 128, 64, 4, 64, 64, seed=13)
    with pytest.raises(ValueError):
        eng.forward_few(n(4, 128))


def test_forward_takes_it_below_few_tokens(cuda):
    """few_tokens switches forward(), capture() and the layers over; forward_normed is the norm and then
    the block."""
    from dsca_moe_b200 import add_rms_norm

    eng, w, router, gate, n = _engine(cuda, 512, 16, 4, 256, 128, seed=11)
    x, res, nw = n(8, 512, std=1.0), n(8, 512, std=3.0), 1 + n(512, std=0.2)
    few = _run(eng, x)["out"]
    plain = eng.forward(x)
    assert "token_row" in plain
    eng.few_tokens = 8
    assert torch.equal(eng.forward(x)["out"], few) and "token_row" not in eng.forward(x)
    assert "token_row" in eng.forward(n(9, 512))
    graph = eng.capture(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(graph.out, few)
    y = add_rms_norm(x, nw, 1e-6, res)
    r = eng.forward_normed(x, nw, 1e-6, res)
    torch.cuda.synchronize()
    eng.check()
    assert torch.equal(r["normed"], y.y) and torch.equal(r["residual"], y.residual)
    assert torch.equal(r["out"], eng.forward_few(y.y)["out"])
    _check({key: r[key] for key in ("out", "logits", "topk_ids", "topk_w", "expert_index")}, y.y, w, router, gate, 4)


def test_error_word_is_reported_and_workspaces_dropped(cuda):
    """An error word (as a wait that gave up writes it) raises at check() and drops the workspaces, whose
    counters may be anything then; the calls behind it are right again."""
    eng, w, router, gate, n = _engine(cuda, 256, 12, 2, 100, 72, seed=12)
    x = n(4, 256, std=1.0)
    want = _run(eng, x)["out"].clone()
    eng.err.fill_(1)
    from dsca_moe_b200._lib import DscaError
    with pytest.raises(DscaError):
        eng.check()
    assert eng._few_ws == {}
    assert torch.equal(_run(eng, x)["out"], want)
