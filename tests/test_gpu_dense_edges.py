"""Dense blocks and 8-bit products at the edges of what their descriptions allow, against their definitions in 64 bits."""
import pytest
import torch

import dense_ref as R

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _randn(dev, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return lambda *shape: torch.randn(*shape, generator=g, device=dev)


@pytest.mark.parametrize("T,k,n", [(9, 2048, 8250), (12, 2048, 8250), (16, 4096, 4130), (33, 256, 320), (48, 144, 512),
                                   (49, 256, 1000), (97, 512, 264), (100, 320, 777), (112, 256, 2000), (130, 128, 264), (259, 640, 520)])
def test_int8_partial_tiles(cuda, T, k, n):
    """8-bit tiles whose last 32 columns are not full: few tokens on weights of more than 16 MB, token counts just past
    a multiple of 32 or 16, and columns of many tokens that end so."""
    from dsca_moe_b200 import check_dense, int8_linear, pack_int8, quantize_rows

    randn = _randn(cuda, T + k + n)
    x, w = randn(T, k).to(BF16), pack_int8(randn(n, k).to(BF16))
    q, s = quantize_rows(x)
    R.close(int8_linear(x, w), R.int8_linear(q, s, w.q, w.scale, BF16))
    check_dense()


def _ffn_int8_defined(x, wg, wu, wd, name):
    """(value, bound) of the block on fp32 tokens with the codes of the intermediate in 64 bits and no allowance at their borders.
    The row's largest is off by 16 units of 2^-24 at most (the gate's exponential 5, 1 + e 1, its reciprocal 2, their product 1, the
    product with g 2, u 4, h 1) where no code hangs on it, its scale rounds once; the sum's conversion and two products 3."""
    q, s = R.codes(x.double())
    g, u = ((q @ w.q.double().T) * s[:, None] * w.scale.double() for w in (wg, wu))
    hq, hs = R.codes(R.act(g, name)[0] * u)
    y = (hq @ wd.q.double().T) * hs[:, None] * wd.scale.double()
    return y, 20.1 * 2.0 ** -24 * y.abs()


@pytest.mark.parametrize("name", R.ACTS)
@pytest.mark.parametrize("T,d,I", [(1, 2048, 5632), (1, 8, 3), (7, 264, 1021), (12, 768, 2048), (16, 1000, 520), (24, 2048, 1408), (40, 512, 2050),
                                   (128, 320, 264), (300, 777, 1000), (2800, 2000, 843), (1500, 256, 2056), (5000, 64, 520),
                                   (3, 64, 9001), (700, 40, 8300), (1300, 2048, 5632), (900, 520, 1000)])
def test_int8_block_codes_of_f32_tokens(cuda, T, d, I, name):
    """fp32 tokens: every code of the intermediate is that of the 64-bit definition (a single one on the other side of its
    border moves some of that token's y by many of the bounds)."""
    from dsca_moe_b200 import check_dense, gated_ffn_int8, pack_int8

    randn = _randn(cuda, T + d + I)
    x = randn(T, d) * torch.exp(0.3 * randn(T, 1))
    wg, wu, wd = (pack_int8(randn(*s) * s[1] ** -0.5) for s in ((I, d), (I, d), (d, I)))
    R.close(gated_ffn_int8(x, wg, wu, wd, act=name), _ffn_int8_defined(x, wg, wu, wd, name))
    check_dense()


@pytest.mark.parametrize("T", [2, 30, 300])
def test_int8_block_of_f32_tokens_range(cuda, T):
    """Gates far from zero, rows of every size, a row of zeros, rows that are not finite beside rows that are; the same call
    again gives the same bits."""
    from dsca_moe_b200 import gated_ffn_int8, pack_int8

    randn = _randn(cuda, T)
    wg, wu, wd = (pack_int8(randn(*s)) for s in ((200, 136), (200, 136), (136, 200)))
    x = randn(T, 136) * 10 ** torch.linspace(-9, 6, T, device=cuda)[:, None]
    x[T // 2] = 0
    for name in R.ACTS:
        y = gated_ffn_int8(x, wg, wu, wd, act=name)
        R.close(y, _ffn_int8_defined(x, wg, wu, wd, name), name)
        assert not y[T // 2].any() and torch.equal(y, gated_ffn_int8(x, wg, wu, wd, act=name))
        for bad in (float("nan"), float("inf")):
            xb = x.clone()
            xb[T // 2, 3] = bad
            got, keep = gated_ffn_int8(xb, wg, wu, wd, act=name), torch.arange(T, device=cuda) != T // 2
            assert not torch.isfinite(got[T // 2]).any() and torch.equal(got[keep], y[keep])


def test_int8_block_of_f32_tokens_captured(cuda):
    """Captured, with new tokens in the buffers at each replay; and a batch in front, rows of a wider buffer."""
    from dsca_moe_b200 import gated_ffn_int8, pack_int8

    randn = _randn(cuda, 0)
    w = [pack_int8(randn(*s) * s[1] ** -0.5) for s in ((264, 128), (264, 128), (128, 264))]
    x = randn(2, 20, 133)[..., :128]
    gated_ffn_int8(x, *w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = gated_ffn_int8(x, *w)
    for _ in range(3):
        x.copy_(randn(2, 20, 128))
        graph.replay()
        R.close(y.view(40, 128), _ffn_int8_defined(x.reshape(40, 128), *w, "silu"))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,d,I,gap", [(3, 40, 24, 8), (40, 96, 136, 16), (150, 136, 264, 8), (300, 130, 66, 3)])
def test_saved_tensor_hooks(cuda, T, d, I, gap, dtype):
    """Hooks that return what was saved in other strides (offloading to the host lays it out densely): rows of wider buffers
    keep their gradients."""
    from dsca_moe_b200 import gated_ffn

    randn = _randn(cuda, T)
    x, wg, wu, wd = ((randn(r, c + gap) * c ** -0.5).to(dtype)[:, :c] for r, c in ((T, d), (I, d), (I, d), (d, I)))
    dy = randn(T, d).to(dtype)
    ref = R.ffn(x, wg, wu, wd, "silu", dtype, dy)

    def transposed(t):
        return t.t().contiguous().t() if t.dim() == 2 else t

    for hooks in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t),
                  torch.autograd.graph.saved_tensors_hooks(lambda t: t, transposed)):
        p = [t.detach().requires_grad_() for t in (x, wg, wu, wd)]
        with hooks:
            y = gated_ffn(*p)
        for got, k in zip(torch.autograd.grad(y, p, dy), ("dx", "d_gate", "d_up", "d_down")):
            R.close(got, ref[k], k)
    for change in (lambda t: t[..., :-1], lambda t: t.double() if t.is_floating_point() else t):
        p = [t.detach().requires_grad_() for t in (x, wg, wu, wd)]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            y = gated_ffn(*p)
        with pytest.raises(RuntimeError, match="came back"):
            y.backward(dy)


def _mlp(dev, dtype, d=64, inter=200):
    class M(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.gate_proj, self.up_proj = torch.nn.Linear(d, inter, bias=False), torch.nn.Linear(d, inter, bias=False)
            self.down_proj, self.act_fn = torch.nn.Linear(inter, d, bias=False), torch.nn.SiLU()

    torch.manual_seed(3)
    return M().to(dev, dtype)


def test_module_under_autocast(cuda):
    """fp32 parameters under bf16 autocast: the block on bf16 values, gradients in the parameters' type; fp16 autocast runs the
    layers."""
    from dsca_moe_b200 import GatedFFN, pack_int8

    m = GatedFFN(_mlp(cuda, F32))
    randn = _randn(cuda, 5)
    w = [m.gate_proj.weight, m.up_proj.weight, m.down_proj.weight]
    for dtype in (BF16, F32):
        x, dy = randn(70, 64).to(dtype).requires_grad_(), randn(70, 64).to(BF16)
        ref = R.ffn(x.detach().to(BF16), *(t.detach().to(BF16) for t in w), "silu", BF16, dy)
        with torch.autocast("cuda", torch.bfloat16):
            y = m(x)
        assert y.dtype == BF16
        R.close(y.detach(), ref["y"])
        for got, p, k in zip(torch.autograd.grad(y, [x] + w, dy), [x] + w, ("dx", "d_gate", "d_up", "d_down")):
            assert got.dtype == p.dtype
            R.close(got, ref[k], k)
    with torch.autocast("cuda", torch.float16):
        assert m(x).dtype == torch.float16
    q = GatedFFN(_mlp(cuda, F32), int8=True)
    with torch.autocast("cuda", torch.bfloat16):
        y = q(x.detach())
    R.close(y, R.ffn_int8(x.detach().to(BF16), *(pack_int8(t) for t in w), "silu", BF16))


def test_t5_block_in_eval_mode(cuda):
    """T5's gated MLP with its dropout off runs as the block; on 8-bit weights a dropout that is on is refused."""
    from transformers import T5Config
    from transformers.models.t5.modeling_t5 import T5DenseGatedActDense

    from dsca_moe_b200 import GatedFFN

    torch.manual_seed(2)
    old = T5DenseGatedActDense(T5Config(d_model=64, d_ff=200, feed_forward_proj="gated-gelu")).to(cuda, BF16)
    x = _randn(cuda, 8)(40, 64).to(BF16)
    m = GatedFFN(old.eval())
    ref = R.ffn(x, old.wi_0.weight.detach(), old.wi_1.weight.detach(), old.wo.weight.detach(), "gelu", BF16)
    R.close(m(x).detach(), ref["y"])
    q = GatedFFN(old, int8=True)
    q(x)
    with pytest.raises(RuntimeError, match="dropout"):
        q.train()(x)


def test_patched_model_refuses_gradients_through_moe_blocks(cuda):
    """A model whose MoE blocks are swapped: logits with autograd on are those without it, a loss that would reach a layer
    through a block raises, and what lies behind the last block trains."""
    from test_gpu_dense import _tiny_qwen

    from dsca_moe_b200 import patch

    m = _tiny_qwen()
    patch(m, 0, 1, dense_ffn="same")
    ids = torch.randint(0, 97, (2, 11), device=cuda)
    with torch.no_grad():
        want = m(ids).logits
    y = m(ids).logits
    assert torch.equal(y, want)
    with pytest.raises(RuntimeError, match="MoE block"):
        y.float().square().mean().backward()
    m.requires_grad_(False)
    m.lm_head.weight.requires_grad_()
    y = m(ids).logits
    (grad,) = torch.autograd.grad(y.float().square().mean(), m.lm_head.weight)
    assert grad.abs().sum() > 0


def test_calls_without_gradients(cuda):
    """8-bit calls on what wants a gradient: the values of a call without autograd, and an error from the backward pass that
    reaches them; forward-mode tangents are refused by every call."""
    import torch.autograd.forward_ad as fwad

    from dsca_moe_b200 import GatedFFN, gated_ffn, gated_ffn_int8, int8_linear, pack_int8, quantize_rows

    m = GatedFFN(_mlp(cuda, BF16), int8=True)
    randn = _randn(cuda, 6)
    lin = torch.nn.Linear(64, 64, bias=False).to(cuda, BF16)
    x, w = randn(5, 64).to(BF16), [pack_int8(randn(*s).to(BF16)) for s in ((200, 64), (200, 64), (64, 200))]
    bias = randn(200).to(BF16).requires_grad_()
    q, s = quantize_rows(x)
    for name, call in (("gated_ffn_int8", lambda t: t + m(t)), ("gated_ffn_int8", lambda t: gated_ffn_int8(t, *w)),
                       ("int8_linear", lambda t: int8_linear(t, w[0])), ("quantize_rows", lambda t: quantize_rows(t)[1]),
                       ("int8_linear", lambda t: int8_linear(q, w[0], bias=bias, x_scale=s)),
                       ("int8_linear", lambda t: int8_linear(q, w[0], x_scale=quantize_rows(t)[1]))):
        y = call(lin(x))
        with torch.no_grad():
            assert torch.equal(call(lin(x)), y)
        with pytest.raises(RuntimeError, match=name + " has no backward"):
            y.float().sum().backward()
        call(lin(x).detach())
    assert not pack_int8(lin.weight).scale.requires_grad
    wg, wd = randn(200, 64).to(BF16), randn(64, 200).to(BF16)
    with fwad.dual_level():
        t = fwad.make_dual(x, x)
        for call in (lambda: gated_ffn(t, wg, wg, wd), lambda: gated_ffn(x, wg, fwad.make_dual(wg, wg), wd), lambda: quantize_rows(t),
                     lambda: int8_linear(t, w[0]), lambda: gated_ffn_int8(t, *w)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        gated_ffn(x, wg, wg, wd)


@pytest.mark.parametrize("rows", [1, 2, 8, 12, 16, 17, 40, 200])
@pytest.mark.parametrize("k", [1, 15, 50, 63, 64, 113, 1000])
def test_codes_and_weights_of_wider_ones(cuda, rows, k):
    """Codes and weights that are both views of wider ones: what lies behind the k-th column counts for no number of rows."""
    from dsca_moe_b200 import Int8Weight, gated_ffn_int8, int8_linear, pack_int8, quantize_rows

    randn = _randn(cuda, rows + k)
    q, s = quantize_rows(randn(rows, 1040).to(BF16))
    w = pack_int8(randn(96, 1040).to(BF16))
    part = Int8Weight(w.q[:, :k], w.scale)
    for n in (0, rows - 1):  # one row alone as well
        R.close(int8_linear(q[n:n + 1, :k], part, x_scale=s[n:n + 1]), R.int8_linear(q[n:n + 1, :k], s[n:n + 1], part.q, w.scale, BF16))
    R.close(int8_linear(q[:, :k], part, x_scale=s), R.int8_linear(q[:, :k], s, part.q, w.scale, BF16))
    R.close(int8_linear(q[0, :k], part, x_scale=s[0])[None], R.int8_linear(q[:1, :k], s[:1], part.q, w.scale, BF16))
    x = randn(rows, k)
    down = pack_int8(randn(k, 96))
    R.close(gated_ffn_int8(x, part, part, down), _ffn_int8_defined(x, part, part, down, "silu"))
    wide = pack_int8(randn(96, k + 200))
    x = randn(rows, 96)
    up, down = pack_int8(randn(k, 96)), Int8Weight(wide.q[:, :k], wide.scale)
    R.close(gated_ffn_int8(x, up, up, down), _ffn_int8_defined(x, up, up, down, "silu"))


@pytest.mark.parametrize("T", [1, 12, 40, 300])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_int8_scales_of_every_size(cuda, T, dtype):
    """Rows and weights so small or large that the product of their two scales is no normal number while the result is."""
    from dsca_moe_b200 import gated_ffn_int8, int8_linear, pack_int8, quantize_rows

    randn = _randn(cuda, T)
    for sx, sw in ((2.0 ** -112, 2.0 ** -10), (2.0 ** -90, 2.0 ** -30), (2.0 ** 100, 2.0 ** 20), (2.0 ** 120, 2.0 ** -60), (2.0 ** -100, 2.0 ** 80)):
        x, w = (randn(T, 264) * sx).to(dtype), pack_int8((randn(136, 264) * sw).to(dtype))
        q, s = quantize_rows(x)
        R.close(int8_linear(x, w), R.int8_linear(q, s, w.q, w.scale, dtype), (sx, sw))
        # gate and up of some 2^-20 to 2^0 each: their sums stay normal numbers while the scales' products do not
        up, down = pack_int8((randn(136, 264) * 2.0 ** -8 / sx).to(dtype)), pack_int8(randn(264, 136).to(dtype))
        if 2.0 ** -8 / sx < 2.0 ** 90:
            R.close(gated_ffn_int8(x, up, up, down, act="relu"), R.ffn_int8(x, up, up, down, "relu", dtype), sx)


@pytest.mark.parametrize("T", [1, 12, 40, 300])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_int8_products_of_subnormal_scales(cuda, T, dtype):
    """Scales whose product, near 1e-42, has some ten bits left; the results are normal numbers (all terms of one sign)."""
    from dsca_moe_b200 import int8_linear, pack_int8, quantize_rows

    randn = _randn(cuda, T)
    for sx, sw in ((2.0 ** -115, 2.0 ** -10), (2.0 ** -105, 2.0 ** -20), (2.0 ** -60, 2.0 ** -65), (2.0 ** -5, 2.0 ** -120)):
        x, w = (randn(T, 264).abs() * sx).to(dtype), pack_int8((randn(136, 264).abs() * sw).to(dtype))
        q, s = quantize_rows(x)
        v, e = R.int8_linear(q, s, w.q, w.scale, dtype)
        assert v.min() > 2.0 ** -126 and (s[0].double() * w.scale[0].double()) < 2.0 ** -130
        assert ((int8_linear(x, w).double() - v).abs() <= e + 2.0 ** -149).all(), (sx, sw)


@pytest.mark.parametrize("T", [65536, 65536 * 2 + 1, 900000, 3000001])
def test_weight_gradients_of_many_tokens(cuda, T):
    """Sums of one sign over many tokens, whose terms are exact, so that only the sum's own additions and the final rounding
    count.  An accumulator takes 65536 tokens in steps of 16 at most: 4096 additions cut off at 2^-23 of the running sum, which is
    half the final one on average, 2^-12 of the sum; twice that for what is cut off inside a step."""
    from dsca_moe_b200 import check_dense, gated_ffn

    d = I = 64
    g = torch.Generator(device=cuda)
    g.manual_seed(1)
    top = torch.linspace(2, 64, 32, device=cuda).round()  # columns of different means
    a = 1 + (torch.rand(T, 32, generator=g, device=cuda) * (top + 1)).floor().clamp_max(64) / 64
    x = torch.cat([a, 4 - a], 1).to(BF16)  # a row's sum is 128: with weights of 1 / 128 g = u = 1
    c = (1 + torch.randint(0, 128, (T, 1), generator=g, device=cuda) / 128).to(BF16)
    wg, wu = (torch.full((I, d), 1 / 128, dtype=BF16, device=cuda, requires_grad=True) for _ in range(2))
    wd = torch.full((d, I), 1 / I, dtype=BF16, device=cuda, requires_grad=True)
    y = gated_ffn(x, wg, wu, wd, act="relu")
    assert (y == 1).all()
    got = torch.autograd.grad(y, (wg, wu, wd), c.expand(T, d).contiguous())
    ref = sum((x[i:i + 500000].double() * c[i:i + 500000].double()).sum(0) for i in range(0, T, 500000))  # dh = dg = du = c, h = 1
    for v, r in zip(got, (ref.expand(I, d), ref.expand(I, d), c.double().sum().expand(d, I))):
        half = 2.0 ** (torch.floor(torch.log2(r)) - 8)
        assert ((v.double() - r).abs() <= half + 2.0 ** -11 * r).all(), float(((v.double() - r) / r).abs().max())
    check_dense()


def test_error_word_is_there_before_its_address_is(cuda, monkeypatch):
    """The word's zeros have landed when the first call gets its address, whatever its stream was busy with: a call on another
    stream may record an error at once."""
    import dsca_moe_b200.dense as D

    monkeypatch.setattr(D, "_ERR", {})
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        torch.zeros(64, dtype=torch.int32, device=cuda)  # its memory is at hand: no allocation that waits by itself
        torch.cuda._sleep(400_000_000)
        D._err(torch.device("cuda", torch.cuda.current_device()))
        assert stream.query()


@pytest.mark.parametrize("T,inter", [(3, 40), (5, 1300), (700, 40)])
def test_int8_block_of_f32_tokens_equal_and_tiny_values(cuda, T, inter):
    """Rows whose values are all the largest, or all on a border of two codes, or all below fp32's normal numbers in between."""
    from dsca_moe_b200 import Int8Weight, gated_ffn_int8, pack_int8

    randn = _randn(cuda, T)
    down = pack_int8(randn(64, inter))
    x = randn(T, 64)
    same = pack_int8(torch.ones(inter, 64, device=cuda))
    R.close(gated_ffn_int8(x, same, same, down), _ffn_int8_defined(x, same, same, down, "silu"))
    # u = 1 and g from 1 to 127 half steps of the largest: 127 h / max|h| = n + 1 / 2 for odd ones
    q = torch.zeros(inter, 64, dtype=torch.int8, device=cuda)
    q[:, 0] = torch.arange(inter, device=cuda) % 127 + 1
    ones = torch.ones(inter, device=cuda)
    x = torch.zeros(T, 64, device=cuda)
    x[:, 0] = 1
    q2 = q.clone()
    q2[:, 0] = 1
    q[0, 0] = 127
    half = torch.where(torch.arange(inter, device=cuda) > 0, 0.5, 1.0).float()
    gate, up = Int8Weight(q, half), Int8Weight(q2, ones)
    R.close(gated_ffn_int8(x, gate, up, down, act="relu"), _ffn_int8_defined(x, gate, up, down, "relu"))
    for scale in (1e-18, 1e-12):  # h near 1e-36 and 1e-24 beside a gate and up of 1e-18 and 1e-12
        wide = Int8Weight(down.q, down.scale / scale / scale)
        w = [pack_int8(randn(inter, 64)) for _ in range(2)]
        for name in R.ACTS:
            x = randn(T, 64) * scale
            y, ref = gated_ffn_int8(x, *w, wide, act=name), _ffn_int8_defined(x, *w, wide, name)
            R.close(y, (ref[0], ref[1] * (1 if scale > 1e-15 else 2 ** 6)), (scale, name))


def test_eight_tokens_of_large_weights(cuda):
    """Calls of at most eight rows take no workspace, whatever the weights' size."""
    import ctypes

    from dsca_moe_b200 import _lib as L
    from dsca_moe_b200 import gated_ffn, int8_linear, pack_int8, quantize_rows

    randn = _randn(cuda, 9)
    x = randn(8, 2048).to(BF16)
    wg, wu, wd = ((randn(*s) * s[1] ** -0.5).to(BF16) for s in ((13000, 2048), (13000, 2048), (2048, 13000)))
    R.close(gated_ffn(x, wg, wu, wd), R.ffn(x, wg, wu, wd, "silu", BF16)["y"])
    w = pack_int8(torch.cat([wg, wu, wg]))
    q, s = quantize_rows(x)
    R.close(int8_linear(x, w), R.int8_linear(q, s, w.q, w.scale, BF16))
    y = torch.empty(8, 39000, dtype=BF16, device=cuda)
    a = L.Int8LinearArgs(None, q.data_ptr(), s.data_ptr(), w.q.data_ptr(), w.scale.data_ptr(), None, y.data_ptr(), 8, 2048, 39000,
                         L.BF16, 2048, 2048, 2048, 39000, None, 0, None)
    assert L.load().dsca_int8_linear_workspace(ctypes.byref(a)) == 0
