"""gated_ffn, its gradients, int8_linear and gated_ffn_int8 against their definitions in 64 bits, value by
value within the bounds that dense_ref derives."""
import pytest
import torch

import dense_ref as R

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _inputs(dev, T, d, I, dtype, seed=0, gap=0):
    g = torch.Generator(device=dev)
    g.manual_seed(seed + 1000 * T + d + I)

    def n(rows, cols, std):
        return (torch.randn(rows, cols + gap, generator=g, device=dev) * std).to(dtype)[:, :cols]

    return (n(T, d, 1.0) * torch.exp(0.3 * torch.randn(T, 1, generator=g, device=dev)).to(dtype), n(I, d, d ** -0.5),
            n(I, d, d ** -0.5), n(d, I, I ** -0.5), n(T, d, 0.3))


# one token to many, sizes on and off every tile border, widths that no 16-byte vector fits
SHAPES = [(1, 8, 8), (1, 2048, 1408), (1, 64, 1), (2, 1, 3), (3, 712, 333), (5, 100, 36), (8, 256, 512), (9, 264, 130),
          (16, 768, 2048), (17, 512, 256), (31, 1021, 901), (33, 128, 64), (48, 2048, 1408), (64, 320, 192), (100, 712, 1021),
          (127, 72, 1000), (129, 256, 264), (200, 1000, 100), (257, 136, 513), (333, 1021, 901), (511, 512, 768),
          (640, 768, 2048), (1100, 96, 2056)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,d,I", SHAPES)
def test_ffn_and_gradients(cuda, T, d, I, dtype):
    from dsca_moe_b200 import check_dense, gated_ffn

    x, wg, wu, wd, dy = _inputs(cuda, T, d, I, dtype)
    name = R.ACTS[(T + d + I) % 3]
    ref = R.ffn(x, wg, wu, wd, name, dtype, dy)
    R.close(gated_ffn(x, wg, wu, wd, act=name), ref["y"], "y")
    p = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    y = gated_ffn(*p, act=name)
    R.close(y.detach(), ref["y"], "y saved")
    for got, k in zip(torch.autograd.grad(y, p, dy), ("dx", "d_gate", "d_up", "d_down")):
        assert got.dtype == dtype
        R.close(got, ref[k], k)
    check_dense()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("name", R.ACTS)
@pytest.mark.parametrize("T", [1, 7, 40, 300])
def test_gates(cuda, T, name, dtype):
    """Every gate over a wide range of g, and the largest magnitudes."""
    from dsca_moe_b200 import gated_ffn

    x, wg, wu, wd, dy = _inputs(cuda, T, 136, 72, dtype, 5)
    wg = (wg.float() * 30).to(dtype)
    p = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    y = gated_ffn(*p, act=name)
    ref = R.ffn(x, wg, wu, wd, name, dtype, dy)
    R.close(y.detach(), ref["y"], "y")
    for got, k in zip(torch.autograd.grad(y, p, dy), ("dx", "d_gate", "d_up", "d_down")):
        R.close(got, ref[k], k)
    big = (x.float() * 1e15).to(dtype)
    y = gated_ffn(big, wg, wu, wd, act=name)
    assert torch.isfinite(y).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,d,I,gap", [(1, 264, 520, 8), (3, 100, 77, 5), (40, 128, 136, 8), (150, 130, 66, 3), (150, 136, 264, 16)])
def test_rows_of_wider_buffers(cuda, T, d, I, gap, dtype):
    from dsca_moe_b200 import gated_ffn

    x, wg, wu, wd, dy = _inputs(cuda, T, d, I, dtype, 9, gap)
    ref = R.ffn(x, wg, wu, wd, "silu", dtype, dy)
    p = [t.detach().requires_grad_() for t in (x, wg, wu, wd)]
    y = gated_ffn(*p)
    R.close(y.detach(), ref["y"], "y")
    for got, k in zip(torch.autograd.grad(y, p, dy), ("dx", "d_gate", "d_up", "d_down")):
        R.close(got, ref[k], k)


@pytest.mark.parametrize("T", [4, 70])
def test_gradients_asked_for(cuda, T):
    """Any subset of the gradients, a broadcast and a transposed dy, a batch in front."""
    from dsca_moe_b200 import gated_ffn

    x, wg, wu, wd, dy = _inputs(cuda, T, 128, 200, BF16, 2)
    ref = R.ffn(x, wg, wu, wd, "silu", BF16, dy)
    for mask in range(1, 16):
        p = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, wg, wu, wd))]
        gated_ffn(*p).backward(dy)
        for i, k in enumerate(("dx", "d_gate", "d_up", "d_down")):
            if mask >> i & 1:
                R.close(p[i].grad, ref[k], k)
            else:
                assert p[i].grad is None
    p = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    gated_ffn(*p).sum().backward()
    R.close(p[0].grad, R.ffn(x, wg, wu, wd, "silu", BF16, torch.ones_like(dy))["dx"])
    xb = x.view(2, T // 2, 128).detach().requires_grad_()
    y = gated_ffn(xb, wg, wu, wd)
    assert y.shape == xb.shape
    (dx,) = torch.autograd.grad(y, xb, dy.view_as(y))
    R.close(dx.view(T, 128), ref["dx"])
    xt = x.detach().requires_grad_()
    (dx,) = torch.autograd.grad(gated_ffn(xt, wg, wu, wd), xt, dy.T.contiguous().T)
    R.close(dx, ref["dx"])
    with torch.no_grad():
        assert not gated_ffn(xt, wg, wu, wd).requires_grad


def test_offsets_beyond_32_bits(cuda):
    """More than 2^31 values of x and y: the first and the last rows."""
    from dsca_moe_b200 import gated_ffn, gated_ffn_int8, int8_linear, pack_int8, quantize_rows

    T, d, I = 270001, 8192, 40
    g = torch.Generator(device=cuda)
    g.manual_seed(1)
    x = torch.randn(T, d, generator=g, device=cuda, dtype=BF16)
    wg, wu, wd = (torch.randn(*s, generator=g, device=cuda).mul_(s[1] ** -0.5).to(BF16) for s in ((I, d), (I, d), (d, I)))
    dy = torch.randn(T, d, generator=g, device=cuda, dtype=BF16)
    last = slice(T - 33, T)
    p = [x.requires_grad_()] + [t.clone().requires_grad_() for t in (wg, wu, wd)]
    y = gated_ffn(*p)
    (dx,) = torch.autograd.grad(y, p[0], dy)
    for rows in (slice(0, 33), last):
        ref = R.ffn(x[rows].detach(), wg, wu, wd, "silu", BF16, dy[rows])
        R.close(y[rows].detach(), ref["y"])
        R.close(dx[rows], ref["dx"])
    del y, dx
    x = x.detach()
    q, s = quantize_rows(x)
    assert torch.equal(q[last].double(), R.codes(x[last].double())[0])
    pw = [pack_int8(w) for w in (wg, wu, wd)]
    wide = pack_int8(torch.randn(d, 64, generator=g, device=cuda, dtype=BF16))
    R.close(int8_linear(q[:, :64], wide, x_scale=s)[last], R.int8_linear(q[last, :64], s[last], wide.q, wide.scale, BF16))
    R.close(gated_ffn_int8(x, *pw)[last], R.ffn_int8(x[last], *pw, "silu", BF16))


@pytest.mark.parametrize("T,d,I,dtype", [(2600, 520, 1544, BF16), (4100, 256, 300, BF16), (3000, 264, 200, F32), (20000, 64, 72, BF16)])
def test_many_tiles(cuda, T, d, I, dtype):
    """More tiles than CTA pairs, ragged ones among them."""
    from dsca_moe_b200 import gated_ffn, gated_ffn_int8, pack_int8

    x, wg, wu, wd, dy = _inputs(cuda, T, d, I, dtype, 31)
    ref = R.ffn(x, wg, wu, wd, "silu", dtype, dy)
    p = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    y = gated_ffn(*p)
    R.close(y.detach(), ref["y"], "y")
    for got, k in zip(torch.autograd.grad(y, p, dy), ("dx", "d_gate", "d_up", "d_down")):
        R.close(got, ref[k], k)
    q = [pack_int8(w) for w in (wg, wu, wd)]
    R.close(gated_ffn_int8(x, *q), R.ffn_int8(x, *q, "silu", dtype))


def test_gradient_against_differences(cuda):
    from dsca_moe_b200 import gated_ffn

    x, wg, wu, wd, dy = _inputs(cuda, 130, 96, 160, F32, 4)
    p = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    grads = torch.autograd.grad(gated_ffn(*p, act="gelu"), p, dy)
    for i in range(4):
        args = [t.double() for t in (x, wg, wu, wd)]
        v = torch.randn_like(args[i])
        step = 1e-6
        lo, hi = list(args), list(args)
        lo[i], hi[i] = args[i] - step * v, args[i] + step * v
        diff = ((R.ffn(*hi, "gelu", F32)["y"][0] - R.ffn(*lo, "gelu", F32)["y"][0]) * dy.double()).sum() / (2 * step)
        # differences are good to 1e-8 here, the fp32 gradients' bounds sum to far less than 1e-4 of |grad| |v|
        assert abs(float(diff - (grads[i].double() * v).sum())) <= 1e-4 * float((grads[i].double() * v).abs().sum())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_no_rows(cuda, dtype):
    from dsca_moe_b200 import gated_ffn, gated_ffn_int8, int8_linear, pack_int8, quantize_rows

    x, wg, wu, wd, _ = _inputs(cuda, 1, 64, 96, dtype)
    p = [t.clone().requires_grad_() for t in (x[:0], wg, wu, wd)]
    y = gated_ffn(*p)
    assert y.shape == (0, 64)
    y.sum().backward()
    assert p[0].grad.shape == (0, 64) and all(not t.grad.any() for t in p[1:])
    q = [pack_int8(w) for w in (wg, wu, wd)]
    assert int8_linear(x[:0], q[0]).shape == (0, 96) and gated_ffn_int8(x[:0], *q).shape == (0, 64)
    assert quantize_rows(x[:0])[0].shape == (0, 64)


@pytest.mark.parametrize("T", [2, 20, 200])
def test_nonfinite_rows_stay_in_their_rows(cuda, T):
    from dsca_moe_b200 import gated_ffn, gated_ffn_int8, int8_linear, pack_int8

    for dtype in (BF16, F32):
        x, wg, wu, wd, _ = _inputs(cuda, T, 136, 200, dtype)
        q = [pack_int8(w) for w in (wg, wu, wd)]
        calls = (lambda t: gated_ffn(t, wg, wu, wd), lambda t: int8_linear(t, q[0]), lambda t: gated_ffn_int8(t, *q))
        for bad in (float("nan"), float("inf")):
            xb = x.clone()
            xb[T // 2, 17] = bad
            for f in calls:
                want, got = f(x), f(xb)
                assert not torch.isfinite(got[T // 2]).any()
                keep = torch.arange(T, device=cuda) != T // 2
                assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,k,gap", [(1, 1, 0), (1, 8, 0), (3, 17, 0), (7, 2048, 0), (33, 1021, 3), (700, 264, 8), (601, 768, 0),
                                        (900, 1000, 1), (650, 2050, 0), (5, 4096, 0), (3, 8200, 0), (2, 20011, 0)])
def test_quantize_rows(cuda, rows, k, gap, dtype):
    """Codes are those of the exact quotient, bit for bit."""
    from dsca_moe_b200 import quantize_rows

    g = torch.Generator(device=cuda)
    g.manual_seed(rows + k)
    x = torch.randn(rows, k + gap, generator=g, device=cuda).to(dtype)[:, :k]
    x[::3] = (x[::3] * 64).round() / 64  # ties among them
    x[0] = 0
    if rows > 1:
        x[1] *= 1e-38
    if rows > 2:
        x[2] *= 3e37
    q, s = quantize_rows(x)
    qr, sr = R.codes(x.double())
    assert q.dtype == torch.int8 and q.shape == x.shape and torch.equal(q.double(), qr)
    # in 64 bits and then rounded: torch divides fp32 tensors by a number through its reciprocal
    assert torch.equal(s, sr.float())
    assert q.stride(0) % 16 == 0
    pad = torch.as_strided(q, (rows, q.stride(0) - k), (q.stride(0), 1), k) if q.stride(0) > k else q[:0]
    assert not pad.any()
    assert ((s.double() - sr).abs() <= 2.0 ** -24 * sr + 1.5e-45).all()


@pytest.mark.parametrize("k,powers", [(2560, 10), (5632, 22)])
def test_quantize_rows_every_quotient(cuda, k, powers):
    """bf16: every pair of eight-bit significands and every power of two between them that leaves a code."""
    from dsca_moe_b200 import quantize_rows

    sig = torch.arange(128, 256, device=cuda, dtype=torch.float64)
    x = torch.cat([s * 2.0 ** -e * sig for e in range(powers) for s in (1, -1)]).repeat(128, 1)
    x = torch.where(x.abs() <= sig[:, None], x, torch.zeros_like(x))  # a row's largest magnitude is its significand
    assert x.shape == (128, k) and torch.equal(x.abs().amax(1), sig)
    x = torch.cat([x * 2.0 ** b for b in (-99, -50, -7, 0, 1, 60, 112)])
    v = x.bfloat16()
    assert torch.equal(v.double(), x)
    q, s = quantize_rows(v)
    qr, sr = R.codes(x)
    assert torch.equal(q.double(), qr) and torch.equal(s, sr.float())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,k,gap", [(1, 4097, 7), (3, 4104, 0), (1300, 4104, 16), (2500, 5632, 0), (900, 6145, 7), (1500, 8192, 0),
                                        (1200, 8185, 7)])
def test_quantize_long_rows(cuda, rows, k, gap, dtype):
    """Rows of more than 4096 values: several for each CTA, the last chunk cut short, a row that is not finite."""
    from dsca_moe_b200 import quantize_rows

    g = torch.Generator(device=cuda)
    g.manual_seed(rows + k)
    x = (torch.randn(rows, k + gap, generator=g, device=cuda) * torch.exp(torch.randn(rows, 1, generator=g, device=cuda))).to(dtype)
    x[:, k:] = float("nan")  # of no row
    x = x[:, :k]
    x[rows // 2] = 0
    x[rows // 3, k - 1] = 1000
    q, s = quantize_rows(x)
    qr, sr = R.codes(x.double())
    assert torch.equal(q.double(), qr) and torch.equal(s, sr.float())
    if q.stride(0) > k:
        assert not torch.as_strided(q, (rows, q.stride(0) - k), (q.stride(0), 1), k).any()
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[rows // 2, 5] = bad
        q2, s2 = quantize_rows(y)
        keep = torch.arange(rows, device=cuda) != rows // 2
        assert torch.equal(q2[keep], q[keep]) and torch.equal(s2[keep], s[keep])
        assert not q2[rows // 2].any() and not torch.isfinite(s2[rows // 2])


@pytest.mark.parametrize("T", [1, 8, 11, 24, 32, 33])
@pytest.mark.parametrize("d,I", [(256, 320), (101, 67)])
def test_f32_few_tokens_range(cuda, T, d, I):
    """fp32 values of every size, the largest among them, and rows that are not finite beside rows that are."""
    from dsca_moe_b200 import gated_ffn

    x, wg, wu, wd, _ = _inputs(cuda, T, d, I, F32)
    for sx, sw in ((2.0 ** 40, 1.0), (2.0 ** -30, 1.0), (2.0 ** -60, 2.0 ** 60)):
        args = (x * sx, wg * sw, wu * sw, wd)
        R.close(gated_ffn(*args, act="relu"), R.ffn(*args, "relu", F32)["y"], (sx, sw))
    big = wg.clone()
    big[I // 2, d // 3] = torch.finfo(F32).max  # no bf16 is as large
    args = (x * 2.0 ** -100, big, wu, wd)
    R.close(gated_ffn(*args, act="relu"), R.ffn(*args, "relu", F32)["y"], "largest")
    want = gated_ffn(x, wg, wu, wd)
    for bad in (float("nan"), float("inf"), -float("inf")):
        y = x.clone()
        y[T // 2, d // 2] = bad
        got, keep = gated_ffn(y, wg, wu, wd), torch.arange(T, device=cuda) != T // 2
        assert not torch.isfinite(got[T // 2]).any() and torch.equal(got[keep], want[keep])


INT8_SHAPES = [(1, 16, 1), (1, 2048, 5632), (1, 33, 77), (4, 1021, 130), (8, 5632, 2048), (9, 256, 1000), (16, 128, 64),
               (20, 2048, 901), (32, 4100, 300), (33, 100, 257), (64, 512, 512), (100, 1021, 1363), (129, 144, 2000),
               (257, 2048, 264), (777, 1021, 1363), (1030, 640, 768)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,k,n", INT8_SHAPES)
def test_int8_linear(cuda, T, k, n, dtype):
    from dsca_moe_b200 import check_dense, int8_linear, pack_int8, quantize_rows

    x, w, *_ = _inputs(cuda, T, k, n, dtype, 3)
    bias = torch.randn(n, device=cuda).to(dtype) if (T + n) % 2 else None
    pw = pack_int8(w)
    q, s = quantize_rows(x)
    ref = R.int8_linear(q, s, pw.q, pw.scale, dtype, bias)
    y = int8_linear(x, pw, bias=bias)
    assert y.dtype == dtype
    R.close(y, ref)
    assert torch.equal(int8_linear(q, pw, bias=bias, x_scale=s, out_dtype=dtype), y)
    check_dense()


def test_int8_linear_extremes(cuda):
    """The largest sums: every code 127, the longest rows; and codes in a batch's shape."""
    from dsca_moe_b200 import Int8Weight, int8_linear, pack_int8, quantize_rows

    for T in (1, 40):
        k = 131072
        q = torch.full((T, k), 127, dtype=torch.int8, device=cuda)
        q[T // 2] = -127
        w = Int8Weight(torch.full((5, k), 127, dtype=torch.int8, device=cuda), torch.ones(5, device=cuda))
        y = int8_linear(q, w, x_scale=torch.ones(T, device=cuda), out_dtype=F32)
        want = torch.full((T, 5), 127.0 * 127 * k, device=cuda)
        want[T // 2] *= -1
        assert torch.equal(y, want)
    x = torch.randn(2, 3, 50, device=cuda)
    w = pack_int8(torch.randn(30, 50, device=cuda))
    y = int8_linear(x, w)
    q, s = quantize_rows(x)
    assert q.shape == x.shape and s.shape == (2, 3)
    assert torch.equal(y.view(6, 30), int8_linear(x.view(6, 50), w))
    assert torch.equal(y, int8_linear(q, w, x_scale=s, out_dtype=F32))
    assert torch.equal(int8_linear(x[0, 0], w), y[0, 0])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,d,I", [(1, 2048, 1408), (1, 40, 24), (3, 333, 77), (8, 256, 512), (16, 768, 2048), (20, 1021, 130),
                                   (33, 128, 1000), (70, 712, 1021), (130, 1024, 272), (333, 1021, 901), (600, 256, 640)])
def test_gated_ffn_int8(cuda, T, d, I, dtype):
    from dsca_moe_b200 import check_dense, gated_ffn_int8, pack_int8

    x, wg, wu, wd, _ = _inputs(cuda, T, d, I, dtype, 6)
    q = [pack_int8(w) for w in (wg, wu, wd)]
    name = R.ACTS[(T + d + I) % 3]
    R.close(gated_ffn_int8(x, *q, act=name), R.ffn_int8(x, *q, name, dtype))
    check_dense()


def _calls(dev, T):
    """One call of each kind on inputs of its own, and its result's 64-bit reference."""
    from dsca_moe_b200 import gated_ffn, gated_ffn_int8, int8_linear, pack_int8

    x, wg, wu, wd, dy = _inputs(dev, T, 264, 520, BF16, 8)
    q = [pack_int8(w) for w in (wg, wu, wd)]
    return x, (lambda t: gated_ffn(t, wg, wu, wd), lambda t: int8_linear(t, q[0]), lambda t: gated_ffn_int8(t, *q))


@pytest.mark.parametrize("T", [1, 12, 90, 700])
def test_streams_and_graphs(cuda, T):
    """The same bits on another stream, in two graphs captured one after the other and replayed in turn, and
    in calls that overlap on two streams."""
    x, calls = _calls(cuda, T)
    x2 = x.flip(0).contiguous() if T > 1 else x * 2
    for f in calls:
        want, want2 = f(x), f(x2)
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        outs = []
        for _ in range(4):
            for s, t in ((s1, x), (s2, x2)):
                with torch.cuda.stream(s):
                    outs.append(f(t))
        torch.cuda.synchronize()
        assert all(torch.equal(o, want if i % 2 == 0 else want2) for i, o in enumerate(outs))
        xs, graphs = [x.clone(), x2.clone()], []
        for t in xs:
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                o = f(t)
            graphs.append((gr, o))
        for _ in range(3):
            for gr, _o in graphs:
                gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want2)
        xs[0].copy_(x2)
        graphs[0][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], want2)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [6, 300])
def test_training_step_in_a_graph(cuda, T, dtype):
    from dsca_moe_b200 import gated_ffn

    x, wg, wu, wd, dy = _inputs(cuda, T, 136, 264, dtype, 12)
    want = None
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
        for _ in range(2):
            want = torch.autograd.grad(gated_ffn(*p), p, dy)
        gr = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(gr, stream=side):
            got = torch.autograd.grad(gated_ffn(*p), p, dy)
    torch.cuda.synchronize()
    for _ in range(2):
        gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("T", [1, 40, 500])
def test_repeats_bit_for_bit(cuda, T):
    from dsca_moe_b200 import gated_ffn

    for dtype in (BF16, F32):
        x, wg, wu, wd, dy = _inputs(cuda, T, 520, 1000, dtype, 1)
        p = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
        runs = []
        for _ in range(3):
            y = gated_ffn(*p)
            runs.append((y.detach(),) + torch.autograd.grad(y, p, dy))
        assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))


def test_refusals_on_the_gpu(cuda):
    from dsca_moe_b200 import Int8Weight, gated_ffn, gated_ffn_int8, int8_linear, pack_int8

    x, wg, wu, wd, dy = _inputs(cuda, 4, 64, 96, BF16)
    with pytest.raises(ValueError, match="w_up"):
        gated_ffn(x, wg, wu[:-1], wd)
    with pytest.raises(ValueError, match="w_down"):
        gated_ffn(x, wg, wu, wd.T.contiguous())
    with pytest.raises(ValueError, match="type"):
        gated_ffn(x, wg, wu.float(), wd)
    with pytest.raises(ValueError, match="device"):
        gated_ffn(x, wg, wu, wd.cpu())
    with pytest.raises(ValueError, match="contiguous"):
        gated_ffn(x, wg.T.contiguous().T, wu, wd)
    with pytest.raises(ValueError, match="overlap"):
        gated_ffn(x[:1].expand(4, 64), wg, wu, wd)
    q = pack_int8(wg)
    with pytest.raises(ValueError, match="weight"):
        int8_linear(x[:, :32].contiguous(), q)
    with pytest.raises(ValueError, match="bias"):
        int8_linear(x, q, bias=torch.zeros(95, device=cuda, dtype=BF16))
    with pytest.raises(ValueError, match="scale"):
        int8_linear(x, Int8Weight(q.q, q.scale[:-1]))
    odd = Int8Weight(torch.zeros(96, 63, dtype=torch.int8, device=cuda), q.scale)
    with pytest.raises(ValueError, match="16 bytes"):
        int8_linear(x[:, :63], odd)
    with pytest.raises(ValueError, match="16 bytes"):
        int8_linear(odd.q, Int8Weight(pack_int8(wg[:, :63]).q, q.scale), x_scale=q.scale)
    # a single row of codes has to lie in whole 16 bytes too: what follows it is multiplied
    with pytest.raises(ValueError, match="16 bytes"):
        int8_linear(x[:, :63], Int8Weight(torch.zeros(1, 63, dtype=torch.int8, device=cuda), q.scale[:1]))
    with pytest.raises(ValueError, match="w_down"):
        gated_ffn_int8(x, q, q, q)
    xr = x.clone().requires_grad_()
    y = gated_ffn(xr, wg, wu, wd)
    (dx,) = torch.autograd.grad(y, xr, dy.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def _tiny_qwen(dtype=BF16):
    from transformers import Qwen2MoeConfig, Qwen2MoeForCausalLM

    cfg = Qwen2MoeConfig(vocab_size=97, hidden_size=64, intermediate_size=176, moe_intermediate_size=48,
                         shared_expert_intermediate_size=80, num_hidden_layers=3, num_attention_heads=4,
                         num_key_value_heads=4, num_experts=8, num_experts_per_tok=2, mlp_only_layers=[1],
                         max_position_embeddings=64)
    torch.manual_seed(0)
    return Qwen2MoeForCausalLM(cfg).to("cuda", dtype).eval()


@pytest.mark.parametrize("mode", ["same", "int8"])
def test_patch_swaps_the_dense_layers(cuda, mode):
    """patch(dense_ffn=...) in a model with a dense layer between sparse ones: logits near the model whose dense layer
    is transformers' own, and the dense layer trainable where it keeps its parameters."""
    from dsca_moe_b200 import GatedFFN, patch

    a, b = _tiny_qwen(), _tiny_qwen()
    patch(a, 0, 1)
    patch(b, 0, 1, dense_ffn=mode)
    mlp = b.model.layers[1].mlp
    assert isinstance(mlp, GatedFFN) and not isinstance(a.model.layers[1].mlp, GatedFFN)
    h = torch.randn(2, 9, 64, device=cuda, dtype=BF16)
    old = a.model.layers[1].mlp
    w = [m.weight for m in (old.gate_proj, old.up_proj, old.down_proj)]
    if mode == "same":
        R.close(mlp(h).detach().view(18, 64), R.ffn(h.view(18, 64), *w, "silu", BF16)["y"])
        assert set(mlp.state_dict()) == set(old.state_dict())
        mlp(h).float().square().sum().backward()
        assert all(getattr(mlp, n).weight.grad.abs().sum() > 0 for n in ("gate_proj", "up_proj", "down_proj"))
    else:
        from dsca_moe_b200 import pack_int8

        R.close(mlp(h).view(18, 64), R.ffn_int8(h.view(18, 64), *[pack_int8(t) for t in w], "silu", BF16))
    ids = torch.randint(0, 97, (2, 11), device=cuda)
    with torch.no_grad():
        la, lb = a(ids).logits.float(), b(ids).logits.float()
    # the swapped layer's roundings go through the rest of the model: near, not equal
    assert (la - lb).norm() <= 0.1 * la.norm()


def test_training_with_the_norm_in_front(cuda):
    """norm -> quantised block -> product as one decode step uses them, and three steps of gradient descent on a
    GatedFFN's own parameters: each step's gradients are the formula's for the weights of that step."""
    from dsca_moe_b200 import GatedFFN, add_rms_norm, gated_ffn_int8, int8_linear, pack_int8

    x, wg, wu, wd, dy = _inputs(cuda, 5, 128, 264, BF16, 21)
    n = add_rms_norm(x, torch.ones(128, device=cuda, dtype=BF16), residual=x)
    q = [pack_int8(w) for w in (wg, wu, wd)]
    y = gated_ffn_int8(n.y, *q)
    R.close(y, R.ffn_int8(n.y, *q, "silu", BF16))
    head = pack_int8(torch.randn(300, 128, device=cuda, dtype=BF16))
    from dsca_moe_b200 import quantize_rows

    R.close(int8_linear(n.residual + y, head), R.int8_linear(*quantize_rows(n.residual + y), head.q, head.scale, BF16))

    class M(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.gate_proj, self.up_proj = torch.nn.Linear(128, 264, bias=False), torch.nn.Linear(128, 264, bias=False)
            self.down_proj, self.act_fn = torch.nn.Linear(264, 128, bias=False), torch.nn.SiLU()

    m = GatedFFN(M().to(cuda, BF16))
    opt = torch.optim.SGD(m.parameters(), lr=0.1)
    for _ in range(3):
        ref = R.ffn(x, m.gate_proj.weight, m.up_proj.weight, m.down_proj.weight, "silu", BF16, dy)
        opt.zero_grad()
        m(x).backward(dy)
        for lin, k in ((m.gate_proj, "d_gate"), (m.up_proj, "d_up"), (m.down_proj, "d_down")):
            R.close(lin.weight.grad, (ref[k][0].detach(), ref[k][1].detach()))
        opt.step()
