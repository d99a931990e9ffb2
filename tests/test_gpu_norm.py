"""add_rms_norm against its definition in 64 bits.

Tolerances.  y is rounded once (half a step: eps / 2 of the type, relative); before that it is an fp32
product of h, 1 / sqrt and w (3 roundings, each 2^-24) with the square root of a sum whose chains
are at most 64 additions in a thread, 5 in the warp and 15 across warps: 84 * 2^-24, halved by the
root.  So |y - exact| <= (eps/2 + 64 * 2^-24) |exact|.  The e4m3 rows add half a step of theirs (2^-4)
where a quotient is rounded, 2^-10 of the row's scale in the subnormal range; the scale itself is off by
what y is off.  h and the two-term rows are compared bit for bit."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

F32 = 64 * 2.0 ** -24


def _inputs(dev, rows, d, dtype, seed, residual=True, gap=0):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    x = torch.randn(rows, d + gap, generator=g, device=dev).to(dtype)[:, :d]
    r = (torch.randn(rows, d, generator=g, device=dev) * 4).to(dtype) if residual else None
    w = (1 + 0.2 * torch.randn(d, generator=g, device=dev)).to(dtype)
    return x, r, w


def _exact(x, r, w, eps=1e-6):
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    t = h.double()
    return h, w.double() * t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps)


def _close(y, ref):
    tol = (torch.finfo(y.dtype).eps / 2 + F32) * ref.abs() + 1e-38
    assert ((y.double() - ref).abs() <= tol).all()


def _split(y):
    """dsca_split_rows of y."""
    from dsca_moe_b200 import _lib as L

    rows, d = y.shape
    kp = (d + 127) // 128 * 128
    q = torch.empty(rows, 2 * kp, dtype=torch.uint8, device=y.device)
    inv = torch.empty(rows, dtype=torch.float32, device=y.device)
    a = L.SplitArgs()
    a.src, a.ld, a.rows, a.K, a.dst, a.inv_scale = y.data_ptr(), d, rows, d, q.data_ptr(), inv.data_ptr()
    L.call("dsca_split_rows", ctypes.byref(a), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    return q, inv


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,d,gap", [(1, 1, 0), (3, 7, 0), (1, 2048, 0), (33, 2048, 0), (300, 768, 0), (5, 8, 8),
                                        (17, 264, 5), (129, 520, 0), (64, 1021, 3), (700, 1024, 0), (9, 2056, 0),
                                        (4, 8192, 0), (3, 8200, 0), (2, 16392, 0), (2, 32768, 0), (2, 32767, 1)])
def test_norm(cuda, dtype, rows, d, gap):
    from dsca_moe_b200 import add_rms_norm

    for residual in (False, True):
        x, r, w = _inputs(cuda, rows, d, dtype, rows + d, residual, gap)
        out = add_rms_norm(x, w, 1e-6, r)
        h, ref = _exact(x, r, w)
        assert out.q is None and out.scale is None
        assert torch.equal(out.residual, h)
        if not residual:
            assert out.residual is x
        _close(out.y, ref)


@pytest.mark.parametrize("rows,d,gap,dtype", [(1, 2048, 0, torch.bfloat16), (37, 768, 0, torch.bfloat16),
                                              (5, 1021, 2, torch.bfloat16), (40, 2048, 0, torch.float32),
                                              (3, 8192, 0, torch.bfloat16), (2, 20000, 0, torch.float32),
                                              (2, 32768, 0, torch.float32),
                                              (11, 96, 5, torch.float32)])
def test_norm_e4m3(cuda, rows, d, gap, dtype):
    from dsca_moe_b200 import add_rms_norm

    x, r, w = _inputs(cuda, rows, d, dtype, 7 * rows + d, True, gap)
    out = add_rms_norm(x, w, residual=r, quant="e4m3")
    h, ref = _exact(x, r, w)
    _close(out.y, ref)
    assert out.q.dtype == torch.float8_e4m3fn and tuple(out.q.shape) == (rows, d)
    s = ref.abs().amax(-1) / 448
    assert ((out.scale.double() - s).abs() <= 2 * F32 * s).all()
    got = out.q.float().double() * out.scale.double()[:, None]
    tol = (2.0 ** -4 + 4 * F32) * ref.abs() + 2.0 ** -10 * s[:, None]
    assert ((got - ref).abs() <= tol).all()
    assert (out.q.float().abs().amax(-1) == 448).all()
    only = add_rms_norm(x, w, residual=r, quant="e4m3", write_y=False)
    assert only.y is None and torch.equal(only.q.view(torch.uint8), out.q.view(torch.uint8))


@pytest.mark.parametrize("rows,d,gap", [(1, 2048, 0), (50, 768, 0), (7, 264, 5), (3, 8192, 0), (2, 16384, 3), (4, 8, 0),
                                        (2, 32768, 0)])
def test_norm_split_rows(cuda, rows, d, gap):
    """The two-term rows are those of dsca_split_rows on y, bit for bit, padding included."""
    from dsca_moe_b200 import add_rms_norm

    x, r, w = _inputs(cuda, rows, d, torch.bfloat16, 11 * rows + d, True, gap)
    x[0] *= 2.0 ** -20
    out = add_rms_norm(x, w, residual=r, quant="split")
    _close(out.y, _exact(x, r, w)[1])
    q, inv = _split(out.y)
    assert torch.equal(out.q.view(torch.uint8), q)
    assert torch.equal(out.scale.view(torch.int32), inv.view(torch.int32))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_norm_special_rows(cuda, dtype):
    """A row of zeros stays zero with scale 1, one with an infinity or a NaN spoils itself alone, and
    magnitudes whose squares leave the type's ordinary range still normalise."""
    from dsca_moe_b200 import add_rms_norm

    x, _, w = _inputs(cuda, 6, 512, dtype, 3, False)
    x = x.contiguous()
    x[0] = 0
    x[1, 5] = float("inf")
    x[2, 9] = float("nan")
    x[3] *= 1e12
    x[4] *= 1e-12
    for quant in (None, "e4m3") + (("split",) if dtype == torch.bfloat16 else ()):
        out = add_rms_norm(x, w, 0.0 if quant is None else 1e-6, quant=quant)
        if quant is None:
            assert torch.isnan(out.y[0].float()).all()  # 0 / 0, as the formula has it
            _close(out.y[3:], _exact(x[3:], None, w, 0.0)[1])
        else:
            assert (out.y[0] == 0).all() and (out.q[0].float() == 0).all()
            _close(out.y[3:], _exact(x[3:], None, w)[1])
        assert torch.isnan(out.y[1, 5].float()) and (out.y[1, 6:] == 0).all()
        assert torch.isnan(out.y[2].float()).all()
        if quant == "e4m3":
            assert out.scale[0] == 1 and torch.isnan(out.scale[1:3]).all() and torch.isfinite(out.scale[3:]).all()


def test_norm_shapes_weights_and_places(cuda):
    """Leading dimensions, an fp32 weight under bf16 rows, unaligned rows, an empty batch, in-place outputs."""
    from dsca_moe_b200 import _lib as L
    from dsca_moe_b200 import add_rms_norm

    x, r, w = _inputs(cuda, 24, 256, torch.bfloat16, 5)
    want = add_rms_norm(x, w, residual=r)
    got = add_rms_norm(x.view(2, 3, 4, 256), w, residual=r.view(2, 3, 4, 256))
    assert got.y.shape == (2, 3, 4, 256) and torch.equal(got.y.view(24, 256), want.y)
    one = add_rms_norm(x[3], w, residual=r[3])
    assert one.y.shape == (256,) and torch.equal(one.y, want.y[3])
    wide = torch.zeros(24, 300, dtype=torch.bfloat16, device=cuda)
    wide[:, 3:259] = x
    assert torch.equal(add_rms_norm(wide[:, 3:259], w, residual=r).y, want.y)
    w32 = w.float() * 1.001
    _close(add_rms_norm(x, w32, residual=r).y, _exact(x, r, w32)[1])
    e = add_rms_norm(x[:0], w, residual=r[:0], quant="e4m3")
    assert e.y.shape == (0, 256) and e.q.shape == (0, 256) and e.scale.shape == (0,)
    a = L.RmsNormArgs()
    xi, ri = x.clone(), r.clone()
    a.x = a.y = xi.data_ptr()
    a.residual = a.residual_out = ri.data_ptr()
    a.weight, a.rows, a.d, a.dtype, a.weight_dtype, a.eps = w.data_ptr(), 24, 256, L.BF16, L.BF16, 1e-6
    a.ld_x = a.ld_y = a.ld_residual = a.ld_residual_out = 256
    L.call("dsca_rms_norm", ctypes.byref(a), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert torch.equal(xi, want.y) and torch.equal(ri, want.residual)
    # rows of y behind the last one are left alone
    y = torch.full((25, 256), 7.0, dtype=torch.bfloat16, device=cuda)
    a.x, a.y, a.residual, a.residual_out = x.data_ptr(), y.data_ptr(), r.data_ptr(), None
    L.call("dsca_rms_norm", ctypes.byref(a), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert torch.equal(y[:24], want.y) and (y[24] == 7).all()


def test_norm_offsets_beyond_32_bits(cuda):
    """Rows more than 2^31 elements apart, and dense rows with as many in front of them."""
    from dsca_moe_b200 import add_rms_norm

    ld, d = 2 ** 31 + 8, 64
    x, r, w = _inputs(cuda, 3, d, torch.bfloat16, 21)
    far = torch.empty(2 * ld + 2 * d, dtype=torch.bfloat16, device=cuda)
    xs, rs = far.as_strided((3, d), (ld, 1)), far.as_strided((3, d), (ld, 1), d)
    xs.copy_(x)
    rs.copy_(r)
    got, want = add_rms_norm(xs, w, residual=rs, quant="split"), add_rms_norm(x, w, residual=r, quant="split")
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    del far, xs, rs
    rows, d = 2 ** 20 + 4096, 2048
    x, w = torch.zeros(rows, d, dtype=torch.bfloat16, device=cuda), _inputs(cuda, 1, d, torch.bfloat16, 22)[2]
    last = torch.randn(5, d, device=cuda).bfloat16()
    x[-5:] = last
    got = add_rms_norm(x, w, quant="e4m3")
    assert not got.y[:-5].any() and (got.scale[:-5] == 1).all()
    _close(got.y[-5:], _exact(last, None, w)[1])
    assert torch.equal(got.residual, x)
    want = add_rms_norm(last, w, quant="e4m3")
    assert ((got.scale[-5:] - want.scale).abs() <= 2 * F32 * want.scale).all()


def test_norm_rows_beyond_32_bits_are_refused(cuda):
    from dsca_moe_b200 import add_rms_norm

    w = torch.ones(1, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(ValueError):
        add_rms_norm(torch.empty(2 ** 31, 1, dtype=torch.bfloat16, device=cuda), w)


def test_norm_refusals(cuda):
    from dsca_moe_b200 import add_rms_norm

    x, r, w = _inputs(cuda, 4, 64, torch.bfloat16, 5)
    for bad in (lambda: add_rms_norm(x, w[:63]), lambda: add_rms_norm(x, w.cpu()), lambda: add_rms_norm(x, w.half()),
                lambda: add_rms_norm(x, w, residual=r[:3]), lambda: add_rms_norm(x, w, residual=r.float()),
                lambda: add_rms_norm(x.t(), w[:4]), lambda: add_rms_norm(x, w, write_y=False),
                lambda: add_rms_norm(x[:, :60].contiguous(), w[:60].contiguous(), quant="split"),
                lambda: add_rms_norm(x.float(), w.float(), quant="split"),
                lambda: add_rms_norm(x[:1].expand(4, 64), w),
                lambda: add_rms_norm(x.view(2, 2, 64).transpose(0, 1), w),
                lambda: add_rms_norm(torch.zeros(1, 32769, device=cuda), torch.ones(32769, device=cuda))):
        with pytest.raises(ValueError):
            bad()


def test_norm_streams_and_graphs(cuda):
    """On another stream, and captured with its outputs in the graph's memory."""
    from dsca_moe_b200 import add_rms_norm

    x, r, w = _inputs(cuda, 64, 512, torch.bfloat16, 5)
    want = add_rms_norm(x, w, residual=r, quant="e4m3")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = add_rms_norm(x, w, residual=r, quant="e4m3")
    side.synchronize()
    assert torch.equal(got.y, want.y) and torch.equal(got.scale, want.scale)
    g = torch.cuda.CUDAGraph()
    xs = torch.zeros_like(x)
    with torch.cuda.graph(g):
        out = add_rms_norm(xs, w, residual=r, quant="e4m3")
    xs.copy_(x)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out.y, want.y) and torch.equal(out.q.view(torch.uint8), want.q.view(torch.uint8))
