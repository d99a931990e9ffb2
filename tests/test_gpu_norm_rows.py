"""add_rms_norm's 8-bit rows where their codes are known bit for bit, and its kernels for many rows.

Tolerances are those of test_gpu_norm."""
import pytest
import torch

from test_gpu_norm import F32, _close, _exact, _inputs, _split

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,d", [(1, 2048), (300, 768), (700, 1021), (2000, 512), (7, 8192)])
def test_e4m3_codes_are_those_of_the_quotient(cuda, rows, d):
    """fp32 rows hold the y that is quantised, so every code is that of y / scale, as weights' rows are quantised: the
    quotient rounded to fp32, then to e4m3.  (A quotient of two fp32 values that is rounded to fp64 first is rounded to
    fp32 as the exact one is: 53 >= 2 * 24 + 2 bits.)"""
    from dsca_moe_b200 import add_rms_norm

    for spread in (0.0, 2.0):
        x, r, w = _inputs(cuda, rows, d, torch.float32, 3 * rows + d)
        x = x * torch.exp2(spread * _inputs(cuda, rows, d, torch.float32, 5 * rows + d, False)[0])
        out = add_rms_norm(x, w, residual=r, quant="e4m3")
        assert torch.equal(out.scale, (out.y.abs().amax(-1).double() / 448).float())
        want = (out.y.double() / out.scale.double()[:, None]).float().to(torch.float8_e4m3fn)
        assert torch.equal(out.q.view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_e4m3_codes_at_the_borders(cuda, dtype):
    """Rows of +1 and -1 without eps have y = +-w, so that w can be laid on the borders between two codes: t s for every
    midpoint t, and the fp32 values beside it."""
    from dsca_moe_b200 import add_rms_norm

    codes = torch.arange(0x7E, dtype=torch.uint8, device=cuda)
    v = torch.cat([codes, codes.new_tensor([0x7E])]).view(torch.float8_e4m3fn).double()
    mid = (v[1:] + v[:-1]) / 2
    g = torch.Generator(device=cuda)
    g.manual_seed(61)
    for _ in range(40):
        top = torch.rand(1, generator=g, device=cuda) * 3 + 0.5
        s = (top.double() / 448).float()
        t = (mid * s.double()).float()
        near = torch.cat([t, torch.nextafter(t, t + 1), torch.nextafter(t, t - 1)])
        w = torch.cat([top, near, top.new_zeros(-(near.numel() + 1) % 8)])
        x = torch.ones(2, w.numel(), dtype=dtype, device=cuda)
        x[1, ::2] = -1
        out = add_rms_norm(x, w, 0.0, quant="e4m3")
        assert torch.equal(out.scale, s.expand(2))
        want = ((w * x.float()).double() / s.double()).float().to(torch.float8_e4m3fn)
        assert torch.equal(out.q.view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("top", [3e-45, 1e-43, 6e-43, 1e-38, 1e-31, 1e32, 3e38])
def test_e4m3_rows_of_extreme_sizes(cuda, top):
    """Scales down to fp32's smallest number (not below it, where they would be zero) and up to its largest."""
    from dsca_moe_b200 import add_rms_norm

    w = torch.tensor([top, 0.0, top * 0.5, top * 0.3, 0.0, top * 0.25, 0.0, -top], dtype=torch.float32, device=cuda)
    out = add_rms_norm(torch.ones(3, 8, dtype=torch.bfloat16, device=cuda), w, 0.0, quant="e4m3")
    s = (w.double().abs().max() / 448).float().clamp_min(2.0 ** -149)
    assert torch.equal(out.scale, s.expand(3))
    want = (w.double() / s.double()).float().to(torch.float8_e4m3fn)
    assert torch.equal(out.q.view(torch.uint8), want.view(torch.uint8).expand(3, 8))


@pytest.mark.parametrize("rows,d", [(40, 2048), (2000, 2048), (3000, 768), (8, 8192)])
def test_bf16_rows_are_rounded_twice_at_most(cuda, rows, d):
    """h w is exact in fp32, so y is its product with the rounded 1 / sqrt, once in fp32 and once in bf16.  Rows of small
    integers have exact sums of squares, and with them a 1 / sqrt that is known bit for bit."""
    from dsca_moe_b200 import add_rms_norm

    g = torch.Generator(device=cuda)
    g.manual_seed(rows + d)
    x = torch.randint(-8, 9, (rows, d), generator=g, device=cuda).bfloat16()
    w = (1 + 0.2 * torch.randn(d, generator=g, device=cuda)).bfloat16()
    mean = ((x.double() ** 2).sum(-1, keepdim=True) / d).float()
    inv = (1 / mean.double().sqrt()).float()
    assert torch.equal(add_rms_norm(x, w, 0.0).y, (x.float() * w.float() * inv).bfloat16())


# With more than four rows an SM a row has 32 to 128 threads: widths on both sides of every border between these
# kernels, and odd ones (single values instead of vectors)
WIDTHS = [8, 250, 256, 257, 264, 511, 512, 520, 768, 761, 776, 1024, 1021, 1032, 2041, 2048, 2056]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [601, 1777])
@pytest.mark.parametrize("d", WIDTHS)
def test_many_rows(cuda, d, rows, dtype):
    """Every form of the output, the last rows of a CTA's among them, and rows behind the last one left alone."""
    from dsca_moe_b200 import add_rms_norm

    for residual, gap in ((True, 0), (False, 5)):
        x, r, w = _inputs(cuda, rows, d, dtype, rows + d, residual, gap)
        x[5] = 0
        h, ref = _exact(x, r, w)
        out = add_rms_norm(x, w, residual=r)
        _close(out.y, ref)
        assert torch.equal(out.residual, h)
        q = add_rms_norm(x, w, residual=r, quant="e4m3")
        assert torch.equal(q.y, out.y) and torch.equal(q.residual, h)
        if dtype == torch.float32:
            s = out.y.abs().amax(-1).double() / 448
            s = torch.where(s > 0, s, torch.ones_like(s)).float()
            want = (out.y.double() / s.double()[:, None]).float().to(torch.float8_e4m3fn)
            assert torch.equal(q.scale, s) and torch.equal(q.q.view(torch.uint8), want.view(torch.uint8))
        else:
            s = ref.abs().amax(-1) / 448
            s = torch.where(s > 0, s, torch.ones_like(s))
            assert ((q.scale.double() - s).abs() <= 2 * F32 * s).all()
            got = q.q.float().double() * q.scale.double()[:, None]
            tol = (2.0 ** -4 + 4 * F32) * ref.abs() + 2.0 ** -10 * s[:, None]
            assert ((got - ref).abs() <= tol).all()
        if dtype == torch.bfloat16 and d % 8 == 0:
            q = add_rms_norm(x, w, residual=r, quant="split")
            assert torch.equal(q.y, out.y) and torch.equal(q.residual, h)
            want, inv = _split(out.y)
            assert torch.equal(q.q.view(torch.uint8), want) and torch.equal(q.scale, inv)
            only = add_rms_norm(x, w, residual=r, quant="split", write_y=False)
            assert only.y is None and torch.equal(only.q.view(torch.uint8), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [256, 768, 1021, 2048])
def test_rows_behind_the_last_are_left_alone(cuda, d, dtype):
    """A last CTA that is only partly filled, with the outputs laid in larger buffers."""
    import ctypes

    from dsca_moe_b200 import _lib as L

    rows, kp = 603, (d + 127) // 128 * 128
    x, r, w = _inputs(cuda, rows, d, dtype, 7, True)
    dt = L.BF16 if dtype == torch.bfloat16 else L.F32
    for quant in (L.NORM_Q_NONE, L.NORM_Q_E4M3, L.NORM_Q_SPLIT):
        if quant == L.NORM_Q_SPLIT and (dtype != torch.bfloat16 or d % 8):
            continue
        width = 2 * kp if quant == L.NORM_Q_SPLIT else d
        y, h = (torch.full((rows + 9, d), 7.0, dtype=dtype, device=cuda) for _ in range(2))
        q = torch.full((rows + 9, width), 0x5A, dtype=torch.uint8, device=cuda)
        scale = torch.full((rows + 9,), 7.0, device=cuda)
        a = L.RmsNormArgs(x.data_ptr(), r.data_ptr(), w.data_ptr(), rows, d, dt, dt, d, d, d, d, 1e-6, quant, y.data_ptr(),
                          h.data_ptr(), q.data_ptr(), scale.data_ptr())
        L.call("dsca_rms_norm", ctypes.byref(a), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        _close(y[:rows], _exact(x, r, w)[1])
        assert (y[rows:] == 7).all() and (h[rows:] == 7).all() and (q[rows:] == 0x5A).all() and (scale[rows:] == 7).all()
        assert (scale[:rows] != 7).all() or quant == L.NORM_Q_NONE
