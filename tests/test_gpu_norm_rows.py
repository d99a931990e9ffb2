"""add_rms_norm's 8-bit rows where their codes are known bit for bit."""
import pytest
import torch

from test_gpu_norm import _inputs

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
