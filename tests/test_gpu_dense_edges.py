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
