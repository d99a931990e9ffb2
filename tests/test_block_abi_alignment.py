"""Pointers of dsca_moe_few that a value cannot lie at are refused, without a GPU."""
import ctypes

import pytest

from test_block_abi import _few_args


@pytest.mark.parametrize("weights", [0, 1, 2])
@pytest.mark.parametrize("change", [
    dict(logits=4097), dict(topk_ids=4098), dict(topk_w=4098), dict(expert_index=4100), dict(err=4097), dict(w1_scale=4098),
    dict(w2_scale=4097), dict(ws1_scale=4098), dict(ws2_scale=4099), dict(out=4104)])
def test_few_misaligned_pointers(lib, change, weights):
    from dsca_moe_b200 import _lib as L

    a = _few_args()
    a.weights, a.expert_index, a.err = weights, 4096, 4096
    a.w1_scale = a.w2_scale = a.ws1_scale = a.ws2_scale = 4096
    for k, v in change.items():
        setattr(a, k, v)
    assert lib.dsca_moe_few(ctypes.byref(a), None) == L.ERR_BAD_ARG


def test_few_logits_of_the_routers_type(lib):
    from dsca_moe_b200 import _lib as L

    a = _few_args()
    a.weights, a.logits = L.F32, 4098
    assert lib.dsca_moe_few(ctypes.byref(a), None) == L.ERR_BAD_ARG
