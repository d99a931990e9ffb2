"""The waits of dsca_moe_few when they run out: the call ends, reports it, and leaves nothing behind.

A counter of the workspace that starts far below zero never reaches its target, so every CTA's wait for it lasts as
long as its limit (20 ms here).  What the call computes then has no meaning, but every index that it uses has to stay
in range, whichever lists the router has written by that time."""
import pytest
import torch

from test_gpu_few import _check, _engine, _run

pytestmark = pytest.mark.gpu

COUNTERS = {"logits": 0, "shared": 2, "routed": 4}


# up to four tokens two warps route beside the others' products, above all warps do; nine tokens and more are
# gathered for each expert
@pytest.mark.parametrize("T", [2, 7, 12])
@pytest.mark.parametrize("kind", ["bf16", "fp8", "f32"])
@pytest.mark.parametrize("counter", list(COUNTERS))
def test_a_wait_that_runs_out(cuda, counter, kind, T):
    from dsca_moe_b200 import _lib as L

    eng, w, router, gate, n = _engine(cuda, 512, 60, 4, 384, 768, kind=kind, seed=31)
    x = n(T, 512, std=1.0)
    want = {key: v.clone() for key, v in _run(eng, x).items()}
    eng.wait_limit_ns = 20_000_000
    (ws,) = eng._few_ws.values()
    assert not ws[:L.FEW_ZERO_BYTES].any()
    ws.view(torch.int32)[COUNTERS[counter]] = -(1 << 20)
    eng.forward_few(x)
    with pytest.raises(L.DscaError) as e:
        eng.check()
    assert e.value.code == L.ERR_WAIT_TIMEOUT
    assert eng._few_ws == {}
    eng.wait_limit_ns = 2_000_000_000
    r = _run(eng, x)
    assert all(torch.equal(r[key], want[key]) for key in want)
    _check(r, x, w, router, gate, 4)


@pytest.mark.parametrize("T", [2, 12])
def test_a_block_without_a_shared_expert(cuda, T):
    from dsca_moe_b200 import _lib as L

    eng, w, router, gate, n = _engine(cuda, 256, 12, 1, 320, act="relu", seed=32)
    x = n(T, 256, std=1.0)
    want = _run(eng, x)["out"].clone()
    for counter in ("logits", "routed"):
        eng.wait_limit_ns = 20_000_000
        (ws,) = eng._few_ws.values()
        ws.view(torch.int32)[COUNTERS[counter]] = -(1 << 20)
        eng.forward_few(x)
        with pytest.raises(L.DscaError):
            eng.check()
        eng.wait_limit_ns = 2_000_000_000
        assert torch.equal(_run(eng, x)["out"], want)
