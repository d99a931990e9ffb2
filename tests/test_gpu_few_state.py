"""forward_few computes with what its engine holds at the call: weights, tables and settings replaced after a first call."""
import pytest
import torch

from test_gpu_few import _check, _engine, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "fp8", "f32"])
@pytest.mark.parametrize("T", [3, 12])
def test_replaced_weights_and_settings(cuda, T, kind):
    eng, w, router, gate, n = _engine(cuda, 256, 12, 2, 100, 72, kind=kind, seed=51)
    other, w2, router2, gate2, _ = _engine(cuda, 256, 12, 2, 100, 72, kind=kind, seed=52)
    x = n(T, 256, std=1.0)
    _check(_run(eng, x), x, w, router, gate, 2)
    eng.router_weight = router2.clone()
    _check(_run(eng, x), x, w, router2, gate, 2)
    eng.experts = other.experts
    _check(_run(eng, x), x, w2, router2, gate, 2)
    eng.shared_gate_weight = gate2.clone()
    _check(_run(eng, x), x, w2, router2, gate2, 2)
    eng.norm_topk = True
    _check(_run(eng, x), x, w2, router2, gate2, 2, norm=True)
    eng.top_k, eng.norm_topk = 5, False  # a larger workspace, too
    _check(_run(eng, x), x, w2, router2, gate2, 5)
    # the same tensor with other memory behind it
    eng.experts.w2.data = eng.experts.w2.data.clone()
    other.experts.w1.data = other.experts.w1.data.clone()
    _check(_run(eng, x), x, w2, router2, gate2, 5)


def test_experts_of_another_width(cuda):
    eng, w, router, gate, n = _engine(cuda, 256, 12, 2, 100, 72, seed=53)
    wide, w2, _, _, _ = _engine(cuda, 256, 12, 2, 2000, 1500, seed=54)
    x = n(7, 256, std=1.0)
    _check(_run(eng, x), x, w, router, gate, 2)
    eng.experts = wide.experts
    _check(_run(eng, x), x, w2, router, gate, 2)
    eng.check()


def test_freed_weights_are_not_read(cuda):
    """The first weights' memory is given to other tensors after they have been replaced."""
    eng, w, router, gate, n = _engine(cuda, 256, 12, 2, 100, 72, seed=55)
    x = n(4, 256, std=1.0)
    want = _run(eng, x)["out"].clone()
    eng.router_weight = eng.router_weight.clone()
    trash = [torch.full_like(router, float("nan")) for _ in range(8)]
    del router
    trash += [torch.full_like(trash[0], float("nan")) for _ in range(8)]
    assert torch.equal(_run(eng, x)["out"], want)
    assert len(trash) == 16
