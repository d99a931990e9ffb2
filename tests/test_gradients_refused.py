"""Calls without a backward pass: the forward pass is what it is without autograd, a backward pass that reaches one raises
instead of leaving a part of the gradient out."""
from types import SimpleNamespace

import pytest
import torch
import torch.autograd.forward_ad as fwad
import torch.nn as nn

from dsca_moe_b200.gradients import refuse_tangents, without_gradient


class _Engine:
    """A block on the host: out = 2 x, logits of four experts."""
    _uses_qos, cache, last_loads = False, None, 0

    def forward(self, x, qos=None):
        return {"out": 2 * x, "logits": x[:, :4].clone(), "expert_index": torch.zeros(len(x), dtype=torch.int64)}


def _qwen(logits):
    from dsca_moe_b200.layers import ShardedQwenMoE

    m = ShardedQwenMoE.__new__(ShardedQwenMoE)
    nn.Module.__init__(m)
    m.engine, m.route_calls, m.return_logits = _Engine(), 0, logits
    return m


def _switch(logits):
    from dsca_moe_b200.layers import QoSMoELayer

    m = QoSMoELayer.__new__(QoSMoELayer)
    nn.Module.__init__(m)
    m.engine, m.runtime_context, m.d_model, m.layer_idx = _Engine(), SimpleNamespace(last_hidden_states=None), 8, 0
    m.config = SimpleNamespace(collect_stats=False, return_router_tuple=logits)
    return m


@pytest.mark.parametrize("make", [_qwen, _switch])
@pytest.mark.parametrize("logits", [False, True])
def test_blocks(make, logits):
    block, first, last = make(logits), nn.Linear(8, 8), nn.Linear(8, 8)
    x = torch.randn(2, 3, 8)

    def call(h):
        r = block(h)
        return r if torch.is_tensor(r) else r[0]

    with torch.no_grad():
        want = last(first(x) + call(first(x)))
    h = first(x)
    y = last(h + call(h))
    assert torch.equal(y, want)
    with pytest.raises(RuntimeError, match="MoE block"):
        y.sum().backward()
    if logits:
        r = block(first(x))[1]
        with pytest.raises(RuntimeError, match="MoE block"):
            (r if torch.is_tensor(r) else r[0]).sum().backward()
    # frozen up to the block: what lies behind it trains
    first.requires_grad_(False)
    h = first(x)
    out = call(h)
    assert not out.requires_grad
    (grad,) = torch.autograd.grad(last(h + out).sum(), last.weight)  # (the refused pass may have left a part in .grad)
    assert torch.allclose(grad, (h + out).reshape(-1, 8).sum(0).expand(8, 8))
    with fwad.dual_level(), pytest.raises(NotImplementedError, match="MoE block"):
        block(fwad.make_dual(x, x))


def test_helpers():
    x, w = torch.randn(3), torch.randn(3, requires_grad=True)
    assert without_gradient("it", x, x, None) is x
    with torch.no_grad():
        assert without_gradient("it", x, w) is x
    y = without_gradient("it", x, None, w)
    assert y.requires_grad and torch.equal(y, x)
    with pytest.raises(RuntimeError, match="it has no backward pass"):
        (y * w).sum().backward()
    refuse_tangents("it", x, w, None)
    with fwad.dual_level():
        refuse_tangents("it", x, w, None)
        with pytest.raises(NotImplementedError, match="it has no forward-mode"):
            refuse_tangents("it", x, fwad.make_dual(x, x))


@pytest.mark.parametrize("make", [_qwen, _switch])
def test_results_in_place(make):
    """A decoder that adds to the block's result in place."""
    block, first, x = make(False), nn.Linear(8, 8), torch.randn(2, 3, 8)
    with torch.no_grad():
        want = (block(first(x)) * 3).add_(first(x))
    out = block(first(x))
    out.mul_(3)
    out += first(x)
    assert torch.equal(out, want)
    with pytest.raises(RuntimeError, match="MoE block"):
        out.sum().backward()
