"""Results without a gradient.

Some of the framework's calls (MoE blocks, 8-bit products) have no backward pass.  Where an input wants a gradient, their
results stay part of the graph, and a backward pass that reaches them raises: as constants they would take a part of
the gradient away without a word.  The forward pass is what it is without autograd.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

__all__ = ["refuse_tangents", "without_gradient"]


class _WithoutGradient(torch.autograd.Function):
    @staticmethod
    def forward(ctx, what, out, *inputs):
        ctx.what = what
        return out.detach()  # no view: callers may add to it in place

    @staticmethod
    def backward(ctx, dy):
        raise RuntimeError(f"{ctx.what} has no backward pass: freeze what lies before it, or detach its input")


def refuse_tangents(what: str, *inputs) -> None:
    """Raise where an input carries a forward-mode tangent, which `what` would drop."""
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                                             for t in inputs):
        raise NotImplementedError(f"{what} has no forward-mode derivative")


def without_gradient(what: str, out: torch.Tensor, *inputs) -> torch.Tensor:
    """`out`; a backward pass through it raises where one of `inputs` wants a gradient."""
    for t in inputs:
        if t is not None and t.requires_grad:
            return _WithoutGradient.apply(what, out, *inputs) if torch.is_grad_enabled() else out
    return out
