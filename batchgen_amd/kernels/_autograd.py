"""Gradients that have none of their own: under ``create_graph=True`` such a gradient is returned as a function of
everything its value depends on, and differentiating it raises.  (torch's ``once_differentiable`` looks only at the
incoming gradient: with a constant one, ``out.sum()``, it returns a constant, and a penalty on that gradient would be
differentiated as zero.)"""
from __future__ import annotations

from typing import Optional

import torch


class _Refuse(torch.autograd.Function):
    @staticmethod
    def forward(ctx, name, grad, *sources):
        ctx.op = name
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.op}: its gradient has no gradient of its own")


def no_second_gradient(name: str, grad: Optional[torch.Tensor], *sources) -> Optional[torch.Tensor]:
    """``grad``, computed from ``sources`` (None: not there): tied to those that require a gradient."""
    sources = [t for t in sources if t is not None and t.requires_grad]
    return grad if grad is None or not sources else _Refuse.apply(name, grad, *sources)
