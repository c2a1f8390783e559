"""Derivatives that there are not: asked for, they raise instead of being left out of a sum.

The kernels' results have no history of their own.  Where a result depends on tensors that require a gradient, and the operator has no
derivative for it (a second one, or any of the attention over a cache), it is computed within a function whose backward raises.
``torch.autograd.function.once_differentiable`` looks at the incoming gradients alone: of a loss that is linear in the result they require none, and
the term that the inputs have in a second derivative was dropped.
"""
import torch
from torch.autograd import forward_ad

__all__ = ["Undifferentiable", "forward_mode"]


def forward_mode() -> bool:
    """Whether tensors may carry tangents here (then they go through an autograd function, which has no forward-mode rule and says so)."""
    return forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled()


class Undifferentiable(torch.autograd.Function):
    """``apply(what, compute, *tensors)``: the results of ``compute()``, which depend on ``tensors``."""

    @staticmethod
    def forward(ctx, what, compute, *tensors):
        ctx.what = what
        return compute()

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.what} has no derivative")
