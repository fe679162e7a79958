"""Whether a call's derivatives are asked for: what decides between an operator's autograd function and the shorter
path without one."""

from __future__ import annotations

import torch
from torch.autograd import forward_ad


_grad_enabled = torch.is_grad_enabled


def forward_mode() -> bool:
    """Inside ``forward_ad.dual_level``: a tensor may carry a tangent, which ``requires_grad`` does not tell and grad
    mode does not stop. (Nowhere else has one a tangent.)"""
    return forward_ad._current_level >= 0


def wanted(*tensors: torch.Tensor | None) -> bool:
    """Whether the call goes through its autograd function: a gradient will be asked for, or a tangent may be there
    (the functions have no forward-mode rule and raise at one)."""
    for x in tensors:
        if x is not None and x.requires_grad:
            return _grad_enabled() or forward_ad._current_level >= 0
    return forward_ad._current_level >= 0


def _has_tangent(x: torch.Tensor) -> bool:
    try:
        return forward_ad.unpack_dual(x).tangent is not None
    except RuntimeError:  # inside a registered operator, below autograd: nothing to read there
        return False


def refuse_tangents(name: str, *tensors: torch.Tensor | None) -> None:
    """Raise where a tensor carries a tangent: registered operators drop it silently."""
    if forward_mode() and any(x is not None and _has_tangent(x) for x in tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative (jvp)")


def refuse_gradients(name: str, *tensors: torch.Tensor | None) -> None:
    """Raise where a derivative would be asked for of an operator that writes its results in place and has none."""
    refuse_tangents(name, *tensors)
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in tensors):
        raise RuntimeError(f"{name} has no gradients: call it under torch.no_grad() or with detached inputs")


class NoBackward(torch.autograd.Function):
    """``outs``, what an operator without a backward pass made of ``tensors``, in their graph: differentiating it raises,
    where outputs outside the graph would end a gradient silently."""

    @staticmethod
    def forward(ctx, name, outs, *tensors):
        ctx.name = name
        return outs

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.name} has no gradients")
