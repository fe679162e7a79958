"""Whether a call's derivatives are asked for: what decides between an operator's autograd function and the shorter
path without one."""

from __future__ import annotations

import torch
from torch.autograd import forward_ad


def forward_mode() -> bool:
    """Inside ``forward_ad.dual_level``: a tensor may carry a tangent, which ``requires_grad`` does not tell and grad
    mode does not stop. (Nowhere else has one a tangent.)"""
    return forward_ad._current_level >= 0


def wanted(*tensors: torch.Tensor | None) -> bool:
    """Whether the call goes through its autograd function: a gradient will be asked for, or a tangent may be there
    (the functions have no forward-mode rule and raise at one)."""
    if forward_mode():
        return True
    if not torch.is_grad_enabled():
        return False
    for x in tensors:
        if x is not None and x.requires_grad:
            return True
    return False


def refuse_tangents(name: str, *tensors: torch.Tensor | None) -> None:
    """Raise where a tensor carries a tangent: registered operators drop it silently."""
    if forward_mode() and any(x is not None and forward_ad.unpack_dual(x).tangent is not None for x in tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative (jvp)")
