"""No window or tree operator returns outputs whose derivative was asked for and silently left out. On the CPU, with C calls
that do nothing: what is tested is the path that a call takes."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import msa_triton_amd as msa
from msa_triton_amd import custom_ops
from tests.test_derivatives_are_not_dropped import no_kernels  # noqa: F401

OPS = pytest.mark.parametrize("ops", (msa, custom_ops), ids=("eager", "library"))


def _call(name, ops):
    """(tensors that may be differentiated, a call of them)"""
    q, k, v = (torch.ones(3, h, 16, dtype=torch.bfloat16) for h in (4, 2, 2))
    cu, ctx = torch.tensor([0, 3], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    if name == "packed":
        return [q, k, v], lambda *x: ops.m3_window_attention(*x, cu, 3, window_size=2, return_lse=True)
    table = torch.zeros(1, 2, dtype=torch.int32)
    kc, vc = (torch.zeros(2, 2, 16, 16, dtype=torch.bfloat16) for _ in range(2))
    if name == "paged":
        return [q, kc, vc], lambda *x: ops.m3_window_attention_paged(*x, table, cu, ctx, window_size=2, return_lse=True)
    parents = torch.full((3,), -1, dtype=torch.int32)
    return [q, kc, vc], lambda *x: ops.m3_tree_attention_paged(*x, table, cu, ctx, parents, return_lse=True)


@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("name", ("packed", "paged", "tree"))
@OPS
def test_gradients(ops, name, which, no_kernels):  # noqa: F811
    x, call = _call(name, ops)
    assert not any(y.requires_grad for y in call(*x))
    x[which].requires_grad_()
    with torch.no_grad():
        assert not any(y.requires_grad for y in call(*x))
    out, lse = call(*x)
    assert out.requires_grad
    if name == "packed":
        assert not lse.requires_grad
        out.float().sum().backward()
        assert [y.grad is not None for y in x] == [i == which for i in range(3)]
        return
    with pytest.raises(RuntimeError, match="no gradients|no autograd formula"):
        out.float().sum().backward()


@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("name", ("packed", "paged", "tree"))
@pytest.mark.parametrize("grad", (False, True))
@OPS
def test_forward_mode(ops, name, which, grad, no_kernels):  # noqa: F811
    x, call = _call(name, ops)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        call(*x)  # (no tangent: as outside)
        x[which] = forward_ad.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(NotImplementedError, match="jvp"):
            call(*x)
