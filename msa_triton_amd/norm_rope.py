"""RMS norm of query and key heads with the position rotation, in one pass, with autograd.

The projections' outputs become what the indexer and the attention take: per head
``y = rotate(x / sqrt(mean(x^2) + eps) * weight)``, with the rotation of a token's position over
the first ``rotary_dim`` dims (pairs ``i``, ``i + rotary_dim / 2``). Positions come from the
packed metadata that every operator takes, plus the tokens that a cache already holds
(``context_lens``), so one call serves training, prompts and single tokens.

Execution: ``msa_qk_norm_rope`` / ``msa_qk_norm_rope_bwd`` (one launch, and a second one for the
gradients of the weights). fp32 arithmetic whatever the input type, each output rounded once.
Saved state is the inputs; the backward recomputes the norm from them.
"""

from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .derivatives import wanted
from .layout import context_of, packed_tokens

_TYPES = (torch.bfloat16, torch.float16, torch.float32)
MAX_HEAD_DIM = 512


def rope_table(num_positions: int, rotary_dim: int, *, base: float = 10000.0, device=None) -> torch.Tensor:
    """cos and sin of ``position * base**(-2 i / rotary_dim)``, fp32 ``[num_positions, rotary_dim]``:
    the ``rotary_dim / 2`` cosines of a position, then its sines. Angles are formed in float64 (fp32 angles of
    far positions are off by whole radians)."""
    if not isinstance(num_positions, int) or num_positions < 0:
        raise ValueError("num_positions must be a nonnegative integer")
    if not isinstance(rotary_dim, int) or rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be a positive even integer")
    if not (math.isfinite(base) and base > 0):
        raise ValueError("base must be positive and finite")
    half = rotary_dim // 2
    freq = float(base) ** (-torch.arange(half, dtype=torch.float64, device=device) / half)
    angle = torch.arange(num_positions, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def check_table(cos_sin, head_dim, device):
    """The rotation table's checks: (contiguous table or None, rows, rotary dim)."""
    if cos_sin is None:
        return None, 0, 0
    shape = cos_sin.shape
    if len(shape) != 2 or cos_sin.dtype != torch.float32 or shape[1] % 2:
        raise ValueError("cos_sin must be fp32 [positions, rotary_dim] with an even rotary_dim")
    rows, rot = shape
    if rot > head_dim:
        raise ValueError("rotary_dim must not exceed the head dimension")
    if cos_sin.device != device:
        raise ValueError("cos_sin must be on the input device")
    return cos_sin.contiguous(), rows, rot


def check_weight(weight, name, dim, dtype, device):
    if weight is None or weight.shape != (dim,) or (weight.dtype != dtype and weight.dtype != torch.float32):
        raise ValueError(f"{name} must be [head dim], of the input dtype or fp32")
    if weight.device != device:
        raise ValueError(f"{name} must be on the input device")


def _unit_rows(x):
    return x if x is None or x.stride(2) == 1 else x.contiguous()


def _call_args(q, k, wq, wk, table, rows, rot, cu, num_seqs, context, eps):
    """The arguments that both C calls begin with."""
    total, heads, dim = q.shape
    return (q.data_ptr(), *q.stride()[:2], heads, *((None, 0, 0, 0) if k is None else
                                                    (k.data_ptr(), *k.stride()[:2], k.shape[1])),
            _lib.DTYPE_CODE[q.dtype], wq.data_ptr(), None if wk is None else wk.data_ptr(), _lib.DTYPE_CODE[wq.dtype],
            None if table is None else table.data_ptr(), rows, rot, cu.data_ptr(), num_seqs,
            None if context is None else context.data_ptr(), total, dim, eps)


def _forward(q, k, call):
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format, requires_grad=False)
    k_out = None if k is None else torch.empty_like(k, memory_format=torch.contiguous_format, requires_grad=False)
    if q.shape[0]:
        with _lib.on_device(q.device):
            status = _lib.lib().msa_qk_norm_rope(*call, q_out.data_ptr(), None if k is None else k_out.data_ptr(),
                                                 _lib.stream_of(q.device))
        _lib.check(status, "msa_qk_norm_rope")
    return q_out, k_out


def _side_gradients(x, w, g, need_x, need_w):
    """(incoming gradient, dx, dw, heads) of one side, as the backward call takes them: 0 heads where nothing of it is
    needed or no gradient came in."""
    if x is None or g is None or not (need_x or need_w):
        return None, None, None, 0
    if g.dtype != x.dtype or not g.is_contiguous():
        g = g.to(x.dtype).contiguous()
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need_x else None
    dw = (torch.empty_like if x.shape[0] else torch.zeros_like)(w) if need_w else None
    return g, dx, dw, x.shape[1]


def _backward(q, k, wq, wk, call, dq_out, dk_out, need):
    """Gradients (q, k, q_weight, k_weight), None where not needed or no gradient came in."""
    gq, dq, dwq, hq = _side_gradients(q, wq, dq_out, need[0], need[2])
    gk, dk, dwk, hk = _side_gradients(k, wk, dk_out, need[1], need[3])
    total, _, dim = q.shape
    if total and (hq or hk):
        lib = _lib.lib()
        size, workspace = 0, None
        if dwq is not None or dwk is not None:
            size = lib.msa_qk_norm_rope_bwd_workspace_bytes(total, hq, hk, dim)
            workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
        with _lib.on_device(q.device):
            status = lib.msa_qk_norm_rope_bwd(
                *call, *[None if x is None else x.data_ptr() for x in (gq, gk, dq, dk, dwq, dwk, workspace)], size,
                _lib.stream_of(q.device))
        _lib.check(status, "msa_qk_norm_rope_bwd")
    return dq, dk, dwq, dwk


class _NormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, table, cu, context, sizes, eps):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, wq, wk, table, cu, context)
        ctx.sizes, ctx.eps = sizes, eps
        return _forward(q, k, _call_args(q, k, wq, wk, table, *sizes[:2], cu, sizes[2], context, eps))

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        # (checkpointing and offloading hand back other tensors than the ones that were saved)
        q, k, wq, wk, table, cu, context = ctx.saved_tensors
        q, k = _unit_rows(q), _unit_rows(k)
        call = _call_args(q, k, wq, wk, table, *ctx.sizes[:2], cu, ctx.sizes[2], context, ctx.eps)
        return (*_backward(q, k, wq, wk, call, dq_out, dk_out, ctx.needs_input_grad), None, None, None, None, None)


def _validate(q, k, q_weight, k_weight, cos_sin, cu_seqlens, eps, context_lens):
    """m3_qk_norm_rope's checks; returns the kernels' arguments."""
    if q.ndim != 3 or (k is not None and k.ndim != 3):
        raise ValueError("q and k must be rank-3 TND tensors")
    total, heads, dim = q.shape
    if heads < 1 or dim < 1 or (k is not None and (k.shape[0] != total or k.shape[1] < 1 or k.shape[2] != dim)):
        raise ValueError("expected q[T,Hq,D] and k[T,Hkv,D] with positive heads and D")
    dtype, device = q.dtype, q.device
    if dtype not in _TYPES:
        raise TypeError("q must have BF16, FP16, or FP32 dtype")
    if k is not None and (k.dtype != dtype or k.device != device):
        raise ValueError("q and k must share dtype and device")
    check_weight(q_weight, "q_weight", dim, dtype, device)
    if k is None:
        if k_weight is not None:
            raise ValueError("k_weight without k")
    else:
        check_weight(k_weight, "k_weight", dim, dtype, device)
        if k_weight.dtype != q_weight.dtype:
            raise ValueError("q_weight and k_weight must share a dtype")
    table, rows, rot = check_table(cos_sin, dim, device)
    if not (isinstance(eps, (int, float)) and math.isfinite(eps) and eps >= 0):
        raise ValueError("eps must be nonnegative and finite")
    cu, num_seqs = packed_tokens(cu_seqlens, total, device)
    context = context_of(context_lens, num_seqs, device)
    if dim > MAX_HEAD_DIM:
        raise NotImplementedError(f"m3_qk_norm_rope takes head dims up to {MAX_HEAD_DIM}")
    _lib.require_gpu(q, "m3_qk_norm_rope")
    return (_unit_rows(q), _unit_rows(k), q_weight.contiguous(), None if k is None else k_weight.contiguous(), table,
            rows, rot, cu, num_seqs, context, float(eps))


def m3_qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor | None,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor | None,
    cos_sin: torch.Tensor | None,
    cu_seqlens,
    *,
    eps: float = 1e-6,
    context_lens: torch.Tensor | None = None,
):
    """Per-head RMS norm of ``q[T,Hq,D]`` and ``k[T,Hkv,D]`` with their weights ``[D]``, then the
    rotation of each token's position: ``(q_out, k_out)``, differentiable in all four.

    ``k`` (and ``k_weight``) may be None; then ``k_out`` is None. ``cos_sin`` (``rope_table``) is fp32
    ``[positions, rotary_dim]``; None leaves the rotation out. A token's position is its offset in its
    packed sequence plus ``context_lens`` of that sequence (int32 ``[N]`` on the device, default 0); where the
    table has no row for it, the rotated dims are NaN. Token and head strides of ``q`` and ``k`` are free
    (slices of a fused projection are read in place). The index heads go through the same call."""
    q, k, wq, wk, table, rows, rot, cu, num_seqs, context, eps = _validate(q, k, q_weight, k_weight, cos_sin, cu_seqlens,
                                                                           eps, context_lens)
    if wanted(q, k, wq, wk):
        return _NormRope.apply(q, k, wq, wk, table, cu, context, (rows, rot, num_seqs), eps)
    return _forward(q, k, _call_args(q, k, wq, wk, table, rows, rot, cu, num_seqs, context, eps))
