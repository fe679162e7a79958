"""Causal attention of packed sequences with a sliding window and a few first tokens that stay visible, with autograd.

The attention of the layers that stand beside the block-sparse ones: token ``i`` of a sequence sees the keys
``j <= i`` with ``i - j < window_size``, and the first ``sink_tokens`` tokens; without a window it is plain causal
attention. Packed tensors and conventions are those of ``m3_sparse_attention``.

Execution: ``msa_window_attn_fwd`` (one launch), ``msa_window_attn_bwd`` (three launches: delta, dQ, dK and dV; a fourth
where first tokens are seen from behind the window). Matrix products on the input type, everything between them
in fp32, all sums in fixed orders. Saved state is q, k, v, out, the lse and, in 16 bits, what the rounding of out left
out (delta = dO . O is formed from both).
"""

from __future__ import annotations

import struct

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .derivatives import wanted
from .layout import PackedSequences, packed_tokens, sequence_lengths

_TYPES = (torch.bfloat16, torch.float16, torch.float32)
MAX_HEAD_DIM = 256


def check_window(window_size, sink_tokens):
    """``window_size`` as the kernels take it (0: none)."""
    if window_size is not None and (not isinstance(window_size, int) or isinstance(window_size, bool) or window_size <= 0):
        raise ValueError("window_size must be a positive integer or None")
    if not isinstance(sink_tokens, int) or isinstance(sink_tokens, bool) or sink_tokens < 0:
        raise ValueError("sink_tokens must be a nonnegative integer")
    most = 2147483647
    return 0 if window_size is None or window_size >= most else window_size, min(sink_tokens, most)


def check_scale(scale, dim):
    """The scale of a call. Kernels hold scale * log2(e) in fp32, where it has to be finite as well."""
    scale = dim ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= 2e38:
        raise ValueError("scale must be finite, of at most 2e38.")
    return scale


def aligned_rows(x, near_heads=0):
    """A rank-3 tensor whose rows are contiguous, 16-byte aligned and near each other, as the kernels address them, and its token
    and head strides: 33 tokens within 2^30 elements, with ``near_heads`` heads where a tile's rows are of so many."""
    of_token, of_head, of_dim = x.stride()
    tokens, heads, dim = x.shape
    if tokens == 1:  # (a stride that nothing steps over may be anything)
        of_token = 0
    if heads == 1:
        of_head = 0
    unit = 16 // x.element_size()
    if ((of_dim == 1 or dim == 1) and of_token % unit == 0 and of_head % unit == 0 and x.data_ptr() % 16 == 0
            and of_token < 1 << 25 and of_head < 1 << 30 and 33 * of_token + near_heads * of_head < 1 << 30):
        return x, of_token, of_head
    x = x.contiguous()
    if x.data_ptr() % 16:
        x = x.clone()
    return x, heads * dim, dim


_pack6, _pack8 = struct.Struct("6q").pack, struct.Struct("8q").pack


def _forward(q, k, v, cu, num_seqs, window, sinks, scale, need_lse, need_grad):
    """(out, lse or None, out_lo or None)."""
    total, heads, dim = q.shape
    groups = k.shape[1]
    out = torch.empty((total, heads, dim), dtype=q.dtype, device=q.device)
    lse = torch.empty((total, heads), dtype=torch.float32, device=q.device) if need_lse or need_grad else None
    lo = torch.empty_like(out) if need_grad and q.dtype != torch.float32 else None
    if total:
        q, *of_q = aligned_rows(q, heads // groups)
        k, *of_k = aligned_rows(k)
        v, *of_v = aligned_rows(v)
        with _lib.on_device(q.device):
            status = _lib.lib().msa_window_attn_fwd(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), _lib.DTYPE_CODE[q.dtype], _pack6(*of_q, *of_k, *of_v),
                cu.data_ptr(), num_seqs, total, heads, groups, dim, window, sinks, scale, out.data_ptr(), _lib.ptr(lo),
                _lib.ptr(lse), _lib.stream_of(q.device))
        _lib.check(status, "msa_window_attn_fwd")
    return out, lse, lo


def _backward(q, k, v, cu, num_seqs, longest, window, sinks, scale, out, lo, lse, grad, need_q, need_k, need_v):
    """(dq, dk, dv), None where not needed."""
    total, heads, dim = q.shape
    groups, device = k.shape[1], q.device
    dq = torch.empty(q.shape, dtype=q.dtype, device=device) if need_q else None
    dk = torch.empty(k.shape, dtype=q.dtype, device=device) if need_k else None
    dv = torch.empty(v.shape, dtype=q.dtype, device=device) if need_v else None
    if total and (need_q or need_k or need_v):
        lib = _lib.lib()
        q, *of_q = aligned_rows(q, heads // groups)
        k, *of_k = aligned_rows(k)
        v, *of_v = aligned_rows(v)
        grad, *of_grad = aligned_rows(grad, heads // groups)
        out = out.contiguous()
        lse = lse.contiguous()
        lo = lo if lo is None else lo.contiguous()
        code = _lib.DTYPE_CODE[q.dtype]
        size = lib.msa_window_attn_bwd_workspace_bytes(code, total, num_seqs, longest, heads, groups, dim, window, sinks)
        workspace = torch.empty(size, dtype=torch.uint8, device=device)
        with _lib.on_device(device):
            status = lib.msa_window_attn_bwd(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), code, _pack8(*of_q, *of_k, *of_v, *of_grad), cu.data_ptr(),
                num_seqs, longest, total, heads, groups, dim, window, sinks, scale, out.data_ptr(), _lib.ptr(lo),
                lse.data_ptr(), grad.data_ptr(), _lib.ptr(dq), _lib.ptr(dk), _lib.ptr(dv), workspace.data_ptr(), size,
                _lib.stream_of(device))
        _lib.check(status, "msa_window_attn_bwd")
    return dq, dk, dv


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu, num_seqs, longest, window, sinks, scale):
        out, lse, lo = _forward(q, k, v, cu, num_seqs, window, sinks, scale, True, True)
        ctx.save_for_backward(q, k, v, cu, out, lo, lse)
        ctx.call = num_seqs, longest, window, sinks, scale
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, grad_lse):
        q, k, v, cu, out, lo, lse = ctx.saved_tensors
        num_seqs, longest, window, sinks, scale = ctx.call
        return (*_backward(q, k, v, cu, num_seqs, longest, window, sinks, scale, out, lo, lse, grad.to(q.dtype),
                           *ctx.needs_input_grad[:3]), None, None, None, None, None, None)


def _validate(q, k, v, cu_seqlens, max_seqlen, window_size, sink_tokens, scale):
    """The checked call: cu_seqlens on the device, sequences, the longest of them, window, sinks and scale."""
    if q.ndim != 3 or k.ndim != 3 or v.shape != k.shape:
        raise ValueError("Expected q[T,Hq,D] and matching k/v[T,G,D].")
    total, heads, dim = q.shape
    if k.shape[0] != total or k.shape[2] != dim:
        raise ValueError("q/k/v must have matching token and head dimensions.")
    if k.shape[1] <= 0 or heads <= 0 or heads % k.shape[1]:
        raise ValueError("Hq must be a positive multiple of G.")
    if dim <= 0:
        raise ValueError("Head dimension must be positive.")
    if q.dtype not in _TYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("q/k/v must share a BF16, FP16, or FP32 dtype.")
    if k.device != q.device or v.device != q.device:
        raise ValueError("All inputs must reside on the same device.")
    if not isinstance(max_seqlen, int) or max_seqlen <= 0:
        raise ValueError("max_seqlen must be a positive integer.")
    window, sinks = check_window(window_size, sink_tokens)
    if isinstance(cu_seqlens, PackedSequences):
        cu, num_seqs = packed_tokens(cu_seqlens, total, q.device)
        longest = cu_seqlens.max_seqlen
    else:
        if not isinstance(cu_seqlens, torch.Tensor):
            raise TypeError("cu_seqlens must be a tensor or PackedSequences")
        lengths = sequence_lengths(cu_seqlens, total)
        if cu_seqlens.device != q.device:
            raise ValueError("All inputs must reside on the same device.")
        cu, num_seqs, longest = cu_seqlens.contiguous(), len(lengths), max(lengths)
    if longest > max_seqlen:
        raise ValueError("max_seqlen is smaller than an actual sequence.")
    effective_scale = check_scale(scale, dim)
    if dim > MAX_HEAD_DIM or dim % 8:
        raise NotImplementedError("m3_window_attention takes head dims that are multiples of 8 up to 256")
    if heads * dim >= 1 << 24:
        raise NotImplementedError("m3_window_attention takes fewer than 2^24 values a token")
    if total * (heads // k.shape[1]) >= 0x7FFF0000:
        raise NotImplementedError("m3_window_attention takes fewer than 2^31 rows of a key head")
    _lib.require_gpu(q, "m3_window_attention")
    return cu, num_seqs, longest, window, sinks, effective_scale


def m3_window_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens,
    max_seqlen: int,
    *,
    window_size: int | None,
    sink_tokens: int = 0,
    scale: float | None = None,
    return_lse: bool = False,
):
    """Causal attention of packed ``q[T,Hq,D]``, ``k[T,G,D]``, ``v[T,G,D]``: ``out[T,Hq,D]``.

    Token ``i`` of a sequence sees its last ``window_size`` keys, itself among them (None: all), and the sequence's
    first ``sink_tokens`` keys. Each contiguous group of ``Hq / G`` query heads shares a key head. Rows must be
    contiguous and 16-byte aligned to be read in place (slices of a fused projection are); others are copied. The
    optional natural-log LSE is FP32 and non-differentiable. What is not finite reaches the rows that see it and
    no others: a value that is an infinity makes its dim one whatever the weight (NaN where both signs meet). A row whose
    logits are all -inf has an output of 0 and an LSE of -inf, as in ``m3_sparse_attention``. ``scale`` (default ``D ** -0.5``) is at
    most 2e38 in magnitude. Head dims are multiples of 8 up to 256."""
    cu, num_seqs, longest, window, sinks, effective_scale = _validate(q, k, v, cu_seqlens, max_seqlen, window_size,
                                                                      sink_tokens, scale)
    if wanted(q, k, v):
        out, lse = _WindowAttention.apply(q, k, v, cu, num_seqs, longest, window, sinks, effective_scale)
    else:
        out, lse, _ = _forward(q, k, v, cu, num_seqs, window, sinks, effective_scale, return_lse, False)
    return (out, lse) if return_lse else out
