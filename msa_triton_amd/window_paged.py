"""Attention of new tokens over a paged cache: with a sliding window and visible first tokens, and of a drafted tree.

``m3_window_attention`` for serving (single tokens, drafted runs, a prompt's next part), and the verification of a
tree of drafted tokens, whose nodes see the cached tokens and their own ancestors. Caches, pages and lengths are those of
the other paged operators; the new tokens are in the cache already (``m3_cache_append``). One C call
(``msa_window_attn_paged``: a launch that shares all sequences' keys out evenly over the GPU whatever their lengths, and
one that joins the parts of rows that were split). Lengths, page entries and parents are read on the device
only. No gradients: differentiating the outputs raises.
"""

from __future__ import annotations

import struct

import torch

from . import _lib
from .derivatives import NoBackward, wanted
from .layout import PackedSequences
from .paged import check_kv_caches, check_pages, sixteen_bit
from .window_attention import check_scale, check_window

_pack_strides = struct.Struct("6q").pack
MAX_TREE_NODES = 512


def _attend(name, q, k_cache, v_cache, page_table, cu_seqlens, context_lens, parents, window_size, sink_tokens, scale,
            k_scale, v_scale, return_lse):
    if q.ndim != 3 or q.shape[1] < 1 or q.shape[2] < 1:
        raise ValueError("expected q[T,Hq,D] with Hq, D > 0")
    total, heads, dim = q.shape
    sixteen_bit(q, name)
    dtype, device = q.dtype, q.device
    groups = k_cache.shape[1] if k_cache.ndim == 4 else 0
    if groups < 1 or heads % groups:
        raise ValueError("k_cache must be [pages, G, page size, D] with Hq a positive multiple of G")
    page, strides, fp8 = check_kv_caches(k_cache, v_cache, k_scale, v_scale, groups, dim, dtype, device)
    window, sinks = check_window(window_size, sink_tokens)
    effective_scale = check_scale(scale, dim)
    pages, cu, num_seqs, context, page_map = check_pages(page_table, cu_seqlens, context_lens, total, page, k_cache, device)
    if isinstance(cu_seqlens, PackedSequences):
        longest = cu_seqlens.max_seqlen
    else:
        bounds = cu_seqlens.tolist()
        longest = max(b - a for a, b in zip(bounds, bounds[1:]))
    if parents is not None:
        if not isinstance(parents, torch.Tensor) or parents.dtype != torch.int32:
            raise TypeError("parents must be int32")
        if parents.shape != (total,):
            raise ValueError("parents must hold one entry per token")
        if parents.device != device:
            raise ValueError("parents must be on the input device")
        parents = parents.contiguous()
    if dim % 16 or dim > 256:
        raise NotImplementedError(f"{name} takes head dims that are multiples of 16 up to 256")
    if max(k_cache.stride(2), v_cache.stride(2)) >= 1 << 27:
        raise NotImplementedError(f"{name} takes caches whose slots lie fewer than 2^27 values apart")
    if total * (heads // groups) >= 0x7FFF0000:
        raise NotImplementedError(f"{name} takes fewer than 2^31 rows of a key head")
    if parents is not None and longest > MAX_TREE_NODES:
        raise NotImplementedError(f"{name} takes trees of up to {MAX_TREE_NODES} nodes")
    _lib.require_gpu(q, name)
    q = q.contiguous()
    if q.data_ptr() % 16:
        q = q.clone()
    out = torch.empty_like(q, requires_grad=False)
    lse = torch.empty((total, heads), dtype=torch.float32, device=device) if return_lse else None
    if total:
        lib = _lib.lib()
        size = lib.msa_window_attn_paged_workspace_bytes(total, num_seqs, longest, heads, groups, dim, page_map[2], page,
                                                         window, sinks)
        workspace = torch.empty(size, dtype=torch.uint8, device=device)
        with _lib.on_device(device):
            status = lib.msa_window_attn_paged(
                q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _lib.DTYPE_CODE[dtype], fp8,
                k_scale.data_ptr() if fp8 else None, v_scale.data_ptr() if fp8 else None, _pack_strides(*strides),
                None if parents is None else parents.data_ptr(), *page_map, cu.data_ptr(), num_seqs, longest,
                context.data_ptr(), total, heads, groups, dim, window, sinks, effective_scale, workspace.data_ptr(), size,
                out.data_ptr(), lse.data_ptr() if return_lse else None, _lib.stream_of(device))
        _lib.check(status, "msa_window_attn_paged")
    if wanted(q, k_cache, v_cache) or fp8 and wanted(k_scale, v_scale):
        out, lse = NoBackward.apply(name, (out, lse), q, k_cache, v_cache, k_scale, v_scale)
    return (out, lse) if return_lse else out


def m3_window_attention_paged(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    cu_seqlens,
    context_lens: torch.Tensor,
    *,
    window_size: int | None,
    sink_tokens: int = 0,
    scale: float | None = None,
    k_scale: torch.Tensor | None = None,
    v_scale: torch.Tensor | None = None,
    return_lse: bool = False,
):
    """Attend ``q[T,Hq,D]`` to paged caches ``[P,G,page,D]`` (``G`` divides ``Hq``): ``out[T,Hq,D]``.

    A new token sees the keys up to its own slot: the last ``window_size`` of them (None: all) and the first
    ``sink_tokens``. 8-bit caches (``torch.float8_e4m3fn``) come with ``k_scale`` and ``v_scale`` (fp32 ``[P,G]``). Keys
    in missing pages do not exist (pages that lie wholly between the first tokens and the window may be given
    back); rows without keys, and those of an absent sequence (negative ``context_lens``), give zero output and an LSE of
    -inf. Values that are not finite give what the formula gives, as in ``m3_sparse_attention_paged``; a row whose logits are
    all -inf has an output of 0. ``D`` is a multiple of 16 up to 256. How softmax weights are rounded goes by the
    longest sequence of the call, so a request's last bits depend on its batch."""
    return _attend("m3_window_attention_paged", q, k_cache, v_cache, page_table, cu_seqlens, context_lens, None, window_size,
                   sink_tokens, scale, k_scale, v_scale, return_lse)


def m3_tree_attention_paged(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    cu_seqlens,
    context_lens: torch.Tensor,
    parents: torch.Tensor,
    *,
    window_size: int | None = None,
    sink_tokens: int = 0,
    scale: float | None = None,
    k_scale: torch.Tensor | None = None,
    v_scale: torch.Tensor | None = None,
    return_lse: bool = False,
):
    """``m3_window_attention_paged`` where each sequence's new tokens are the nodes of a tree (or several).

    ``parents`` (int32 ``[T]``) holds each node's parent by its place among its sequence's new tokens; parents come in
    front of their children, and anything outside ``[0, own place)`` (-1, say) is a child of the context. A node
    sees the cached tokens and, of the new ones, itself and its ancestors. It lies in slot ``context + place`` of the cache,
    and its position, by which window and first tokens are counted, is ``context + depth`` (the position to rotate it by).
    Up to 512 nodes a sequence."""
    if parents is None:
        raise TypeError("parents must be int32")
    return _attend("m3_tree_attention_paged", q, k_cache, v_cache, page_table, cu_seqlens, context_lens, parents,
                   window_size, sink_tokens, scale, k_scale, v_scale, return_lse)
