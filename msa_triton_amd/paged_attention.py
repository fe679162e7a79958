"""Sparse attention of new tokens over the selected blocks of a paged cache.

``m3_sparse_attention`` for serving: a token attends to the keys up to its position of the blocks that its
group selected (``m3_index_score_topk_paged``), read from a 16-bit cache or an 8-bit one with a scale for
each page and head. One C call (``msa_attn_paged``: a launch that reads the selected keys and values, and, for
few rows, a second one that joins the parts of a row). The new tokens are in the cache already
(``m3_cache_append``). Made for the few tokens of a decoding step: a prompt goes through the packed operators, and
one behind a cached prefix through this call, where each token reads its blocks on its own (512 tokens behind 8192, 32
heads, 16 blocks: 169 us). No gradients: differentiating the outputs raises.
"""

from __future__ import annotations

import math
import struct

import torch

from . import _lib
from .derivatives import NoBackward, wanted
from .paged import check_kv_caches, check_pages, sixteen_bit

_pack_strides = struct.Struct("6q").pack


def m3_sparse_attention_paged(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    indices: torch.Tensor,
    page_table: torch.Tensor,
    cu_seqlens,
    context_lens: torch.Tensor,
    *,
    block_size: int = 128,
    scale: float | None = None,
    k_scale: torch.Tensor | None = None,
    v_scale: torch.Tensor | None = None,
    return_lse: bool = False,
):
    """Attend ``q[T,Hq,D]`` to the selected blocks of paged caches ``[P,G,page,D]``: ``out[T,Hq,D]``.

    ``indices[T,G,K]`` (int32) holds sequence-local block ids with ``-1`` padding, as the selection gives them; ids
    behind the token and repeated ids count for nothing. Each contiguous group of ``Hq / G`` query heads shares a
    selection. 8-bit caches (``torch.float8_e4m3fn``) come with ``k_scale`` and ``v_scale`` (fp32 ``[P,G]``). Keys in
    missing pages do not exist; rows without keys, and those of an absent sequence (negative ``context_lens``),
    give zero output and an LSE of -inf. Values that are not finite give what the formula gives: an
    infinity in a visible key's value is the row's in that dim whatever the key's weight (NaN where both signs meet, or the
    weight is 0, of a logit of -inf), a NaN is NaN. ``block_size`` and ``D`` are multiples of 16, ``D`` at most 256."""
    if q.ndim != 3 or q.shape[1] < 1 or q.shape[2] < 1:
        raise ValueError("expected q[T,Hq,D] with Hq, D > 0")
    total, heads, dim = q.shape
    sixteen_bit(q, "m3_sparse_attention_paged")
    dtype, device = q.dtype, q.device
    if indices.ndim != 3 or indices.shape[0] != total or indices.shape[1] < 1 or indices.dtype != torch.int32:
        raise ValueError("indices must be int32 [T,G,K]")
    _, groups, slots = indices.shape
    if heads % groups:
        raise ValueError("Hq must be a positive multiple of G")
    if indices.device != device:
        raise ValueError("indices must be on the input device")
    page, strides, fp8 = check_kv_caches(k_cache, v_cache, k_scale, v_scale, groups, dim, dtype, device)
    if not isinstance(block_size, int) or block_size <= 0:
        raise ValueError("block_size must be a positive integer")
    if block_size > 2147483647:
        raise ValueError("block_size must fit int32 metadata")
    effective_scale = dim ** -0.5 if scale is None else float(scale)
    if not math.isfinite(effective_scale):
        raise ValueError("scale must be finite")
    pages, cu, num_seqs, context, page_map = check_pages(page_table, cu_seqlens, context_lens, total, page, k_cache, device)
    if block_size % 16 or dim % 16 or dim > 256:
        raise NotImplementedError("m3_sparse_attention_paged takes block sizes and head dims that are multiples of 16, "
                                  "head dims up to 256")
    _lib.require_gpu(q, "m3_sparse_attention_paged")
    q, indices = q.contiguous(), indices.contiguous()
    if q.data_ptr() % 16:
        q = q.clone()
    out = torch.empty_like(q, requires_grad=False)
    lse = torch.empty((total, heads), dtype=torch.float32, device=device) if return_lse else None
    if total:
        lib = _lib.lib()
        size = lib.msa_attn_paged_workspace_bytes(total, heads, groups, dim, slots, block_size)
        workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        with _lib.on_device(device):
            status = lib.msa_attn_paged(
                q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _lib.DTYPE_CODE[dtype], fp8,
                k_scale.data_ptr() if fp8 else None, v_scale.data_ptr() if fp8 else None, _pack_strides(*strides),
                indices.data_ptr(), *page_map,
                cu.data_ptr(), num_seqs, context.data_ptr(), total, heads, groups, dim, slots, block_size,
                effective_scale, workspace.data_ptr() if size else None, size, out.data_ptr(),
                lse.data_ptr() if return_lse else None, _lib.stream_of(device))
        _lib.check(status, "msa_attn_paged")
    if wanted(q, k_cache, v_cache) or fp8 and wanted(k_scale, v_scale):
        out, lse = NoBackward.apply("m3_sparse_attention_paged", (out, lse), q, k_cache, v_cache, k_scale, v_scale)
    return (out, lse) if return_lse else out
