"""Block selection of new tokens against the index keys of a paged cache.

``m3_index_score_topk`` for serving: the same scores (the exact block maxima, rounded the same way) and
the same selection, with the keys in pages and the queries at positions behind ``context_lens`` cached
tokens. One C call (``msa_index_score_topk_paged``: a score launch that reads each cached index key once for 16 query
rows of its sequence, and the top-k launch). The new tokens' index keys are in the cache already
(``m3_cache_append``). No gradients: differentiating the scores raises.
"""

from __future__ import annotations

import math

import torch

from . import _lib
from .derivatives import NoBackward, wanted
from .paged import check_cache, check_pages, sixteen_bit


def m3_index_score_topk_paged(
    index_q: torch.Tensor,
    index_cache: torch.Tensor,
    page_table: torch.Tensor,
    cu_seqlens,
    context_lens: torch.Tensor,
    max_seqlen: int,
    *,
    block_size: int = 128,
    scale: float = 1.0,
    topk_blocks: int = 16,
    local_blocks: int = 1,
):
    """Scores and selections of ``index_q[T,G,Di]`` against ``index_cache[P,1,page,Di]``: ``(scores, indices)``.

    ``scores`` is fp32 ``[T, G, ceil(max_seqlen / block_size)]``, ``indices`` int32 ``[T,G,topk_blocks]``, both as
    ``m3_index_score_topk`` gives them for the whole sequences; ``max_seqlen`` bounds a sequence with its new tokens
    (blocks behind it are neither scored nor selected). Keys in missing pages do not exist; rows of an absent
    sequence (negative ``context_lens``) get -inf and -1. ``block_size`` is a multiple of 16, ``Di`` a multiple
    of 8 up to 256, ``T * G`` below 2^28 (2^31 without a selection). Inputs must be finite."""
    if index_q.ndim != 3 or index_q.shape[1] < 1 or index_q.shape[2] < 1:
        raise ValueError("expected index_q[T,G,Di] with G, Di > 0")
    total, groups, dim = index_q.shape
    sixteen_bit(index_q, "m3_index_score_topk_paged")
    dtype, device = index_q.dtype, index_q.device
    page, strides = check_cache(index_cache, "index_cache", (dtype,), 1, dim, device)
    if not isinstance(block_size, int) or block_size <= 0:
        raise ValueError("block_size must be a positive integer")
    if not isinstance(max_seqlen, int) or max_seqlen <= 0:
        raise ValueError("max_seqlen must be a positive integer")
    if block_size > 2147483647 or max_seqlen > 2147483647:
        raise ValueError("block_size and max_seqlen must fit int32 metadata")
    if not isinstance(topk_blocks, int) or topk_blocks < 0:
        raise ValueError("topk_blocks must be a nonnegative integer")
    if not isinstance(local_blocks, int) or not 0 <= local_blocks <= topk_blocks:
        raise ValueError("local_blocks must satisfy 0 <= local_blocks <= topk_blocks")
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    pages, cu, num_seqs, context, page_map = check_pages(page_table, cu_seqlens, context_lens, total, page, index_cache,
                                                         device)
    if block_size % 16 or dim % 8 or dim > 256:
        raise NotImplementedError(
            "m3_index_score_topk_paged takes blocks of a multiple of 16 keys and index dims of a multiple of 8 up to 256")
    _lib.require_gpu(index_q, "m3_index_score_topk_paged")
    q = index_q.contiguous()
    if q.data_ptr() % 16:
        q = q.clone()
    blocks = (max_seqlen + block_size - 1) // block_size
    scores = torch.empty((total, groups, blocks), dtype=torch.float32, device=device)
    indices = torch.empty((total, groups, topk_blocks), dtype=torch.int32, device=device)
    if total:
        with _lib.on_device(device):
            status = _lib.lib().msa_index_score_topk_paged(
                q.data_ptr(), index_cache.data_ptr(), _lib.DTYPE_CODE[dtype], strides[0],
                strides[2], *page_map, cu.data_ptr(), num_seqs, context.data_ptr(),
                total, groups, dim, blocks, block_size, scale, topk_blocks, local_blocks, scores.data_ptr(),
                indices.data_ptr(), _lib.stream_of(device))
        _lib.check(status, "msa_index_score_topk_paged")
    if wanted(index_q, index_cache):
        return NoBackward.apply("m3_index_score_topk_paged", (scores, indices), index_q, index_cache)
    return scores, indices
