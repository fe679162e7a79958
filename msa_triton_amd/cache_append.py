"""New tokens into a paged cache: keys normed and rotated on the way, values as they are.

The step between a layer's projections and its attention when a cache serves the tokens in front:
``m3_qk_norm_rope`` prepares the queries, this call writes what the queries will read. The keys and values
go to a cache of their own type or to an 8-bit one (e4m3 with a power-of-two scale for each page and
head), the index keys to a 16-bit one (their scores decide which blocks are read, and equal scores have to stay
equal). One launch (``msa_cache_append``); the caches are written in place.
"""

from __future__ import annotations

import math
import struct

import torch

from . import _lib
from .derivatives import forward_mode, refuse_gradients
from .norm_rope import check_table, check_weight
from .paged import check_cache, check_kv_caches, check_pages, sixteen_bit, unit_rows

_pack_strides = struct.Struct("13q").pack
_increment_version = torch.autograd.graph.increment_version


def m3_cache_append(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    cu_seqlens,
    context_lens: torch.Tensor,
    *,
    index_k: torch.Tensor | None = None,
    index_cache: torch.Tensor | None = None,
    k_scale: torch.Tensor | None = None,
    v_scale: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    index_weight: torch.Tensor | None = None,
    cos_sin: torch.Tensor | None = None,
    eps: float = 1e-6,
) -> None:
    """Write ``k``, ``v`` (``[T,H,D]``) and ``index_k`` (``[T,1,Di]``) of new tokens into paged caches
    ``[P,H,page,D]`` (``index_cache``: ``[P,1,page,Di]``), behind ``context_lens`` tokens of each sequence.

    Keys are normed where ``k_weight`` is given and rotated where ``cos_sin`` (``rope_table``) is; index keys
    likewise with ``index_weight``. In an 8-bit cache (``torch.float8_e4m3fn``) a value is its byte times
    ``k_scale`` / ``v_scale`` ``[P,H]``, the smallest power of two that lets the page's largest magnitude fit; the
    scale of a page that already holds tokens only grows, and they are then rounded again. A page whose
    first new token is at slot 0 starts over. Values that are not finite are stored as NaN.

    Tokens of missing pages (entries outside ``[0, P)``, or past the table) and of absent sequences
    (negative ``context_lens``) are left out. No two new tokens may share a slot; in 8 bits no two
    sequences may append to one page. D and Di: multiples of 16 up to 256. No gradients: the caches are
    written outside the graph, so a call whose inputs require grad is refused in grad mode (``torch.no_grad()`` or
    detached inputs)."""
    if (k.requires_grad or v.requires_grad or k_cache.requires_grad or v_cache.requires_grad or forward_mode() or
            (index_k is not None and (index_k.requires_grad or index_cache is not None and index_cache.requires_grad)) or
            (k_weight is not None and k_weight.requires_grad) or (index_weight is not None and index_weight.requires_grad)):
        refuse_gradients("m3_cache_append", k, v, index_k, k_weight, index_weight, k_cache, v_cache, index_cache)
    if k.ndim != 3 or v.shape != k.shape or k.shape[1] < 1 or k.shape[2] < 1:
        raise ValueError("expected k and v [T,H,D] of one shape with H, D > 0")
    total, heads, dim = k.shape
    sixteen_bit(k, "m3_cache_append")
    dtype, device = k.dtype, k.device
    if v.dtype != dtype or v.device != device:
        raise ValueError("k and v must share dtype and device")
    page, of_kv, fp8 = check_kv_caches(k_cache, v_cache, k_scale, v_scale, heads, dim, dtype, device)
    if (index_k is None) != (index_cache is None):
        raise ValueError("index_k and index_cache go together")
    index_dim, of_index = 0, (0, 0, 0)
    if index_k is not None:
        index_dim = index_k.shape[-1] if index_k.ndim else 0
        if index_k.shape != (total, 1, index_dim) or index_dim < 1:
            raise ValueError("expected index_k [T,1,Di] with Di > 0")
        if index_k.dtype != dtype or index_k.device != device:
            raise ValueError("index_k must share dtype and device with k")
        _, of_index = check_cache(index_cache, "index_cache", (dtype,), 1, index_dim, device)
        if index_cache.shape[0] != k_cache.shape[0] or index_cache.shape[2] != page:
            raise ValueError("index_cache must have the pages of k_cache")
    weight_type = dtype
    if k_weight is not None:
        check_weight(k_weight, "k_weight", dim, dtype, device)
        weight_type = k_weight.dtype
    if index_weight is not None:
        if index_k is None:
            raise ValueError("index_weight without index_k")
        check_weight(index_weight, "index_weight", index_dim, dtype, device)
        if k_weight is not None and weight_type != index_weight.dtype:
            raise ValueError("k_weight and index_weight must share a dtype")
        weight_type = index_weight.dtype
    table, rows, rot = check_table(cos_sin, min(dim, index_dim) if index_k is not None else dim, device)
    if not (isinstance(eps, (int, float)) and math.isfinite(eps) and eps >= 0):
        raise ValueError("eps must be nonnegative and finite")
    pages, cu, num_seqs, context, page_map = check_pages(page_table, cu_seqlens, context_lens, total, page, k_cache, device)
    if dim % 16 or dim > 256 or index_dim % 16 or index_dim > 256:
        raise NotImplementedError("m3_cache_append takes head and index dims that are multiples of 16, up to 256")
    _lib.require_gpu(k, "m3_cache_append")
    if not total:
        return
    k, of_new_k = unit_rows(k)
    v, of_new_v = unit_rows(v)
    written = [k_cache, v_cache]
    at_ik = at_ic = at_ks = at_vs = at_wk = at_wi = at_table = None
    of_new_index = 0
    if index_k is not None:
        ik, (of_new_index, _, _) = unit_rows(index_k)
        at_ik, at_ic = ik.data_ptr(), index_cache.data_ptr()
        written.append(index_cache)
    if fp8:
        at_ks, at_vs = k_scale.data_ptr(), v_scale.data_ptr()
        written += (k_scale, v_scale)
    if k_weight is not None:
        wk = k_weight.contiguous()
        at_wk = wk.data_ptr()
    if index_weight is not None:
        wi = index_weight.contiguous()
        at_wi = wi.data_ptr()
    if table is not None:
        at_table = table.data_ptr()
    strides = _pack_strides(of_new_k[0], of_new_k[1], of_new_v[0], of_new_v[1], of_new_index, *of_kv, of_index[0],
                            of_index[2])
    codes = _lib.DTYPE_CODE
    with _lib.on_device(device):
        status = _lib.lib().msa_cache_append(
            k.data_ptr(), v.data_ptr(), at_ik, codes[dtype], heads, dim, index_dim, at_wk, at_wi, codes[weight_type],
            at_table, rows, rot, eps, k_cache.data_ptr(), v_cache.data_ptr(), at_ic, fp8, at_ks, at_vs, strides, *page_map,
            cu.data_ptr(), num_seqs, context.data_ptr(), total, _lib.stream_of(device))
    _lib.check(status, "msa_cache_append")
    # (a backward pass that saved a cache before this write has to notice it, as after torch's own in-place operators)
    _increment_version(written)
