"""What the paged operators share: the checks of a cache and of its page table.

A cache is ``[P, H, page, D]`` (pages, heads, slots of a page, dims); ``page_table`` int32
``[N, M]`` says where each sequence's tokens are: position ``j`` of sequence ``s`` is slot
``j % page`` of page ``page_table[s, j // page]``. Entries outside ``[0, P)`` are pages that do not exist.
New tokens come packed by ``cu_seqlens`` (as everywhere); ``context_lens`` int32 ``[N]`` holds the number of
tokens that the cache has in front of them, so the new token at offset ``i`` of its sequence has
position ``context_lens[s] + i``. A negative length marks a sequence that is not there, as in a batch padded to
a fixed size. ``page_table`` and ``context_lens`` are read on the device only: a step captured in a
graph replays with whatever they hold then.
"""

from __future__ import annotations

import torch

from .layout import context_of, packed_tokens

CACHE_TYPES = (torch.bfloat16, torch.float16)
FP8 = torch.float8_e4m3fn


def check_cache(cache, name, dtypes, heads, dim, device):
    """Shape, type, device and row alignment of a cache; returns its page size and its (page, head, slot) strides."""
    shape = cache.shape
    if len(shape) != 4 or shape[1] != heads or shape[3] != dim:
        raise ValueError(f"{name} must be [pages, {heads}, page size, {dim}]")
    if cache.dtype not in dtypes:
        raise TypeError(f"{name} must have dtype {' or '.join(str(d) for d in dtypes)}")
    if cache.device != device:
        raise ValueError(f"{name} must be on the input device")
    page = shape[2]
    if page < 16 or page > 256 or page & (page - 1):
        raise ValueError("the page size must be a power of two from 16 to 256")
    of_page, of_head, of_slot, of_dim = cache.stride()
    if of_dim != 1 or (cache.data_ptr() | (of_page | of_head | of_slot) * cache.element_size()) & 15:
        raise ValueError(f"{name} rows must be contiguous and 16-byte aligned")
    return page, (of_page, of_head, of_slot)


def check_scale(scale, name, fp8, shape, device):
    """The scales [P, H] that go with an 8-bit cache (and only with one)."""
    if not fp8:
        if scale is not None:
            raise ValueError(f"{name} goes with an 8-bit cache")
        return
    if scale is None or scale.dtype != torch.float32 or scale.shape != shape or not scale.is_contiguous():
        raise ValueError(f"{name} must be contiguous fp32 [pages, heads]")
    if scale.device != device:
        raise ValueError(f"{name} must be on the cache's device")


def check_kv_caches(k_cache, v_cache, k_scale, v_scale, heads, dim, dtype, device):
    """The key and value caches of one layer: of the input type, or both in 8 bits. Returns the page size, the
    strides of both and whether they hold 8 bits."""
    page, of_k = check_cache(k_cache, "k_cache", (dtype, FP8), heads, dim, device)
    held = k_cache.dtype
    _, of_v = check_cache(v_cache, "v_cache", (held,), heads, dim, device)
    shape = k_cache.shape
    if shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must have one shape")
    fp8 = held == FP8
    check_scale(k_scale, "k_scale", fp8, shape[:2], device)
    check_scale(v_scale, "v_scale", fp8, shape[:2], device)
    return page, of_k + of_v, fp8


def check_pages(page_table, cu_seqlens, context_lens, total, page, cache, device):
    """The sequences of a paged call: the page table, cu_seqlens, the sequences, the context lengths (on the device), and
    the page map's arguments of a C call."""
    cu, num_seqs = packed_tokens(cu_seqlens, total, device)
    if context_lens is None:
        raise TypeError("context_lens must be int32")
    context = context_of(context_lens, num_seqs, device)
    if not isinstance(page_table, torch.Tensor) or page_table.dtype != torch.int32:
        raise TypeError("page_table must be int32")
    shape = page_table.shape
    if len(shape) != 2 or shape[0] != num_seqs:
        raise ValueError("page_table must be [sequences, pages]")
    if page_table.device != device:
        raise ValueError("page_table must be on the input device")
    if shape[1] * page > 2147483647:
        raise ValueError("positions must fit int32 metadata")
    of_seq, of_page = page_table.stride()
    if of_page != 1:
        page_table = page_table.contiguous()
        of_seq = page_table.stride(0)
    return page_table, cu, num_seqs, context, (page_table.data_ptr(), of_seq, shape[1], cache.shape[0], page)


def sixteen_bit(x, what):
    if x.dtype == torch.float32:
        raise NotImplementedError(f"{what} takes BF16 or FP16 inputs")
    if x.dtype not in CACHE_TYPES:
        raise TypeError(f"{what} takes BF16 or FP16 inputs")


def unit_rows(x):
    """A rank-3 tensor with unit stride along its rows, and its strides."""
    strides = x.stride()
    if strides[2] == 1:
        return x, strides
    x = x.contiguous()
    return x, x.stride()
