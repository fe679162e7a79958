"""Paged caches for the tests: tables of shuffled pages, a float64 rounding to e4m3, and where tokens lie."""

from __future__ import annotations

import numpy as np
import torch

from msa_triton_amd.paged import FP8

# every nonnegative finite e4m3 value, by code
E4M3 = np.arange(127, dtype=np.uint8)
E4M3 = torch.from_numpy(E4M3).view(FP8).double().numpy()


def round_e4m3(x):
    """The nearest e4m3 value of float64 `x` with |x| <= 448, ties to the even code; NaN for what is not finite."""
    x = np.asarray(x, dtype=np.float64)
    m = np.where(np.isfinite(x), np.abs(x), 0.0)
    hi = np.clip(np.searchsorted(E4M3, m), 1, 126)
    lo = hi - 1
    down, up = m - E4M3[lo], E4M3[hi] - m
    take = (up < down) | ((up == down) & (hi % 2 == 0))
    return np.where(np.isfinite(x), np.copysign(np.where(take, E4M3[hi], E4M3[lo]), x), np.nan)


def scale_for(amax):
    """The smallest power of two s >= 2^-100 with 448 s >= amax; 0 for 0."""
    if amax == 0:
        return 0.0
    k = -100
    while 448.0 * 2.0 ** k < amax:
        k += 1
    return 2.0 ** k


def page_table(totals, page, gen, spare=3, width=None):
    """(table [N, M] on the CPU, pages in all): shuffled pages, -1 behind each sequence."""
    need = [-(-max(n, 0) // page) for n in totals]
    count = sum(need) + spare
    order = torch.randperm(count, generator=gen, dtype=torch.int32)
    table = torch.full((len(totals), width or max(1, *need)), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, count


def place(table, page, s, pos, num_pages):
    """(page, slot) of position `pos` of sequence `s`, or None."""
    if pos < 0 or pos // page >= table.shape[1]:
        return None
    p = int(table[s][pos // page])
    return (p, pos % page) if 0 <= p < num_pages else None


def sequence_rows(cache, scale, table, s, length):
    """The cached rows [H, length, D] of a sequence in float64 (scales applied); missing pages are NaN."""
    pages, heads, page, dim = cache.shape
    out = np.full((heads, length, dim), np.nan)
    held = cache.double().cpu().numpy() if cache.dtype != FP8 else cache.cpu().float().double().numpy()
    for m in range(-(-length // page)):
        p = int(table[s][m]) if m < table.shape[1] else -1
        if not 0 <= p < pages:
            continue
        n = min(page, length - m * page)
        rows = held[p, :, :n]
        if scale is not None:
            rows = rows * scale[p].double().cpu().numpy()[:, None, None]
        out[:, m * page:m * page + n] = rows
    return out
