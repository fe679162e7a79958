"""Which views the packed window operators read in place: what the Python side keeps, the C entry points take."""

from __future__ import annotations

import itertools
import struct

import pytest
import torch

from msa_triton_amd import _lib
from msa_triton_amd.window_attention import aligned_rows

DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _status(strides, dtype, hq, g, d=64, backward=False):
    """Of a call of no tokens: arguments are checked, nothing is launched and no address is read."""
    p, code = 4096, _lib.DTYPE_CODE[dtype]
    if backward:
        return _lib.lib().msa_window_attn_bwd(p, p, p, code, struct.pack("8q", *strides), p, 1, 0, 0, hq, g, d, 0, 0, 1.0, p, None, p, p, p, p,
                                              p, p, 0, None)
    return _lib.lib().msa_window_attn_fwd(p, p, p, code, struct.pack("6q", *strides[:6]), p, 1, 0, hq, g, d, 0, 0, 1.0, p, None, None, None)


def _view(tokens, heads, d, of_token, of_head, dtype):
    """(without memory: only its address and strides are looked at)"""
    return torch.empty_strided((tokens, heads, d), (of_token, of_head, 1), dtype=dtype, device="meta")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,g", [(1, 1), (8, 8), (8, 2), (64, 8), (64, 4), (60, 4), (64, 1), (128, 1)])
def test_views_that_are_kept_are_taken(hq, g, dtype):
    d = 64
    tokens = [0, d, 512, hq * d, (1 << 24) + 8, 32537624, 32537632, (1 << 25) - 8, 1 << 25]
    heads = [0, d, 1 << 20, 1 << 24, (1 << 24) + 8, 1 << 26, (1 << 27) - 8, 1 << 28, (1 << 30) - 8, 1 << 30]
    for of_token, of_head in itertools.product(tokens, heads):
        for n in (1, 40):
            q, *of_q = aligned_rows(_view(n, hq, d, of_token, of_head, dtype), hq // g)
            k, *of_k = aligned_rows(_view(n, g, d, of_token, of_head, dtype))
            assert q.shape == (n, hq, d) and k.shape == (n, g, d)
            strides = (*of_q, *of_k, *of_k, *of_q)
            assert _status(strides, dtype, hq, g) == 0, strides
            assert _status(strides, dtype, hq, g, backward=True) == 0, strides


def test_heads_in_front_are_read_in_place():
    """[heads, tokens, dim], of more query heads a key head than there are key heads."""
    for tokens, dim in ((262144, 256), (1 << 22, 128)):
        k = torch.empty(4, tokens, dim, dtype=torch.bfloat16, device="meta").transpose(0, 1)
        kept, *strides = aligned_rows(k)
        assert kept is k and strides == [dim, tokens * dim]
        q = torch.empty(64, 65536, 256, dtype=torch.bfloat16, device="meta").transpose(0, 1)
        kept, *of_q = aligned_rows(q, 16)
        assert kept is q
        assert _status((*of_q, *strides, *strides, *of_q), k.dtype, 64, 4, 256) == 0
        assert _status((*of_q, *strides, *strides, *of_q), k.dtype, 64, 4, 256, backward=True) == 0


@pytest.mark.parametrize("which", range(8))
def test_strides_past_the_limits_are_refused(which):
    near = [64, 64] * 4
    limits = {0: (1 << 25, 32537632), 1: (1 << 30, 1 << 26)} if which in (0, 1, 6, 7) else {0: (1 << 25, 32537632), 1: (1 << 30, )}
    for far in (*limits[which % 2], -8, 4):
        strides = list(near)
        strides[which] = far
        assert _status(strides, torch.bfloat16, 64, 4, backward=True) == 1
        if which < 6:
            assert _status(strides, torch.bfloat16, 64, 4) == 1
    if which in (3, 5):
        near[which] = (1 << 30) - 8
        assert _status(near, torch.bfloat16, 64, 4, backward=True) == 0
