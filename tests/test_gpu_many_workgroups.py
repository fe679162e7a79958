"""Calls that need 2^24 workgroups and more (a launch holds fewer than 2^32 threads): rows at both ends and at the
launches' borders against small calls of them."""

from __future__ import annotations

import pytest
import torch

import msa_triton_amd as msa
from msa_triton_amd import _lib
from msa_triton_amd.paged import FP8
from tests.helpers import cu_tensor


def _spots(total, *borders):
    """Short token ranges at the ends and around the borders."""
    return [(max(0, b - 9), min(total, b + 9)) for b in (0, *borders, total)]


@pytest.mark.gpu
def test_norm(device):
    total, heads, dim = (1 << 21) + 5, 33, 2  # value by value: four rows a workgroup
    x = torch.randn(total, heads, dim, device=device, generator=torch.Generator(device).manual_seed(1)).bfloat16()
    w = torch.tensor([1.5, 0.5], dtype=torch.bfloat16, device=device)
    table = msa.rope_table(total, dim, device=device)
    assert total * heads / 4 > 1 << 24
    got, _ = msa.m3_qk_norm_rope(x, None, w, None, table, msa.prepare_sequences(cu_tensor([total], device)))
    for a, b in _spots(total, (1 << 25) // heads, (1 << 26) // heads):
        want, _ = msa.m3_qk_norm_rope(x[a:b], None, w, None, table, cu_tensor([b - a], device),
                                      context_lens=torch.tensor([a], dtype=torch.int32, device=device))
        assert torch.equal(got[a:b], want)


@pytest.mark.gpu
def test_append_in_8_bits(device):
    heads, dim, page, seqs = 1 << 19, 16, 16, 9
    gen = torch.Generator(device).manual_seed(1)
    k, v = (torch.randn(seqs, heads, dim, device=device, generator=gen).bfloat16() for _ in range(2))
    w = torch.linspace(0.5, 2, dim, device=device).bfloat16()
    table = torch.arange(seqs, dtype=torch.int32, device=device).flip(0)[:, None].contiguous()
    ctx, cu = torch.arange(seqs, dtype=torch.int32, device=device), msa.prepare_sequences(cu_tensor([1] * seqs, device))

    def run(k, v):
        h = k.shape[1]
        kc, vc = (torch.zeros(seqs, h, page, dim, dtype=FP8, device=device) for _ in range(2))
        ks, vs = (torch.full((seqs, h), 2.0 ** -12, device=device) for _ in range(2))
        msa.m3_cache_append(k, v, kc, vc, table, cu, ctx, k_scale=ks, v_scale=vs, k_weight=w)
        return kc.view(torch.uint8), vc.view(torch.uint8), ks, vs

    got = run(k, v)  # two pages' numbers a sequence, keys and values of each head: 2 x 9 x 2^20 workgroups
    for a, b in ((0, 9), ((1 << 18) - 9, (1 << 18) + 9), (heads - 9, heads)):
        for x, y in zip(got, run(k[:, a:b], v[:, a:b])):
            assert torch.equal(x[:, a:b], y)


@pytest.mark.gpu
def test_append_in_16_bits(device):
    total, heads, dim, page = (1 << 20) + 3, 33, 16, 256
    gen = torch.Generator(device).manual_seed(1)
    k = torch.randn(total * heads * dim + 1, device=device, generator=gen).bfloat16()[1:].view(total, heads, dim)  # 2-byte rows
    pages = -(-total // page)
    order = torch.randperm(pages, device=device, generator=gen).int()
    kc, vc = (torch.zeros(pages, heads, page, dim, dtype=torch.bfloat16, device=device) for _ in range(2))
    assert 2 * total * heads / 4 > 1 << 24
    msa.m3_cache_append(k, k, kc, vc, order[None], msa.prepare_sequences(cu_tensor([total], device)),
                        torch.zeros(1, dtype=torch.int32, device=device))
    for cache in (kc, vc):
        rows = cache[order.long()].transpose(1, 2).reshape(-1, heads, dim)[:total]
        assert torch.equal(rows, k)


@pytest.mark.gpu
def test_attention(device):
    groups, dim, page = 4, 16, 16
    total = (1 << 22) + 11
    gen = torch.Generator(device).manual_seed(1)
    q = torch.randn(total, groups, dim, device=device, generator=gen).bfloat16()
    kc, vc = (torch.randn(3, groups, page, dim, device=device, generator=gen).bfloat16() for _ in range(2))
    ids = torch.randint(-1, 3, (total, groups, 1), device=device, generator=gen).int()
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=device)
    context = torch.zeros(1, dtype=torch.int32, device=device)

    def call(a, b, context):
        return msa.m3_sparse_attention_paged(q[a:b], kc, vc, ids[a:b], table, cu_tensor([b - a], device), context,
                                             block_size=16, return_lse=True)

    out, lse = call(0, total, context)  # a workgroup for each token and group
    for a, b in _spots(total, 1 << 21):
        want, want_lse = call(a, b, context + a)
        assert torch.equal(out[a:b], want) and torch.equal(lse[a:b], want_lse)


def test_score_sizes_that_are_refused():
    """Status 2 before anything is launched (the pointers are never used)."""
    def status(tokens, groups, topk, dim=64):
        p = 4096
        return _lib.lib().msa_index_score_topk_paged(p, p, _lib.DTYPE_CODE[torch.bfloat16], 64 * dim, dim, p, 1, 1, 1, 64, p, 1,
                                                     p, tokens, groups, dim, 1, 16, 1.0, topk, 0, p, p, None)

    assert status(1 << 26, 4, 1) == 2 and status(1 << 29, 4, 0) == 2 and status(16, 1, 1, dim=264) == 2
