"""The paged operators over 5000 sequences in one call, against calls of at most 50 of them: the lookups of a
token's sequence take three steps of 64 entries there, one here.

Appended bytes and scales, scores and selections do not depend on the batch: equal bits. The attention splits rows by
the number of them; each result is within (2 d + 2^-16) max |v| and half a step of the exact one, d = 2^-23 D scale
sum |q||k| the error of a logit (D terms), so the two are within twice that of each other.
"""

from __future__ import annotations

import pytest
import torch

import msa_triton_amd as msa
from msa_triton_amd.paged import FP8
from tests.helpers import cu_list, cu_tensor

N, PAGE, DIM, BLOCK = 5000, 16, 32, 16


def _batch(device):
    gen = torch.Generator().manual_seed(5)
    lengths = [(i * 7) % 3 for i in range(N)]
    context = [(i * 37) % 40 - 3 for i in range(N)]
    total = sum(lengths)
    table = torch.randperm(N * 3, generator=gen).reshape(N, 3).to(torch.int32)
    new = {n: torch.randn(total, h, DIM, generator=gen).bfloat16().to(device)
           for n, h in (("q", 2), ("k", 1), ("v", 1), ("iq", 1), ("ik", 1))}
    return lengths, context, new, table.to(device), torch.tensor(context, dtype=torch.int32, device=device)


def _caches(device):
    gen = torch.Generator().manual_seed(6)
    x = {n: torch.randn(N * 3, 1, PAGE, DIM, generator=gen).to(device) for n in ("k", "v", "i")}
    return (x["k"].to(FP8), x["v"].to(FP8), x["i"].bfloat16(), torch.full((N * 3, 1), 2.0 ** -8, device=device),
            torch.full((N * 3, 1), 2.0 ** -8, device=device))


def _step(new, table, context, lengths, caches, device):
    kc, vc, ic, ks, vs = caches
    cu = cu_tensor(lengths, device)
    rope = msa.rope_table(64, 16, device=device)
    msa.m3_cache_append(new["k"], new["v"], kc, vc, table, cu, context, index_k=new["ik"], index_cache=ic, k_scale=ks,
                        v_scale=vs, cos_sin=rope)
    scores, ids = msa.m3_index_score_topk_paged(new["iq"], ic, table, cu, context, 48, block_size=BLOCK, topk_blocks=2)
    out, lse = msa.m3_sparse_attention_paged(new["q"], kc, vc, ids, table, cu, context, block_size=BLOCK, k_scale=ks,
                                             v_scale=vs, return_lse=True)
    return scores, ids, out, lse


@pytest.mark.gpu
def test_one_call_of_5000_sequences(device):
    lengths, context, new, table, context_lens = _batch(device)
    whole, parts = _caches(device), _caches(device)
    scores, ids, out, lse = _step(new, table, context_lens, lengths, whole, device)
    cu = cu_list(lengths)
    for a in range(0, N, 50):
        rows = slice(cu[a], cu[a + 50])
        part = {n: x[rows] for n, x in new.items()}
        s, i, o, e = _step(part, table[a:a + 50], context_lens[a:a + 50], lengths[a:a + 50], parts, device)
        assert torch.equal(s, scores[rows]) and torch.equal(i, ids[rows])
        seen = torch.isfinite(e)
        assert torch.equal(seen, torch.isfinite(lse[rows]))
        scale = DIM ** -0.5
        most_k = float((parts[0].float().abs() * parts[3][:, :, None, None])[table[a:a + 50].long().flatten()].max())
        most_v = float((parts[1].float().abs() * parts[4][:, :, None, None])[table[a:a + 50].long().flatten()].max())
        d = 2.0 ** -23 * DIM * scale * float(part["q"].float().abs().sum(-1).max()) * most_k + 2.0 ** -20
        bound = 2 * ((2 * d + 2.0 ** -16) * most_v + 2.0 ** -8 * o.float().abs() * (1 + 2.0 ** -7))
        assert ((o.float() - out[rows].float()).abs() <= bound).all()
        assert ((e - lse[rows])[seen].abs() <= 2 * (d + 2.0 ** -20 * e[seen].abs().clamp(min=1))).all()
    for x, y in zip(whole, parts):
        assert torch.equal(x.view(torch.uint8) if x.dtype == FP8 else x, y.view(torch.uint8) if y.dtype == FP8 else y)
