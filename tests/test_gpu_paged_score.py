"""m3_index_score_topk_paged against the float64 oracle of the packed operators: scores and selections are
equal, bit for bit, over page sizes, ragged lengths, several new tokens, near ties, exact ties and odd values."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import msa_triton_amd as msa
from oracle import msa_oracle as O
from tests.helpers import cu_list, cu_tensor
from tests.paged_helpers import page_table, sequence_rows


def _setup(lengths, context, groups, dim, page, dtype, device, seed=7, keys=None):
    gen = torch.Generator().manual_seed(seed)
    totals = [n + c if c >= 0 else 0 for n, c in zip(lengths, context)]
    table, count = page_table(totals, page, gen)
    iq = (torch.randn(sum(lengths), groups, dim, generator=gen) * 2).to(dtype)
    cache = torch.randn(count, 1, page, dim, generator=gen) if keys is None else keys(count, page, dim, gen)
    cache = cache.to(dtype)
    # what is behind a sequence's tokens, and in pages of nobody, is never used
    used = torch.zeros(count, page, dtype=torch.bool)
    for s, n in enumerate(totals):
        for m in range(-(-n // page)):
            used[int(table[s, m]), :min(page, n - m * page)] = True
    cache[~used[:, None]] = float("nan")
    return (iq.to(device), cache.to(device), table, cu_tensor(lengths, device),
            torch.tensor(context, dtype=torch.int32, device=device), totals)


def _oracle(iq, cache, table, lengths, context, blocks, block, topk, local, scale):
    groups = iq.shape[1]
    scores = np.full((sum(lengths), groups, blocks), -np.inf, dtype=np.float32)
    ids = np.full((sum(lengths), groups, topk), -1, dtype=np.int32)
    q = iq.double().cpu().numpy()
    sign = np.sign(scale)
    for s, (a, n) in enumerate(zip(cu_list(lengths), lengths)):
        if context[s] < 0 or not n:
            continue
        rows = sequence_rows(cache, None, table, s, context[s] + n)[0]
        for i in range(n):
            pos = context[s] + i
            # one at a time, each row on its own: no library sum orders
            with np.errstate(invalid="ignore"):
                dots = sign * (rows[None, :pos + 1] * q[a + i][:, None]).sum(-1)
            for b in range(min(blocks, pos // block + 1)):
                part = dots[:, b * block:(b + 1) * block]
                part = np.where(np.isnan(part), -np.inf, part)
                scores[a + i, :, b] = O.public_score(part.max(1), scale)
            ids[a + i] = O.topk_rows(scores[a + i][None], [pos], block_size=block, topk_blocks=topk,
                                     local_blocks=local)[0]
    return scores, ids


def _check(x, lengths, context, block, topk, local, scale=1.0, max_seqlen=None):
    iq, cache, table, cu, ctx, totals = x
    most = max_seqlen or max(1, *totals)
    got_s, got_i = msa.m3_index_score_topk_paged(iq, cache, table.to(iq.device), cu, ctx, most, block_size=block,
                                                 scale=scale, topk_blocks=topk, local_blocks=local)
    want_s, want_i = _oracle(iq, cache, table, lengths, context, -(-most // block), block, topk, local, scale)
    assert np.array_equal(got_s.cpu().numpy(), want_s)
    assert np.array_equal(got_i.cpu().numpy(), want_i)


CASES = [  # lengths, context, groups, Di, page, block, topk, local, dtype, scale
    ([1], [0], 1, 64, 16, 16, 4, 1, torch.bfloat16, 1.0),
    ([1, 1, 1], [700, 31, 2000], 4, 128, 64, 128, 8, 1, torch.bfloat16, 1.0),
    ([5, 0, 1, 3], [126, 9, 0, 640], 4, 128, 16, 128, 4, 2, torch.float16, 1.0),
    ([40, 2], [100, 257], 3, 96, 128, 64, 3, 1, torch.bfloat16, -1.0),
    ([1, 7, 1], [-1, 300, -3], 8, 64, 32, 32, 16, 1, torch.float16, 0.125),
    ([9], [500], 2, 256, 256, 192, 5, 0, torch.bfloat16, 0.3),   # blocks of more than 128 keys, across pages
    ([3], [1000], 40, 8, 64, 1024, 2, 1, torch.bfloat16, 1.0),   # more groups than a tile has rows
    ([2, 2], [90, 900], 2, 136, 16, 48, 70, 3, torch.float16, 1.0),  # more slots than blocks
    ([33], [0], 1, 128, 64, 16, 2, 1, torch.bfloat16, 0.0),
    ([1], [20000], 4, 64, 256, 16, 16, 1, torch.bfloat16, 1.0),  # 1251 blocks
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_scores_and_selection(case, device):
    lengths, context, groups, dim, page, block, topk, local, dtype, scale = case
    _check(_setup(lengths, context, groups, dim, page, dtype, device), lengths, context, block, topk, local, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_near_ties_equal_keys_and_small_values(dtype, device):
    """Keys that differ in their last bits, repeated keys, subnormal ones, and columns that cancel."""

    def keys(count, page, dim, gen):
        base = torch.randn(1, 1, 1, dim, generator=gen)
        k = base + 2 ** -8 * torch.randn(count, 1, page, dim, generator=gen)
        k[:, :, ::3] = base
        k[:, :, 1::3, dim // 2:] = -k[:, :, 1::3, :dim // 2]  # cancels against equal halves of the query
        k[:, :, 5] *= 2 ** -14 if dtype == torch.float16 else 2 ** -130
        return k

    lengths, context = [2, 1, 4], [300, 77, 129]
    x = _setup(lengths, context, 4, 128, 16, dtype, device, keys=keys)
    x[0][:, 1, 64:] = x[0][:, 1, :64]
    x[0][1, 2] = 0
    x[0][2, 3] *= 2 ** -12 if dtype == torch.float16 else 2 ** -128
    _check(x, lengths, context, 64, 4, 1)
    if dtype == torch.bfloat16:  # large values: fp32 overflows, float64 does not
        x[0][0, 0] = 1e30
        x[1][int(x[2][0, 0]), 0, 3] = 1e30
        _check(x, lengths, context, 64, 4, 1)
    x[1][:, :, :, :] = torch.where(torch.isnan(x[1]), x[1], torch.zeros_like(x[1]))  # all equal
    _check(x, lengths, context, 64, 4, 1)


@pytest.mark.gpu
def test_missing_pages_and_short_tables(device):
    lengths, context = [2, 3], [250, 130]
    x = _setup(lengths, context, 4, 64, 32, torch.bfloat16, device)
    x[2][0, 3], x[2][0, 4], x[2][1, 0] = -1, 1000, 2 ** 31 - 1
    table = x[2][:, :6].clone()  # the first sequence goes on behind the table
    _check((x[0], x[1], table, *x[3:]), lengths, context, 64, 4, 1)
    _check((x[0], x[1], table[:, :0], *x[3:]), lengths, context, 64, 4, 1)
    _check(x, lengths, context, 64, 8, 2, max_seqlen=192)    # scores fewer blocks than there are
    _check(x, lengths, context, 64, 8, 2, max_seqlen=1000)   # and more


@pytest.mark.gpu
def test_block_sizes_and_lengths_past_the_table(device):
    """One block that holds every key, and a length that no table holds: what exists is scored, the own block selected."""
    lengths, context = [2], [250]
    x = _setup(lengths, context, 4, 64, 32, torch.bfloat16, device)
    _check(x, lengths, context, 2 ** 31 - 16, 2, 1)
    iq, cache, table, cu, _, _ = x
    table = table[:, :6].to(device)  # 192 positions
    far = torch.tensor([2 ** 31 - 40], dtype=torch.int32, device=device)
    want, _ = msa.m3_index_score_topk_paged(iq[:1], cache, table, cu_tensor([1], device),
                                            torch.tensor([191], dtype=torch.int32, device=device), 192, block_size=64)
    got, ids = msa.m3_index_score_topk_paged(iq, cache, table, cu, far, 256, block_size=64, topk_blocks=5)
    assert torch.equal(got[:1, :, :3], want) and torch.isinf(got[:, :, 3]).all()
    assert (ids.sort(dim=2).values[..., 2:] == torch.tensor([0, 1, 2], device=device)).all()
    got, _ = msa.m3_index_score_topk_paged(iq, cache, table, cu, far, 2 ** 31 - 1, block_size=2 ** 30, topk_blocks=1)
    assert torch.equal(got[0, :, 0], want[0].amax(1)) and torch.isinf(got[:, :, 1]).all()


@pytest.mark.gpu
def test_more_sequences_than_lanes(device):
    """65 and 600 sequences: the lookups that go through LDS and through several steps."""
    for n in (65, 600):
        lengths = [(i * 7) % 3 for i in range(n)]
        context = [(i * 37) % 150 - 5 for i in range(n)]
        _check(_setup(lengths, context, 2, 64, 16, torch.bfloat16, device), lengths, context, 32, 3, 1)


@pytest.mark.gpu
def test_equal_to_the_packed_operator(device):
    """A packed prompt scored whole, and its tail scored against a cache of it."""
    lengths, tails, block = [700, 333, 64], [3, 1, 64], 64
    gen = torch.Generator().manual_seed(2)
    iq, ik = torch.randn(sum(lengths), 4, 128, generator=gen).bfloat16(), torch.randn(sum(lengths), 1, 128, generator=gen).bfloat16()
    iq, ik = iq.to(device), ik.to(device)
    want_s, want_i = msa.m3_index_score_topk(iq, ik, cu_tensor(lengths, device), max(lengths), block_size=block,
                                             topk_blocks=5)
    table, count = page_table(lengths, 16, gen)
    table = table.to(device)
    cache = torch.zeros(count, 1, 16, 128, dtype=torch.bfloat16, device=device)
    zero = torch.zeros(3, dtype=torch.int32, device=device)
    kv = torch.zeros(count, 1, 16, 16, dtype=torch.bfloat16, device=device)
    msa.m3_cache_append(ik[:, :, :16], ik[:, :, :16], kv, kv.clone(), table, cu_tensor(lengths, device), zero,
                        index_k=ik, index_cache=cache)
    starts = cu_list(lengths)
    rows = torch.cat([torch.arange(b - n, b) for b, n in zip(starts[1:], tails)]).to(device)
    ctx = torch.tensor([n - t for n, t in zip(lengths, tails)], dtype=torch.int32, device=device)
    got_s, got_i = msa.m3_index_score_topk_paged(iq[rows], cache, table, msa.prepare_sequences(cu_tensor(tails, device)),
                                                 ctx, max(lengths), block_size=block, topk_blocks=5)
    assert torch.equal(got_s, want_s[rows]) and torch.equal(got_i, want_i[rows])


@pytest.mark.gpu
def test_strided_cache_and_empty_calls(device):
    x = _setup([3], [100], 2, 64, 16, torch.bfloat16, device)
    iq, cache, table, cu, ctx, totals = x
    table = table.to(device)
    want = msa.m3_index_score_topk_paged(iq, cache, table, cu, ctx, 103, block_size=16)
    wide = torch.zeros(cache.shape[0], 2, 16, 128, dtype=cache.dtype, device=device)
    wide[:, 1:, :, 64:] = cache
    off = torch.empty(iq.numel() + 1, dtype=iq.dtype, device=device)[1:].view(iq.shape).copy_(iq)
    got = msa.m3_index_score_topk_paged(off, wide[:, 1:, :, 64:], table.t().contiguous().t(), cu, ctx, 103, block_size=16)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    s, i = msa.m3_index_score_topk_paged(iq, cache, table, cu, ctx, 103, block_size=16, topk_blocks=0, local_blocks=0)
    assert torch.equal(s, want[0]) and i.shape == (3, 2, 0)
    s, i = msa.m3_index_score_topk_paged(iq, cache[:0], table, cu, ctx, 103, block_size=16, topk_blocks=2)
    assert torch.isinf(s).all() and (i[..., 0] == torch.tensor([[6], [6], [6]], device=device)).all()
    s, i = msa.m3_index_score_topk_paged(iq[:0], cache, table, torch.zeros(2, dtype=torch.int32, device=device), ctx, 103)
    assert s.shape == (0, 2, 1) and i.shape == (0, 2, 16)


def test_refusals():
    q = torch.ones(3, 2, 32, dtype=torch.bfloat16)
    cache = torch.zeros(5, 1, 16, 32, dtype=torch.bfloat16)
    cu, ctx = torch.tensor([0, 3], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    table = torch.zeros(1, 2, dtype=torch.int32)
    call = msa.m3_index_score_topk_paged
    with pytest.raises(ValueError, match="expected index_q"):
        call(q[0], cache, table, cu, ctx, 8)
    with pytest.raises(NotImplementedError, match="BF16 or FP16"):
        call(q.float(), cache.float(), table, cu, ctx, 8)
    with pytest.raises(ValueError, match="index_cache must be"):
        call(q, cache.expand(5, 2, 16, 32), table, cu, ctx, 8)
    with pytest.raises(TypeError, match="index_cache"):
        call(q, cache.half(), table, cu, ctx, 8)
    with pytest.raises(ValueError, match="block_size"):
        call(q, cache, table, cu, ctx, 8, block_size=0)
    with pytest.raises(ValueError, match="max_seqlen"):
        call(q, cache, table, cu, ctx, 0)
    with pytest.raises(ValueError, match="local_blocks"):
        call(q, cache, table, cu, ctx, 8, topk_blocks=1, local_blocks=2)
    with pytest.raises(ValueError, match="scale"):
        call(q, cache, table, cu, ctx, 8, scale=float("inf"))
    with pytest.raises(TypeError, match="context_lens"):
        call(q, cache, table, cu, ctx.long(), 8)
    with pytest.raises(ValueError, match="page_table"):
        call(q, cache, table.repeat(2, 1), cu, ctx, 8)
    with pytest.raises(ValueError, match="nondecreasing|end at total_tokens"):
        call(q, cache, table, torch.tensor([0, 4], dtype=torch.int32), ctx, 8)
    with pytest.raises(NotImplementedError, match="multiple of 16"):
        call(q, cache, table, cu, ctx, 8, block_size=24)
    with pytest.raises(RuntimeError, match="ROCm device"):
        call(q, cache, table, cu, ctx, 8)
