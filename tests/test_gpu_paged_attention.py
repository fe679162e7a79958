"""m3_sparse_attention_paged against float64, in both cache widths, and a decoding run of the paged operators
together against the packed ones.

Tolerance: logits are fp32 products of exact terms: a dot of D terms is off by D 2^-23 sum |q||k| at most (the
matrix unit may truncate), times scale; a weight by that error d of its logit (e^d - 1) twice (its own and the
maximum's), its exponential's 2^-22 and the 2^-17 that the second term of its split leaves out; the second
product and its sums add 2^-16. So |out - exact| <= (2 d + 2^-16) max |v| + half a step of the output type.
The lse is off by d and 2^-20 of its size.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import msa_triton_amd as msa
from msa_triton_amd.paged import FP8
from tests.helpers import cu_list, cu_tensor
from tests.paged_helpers import page_table, sequence_rows


def _setup(lengths, context, groups, ratio, dim, page, slots, block, dtype, fp8, device, seed=17):
    gen = torch.Generator().manual_seed(seed)
    totals = [n + c if c >= 0 else 0 for n, c in zip(lengths, context)]
    table, count = page_table(totals, page, gen)
    total = sum(lengths)
    x = dict(q=(torch.randn(total, groups * ratio, dim, generator=gen) * 1.5).to(dtype), ks=None, vs=None)
    used = torch.zeros(count, page, dtype=torch.bool)
    for s, n in enumerate(totals):
        for m in range(-(-n // page)):
            used[int(table[s, m]), :min(page, n - m * page)] = True
    for name in ("k", "v"):
        c = torch.randn(count, groups, page, dim, generator=gen)
        if fp8:
            x[name + "s"] = torch.exp2(torch.randint(-7, -3, (count, groups), generator=gen).float()) * (
                0.7 if name == "k" else 1.3)  # any scale is taken, not powers of two alone
            c = (c / x[name + "s"][:, :, None, None]).clamp(-448, 448).to(FP8)
            c.view(torch.uint8)[~used[:, None].expand(-1, groups, -1)] = 0x7F  # NaN
            x[name + "s"][~used.any(1)] = float("nan")
        else:
            c = c.to(dtype)
            c[~used[:, None].expand(-1, groups, -1)] = float("nan")
        x[name + "c"] = c
    ids = torch.full((total, groups, slots), -1, dtype=torch.int32)
    for s, (a, n) in enumerate(zip(cu_list(lengths), lengths)):
        for i in range(n):
            own = max(0, context[s] + i) // block
            for g in range(groups):
                pick = torch.randperm(own + 1, generator=gen)[:slots]
                if g % 2 == 0 and own not in pick.tolist() and len(pick):
                    pick[0] = own
                ids[a + i, g, :len(pick)] = pick.to(torch.int32)
    x["ids"] = ids
    x = {n: None if v is None else v.to(device) for n, v in x.items()}
    x["table"], x["totals"] = table, totals
    x["cu"] = cu_tensor(lengths, device)
    x["context"] = torch.tensor(context, dtype=torch.int32, device=device)
    return x


def _oracle(x, lengths, context, block, scale):
    """(out, lse, bound on |out|'s error, on lse's) in float64."""
    q, ids = x["q"].double().cpu().numpy(), x["ids"].cpu().numpy()
    total, heads, dim = q.shape
    groups = ids.shape[1]
    ratio = heads // groups
    out, lse = np.zeros((total, heads, dim)), np.full((total, heads), -np.inf)
    tol, lse_tol = np.zeros((total, heads, 1)), np.zeros((total, heads))
    for s, (a, n) in enumerate(zip(cu_list(lengths), lengths)):
        if context[s] < 0 or not n:
            continue
        k = sequence_rows(x["kc"], x["ks"], x["table"], s, context[s] + n)
        v = sequence_rows(x["vc"], x["vs"], x["table"], s, context[s] + n)
        page = x["kc"].shape[2]
        have = np.array([j // page < x["table"].shape[1] and 0 <= int(x["table"][s, j // page]) < x["kc"].shape[0]
                         for j in range(context[s] + n)])
        for i in range(n):
            pos = context[s] + i
            for g in range(groups):
                blocks = sorted({int(b) for b in ids[a + i, g] if 0 <= b <= pos // block})
                keys = np.array([j for b in blocks for j in range(b * block, min((b + 1) * block, pos + 1))
                                 if have[j]], dtype=np.int64)
                if not keys.size:
                    continue
                for h in range(g * ratio, (g + 1) * ratio):
                    logit = k[g, keys] @ q[a + i, h] * scale
                    if (logit == -np.inf).all():
                        continue
                    d = (dim * 2.0 ** -23 * (np.abs(k[g, keys]) @ np.abs(q[a + i, h])) * abs(scale)
                         + 2.0 ** -22 * np.abs(logit))
                    d = d[np.isfinite(d)].max(initial=0.0)
                    m = logit.max()
                    w = np.exp(logit - m)
                    lse[a + i, h] = m + np.log(w.sum())
                    out[a + i, h] = (w / w.sum()) @ v[g, keys]
                    top = np.abs(v[g, keys]).max()
                    tol[a + i, h] = (2 * d + 2.0 ** -16) * top
                    lse_tol[a + i, h] = d + 2.0 ** -20 * max(1.0, abs(lse[a + i, h]))
    return out, lse, tol, lse_tol


def _call(x, block, **change):
    a = dict(x, **change)
    return msa.m3_sparse_attention_paged(a["q"], a["kc"], a["vc"], a["ids"], a["table"].to(a["q"].device), a["cu"],
                                         a["context"], block_size=block, k_scale=a["ks"], v_scale=a["vs"],
                                         scale=a.get("scale"), return_lse=True)


def _check(x, lengths, context, block, scale=None, **change):
    y = dict(x, **change)
    got, lse = _call(y, block, scale=scale)
    dim = y["q"].shape[2]
    want, want_lse, tol, lse_tol = _oracle(y, lengths, context, block, dim ** -0.5 if scale is None else scale)
    step = torch.finfo(got.dtype).eps / 2
    err = np.abs(got.double().cpu().numpy() - want)
    bound = tol * (1 + step) + step * np.abs(want) + torch.finfo(got.dtype).smallest_normal * step
    assert np.isfinite(err).all() and (err <= bound).all(), float((err / np.maximum(bound, 1e-300)).max())
    lse = lse.double().cpu().numpy()
    gone = np.isinf(want_lse)
    assert np.array_equal(np.isneginf(lse), gone)
    assert (np.abs(lse[~gone] - want_lse[~gone]) <= lse_tol[~gone]).all()
    return got, lse


CASES = [  # lengths, context, groups, ratio, D, page, slots, block, dtype
    ([1], [0], 1, 1, 64, 16, 1, 16, torch.bfloat16),
    ([1, 1, 1], [1000, 130, 15], 4, 8, 128, 64, 4, 128, torch.bfloat16),
    ([3, 0, 2, 5], [126, 9, 0, 640], 2, 4, 128, 16, 3, 64, torch.float16),
    ([1, 7], [300, 77], 3, 5, 96, 32, 6, 48, torch.bfloat16),       # half steps, dims and heads that do not fill
    ([2, 1, 1], [-1, 500, -4], 2, 16, 256, 128, 2, 128, torch.bfloat16),
    ([1], [700], 1, 40, 64, 256, 3, 192, torch.float16),            # three tiles of heads
    ([4], [3000], 1, 8, 16, 16, 100, 16, torch.bfloat16),           # many short blocks
    ([70], [20], 2, 2, 48, 16, 2, 32, torch.float16),
    ([2], [9000], 1, 4, 128, 128, 5, 2048, torch.bfloat16),         # more steps than one list holds
    ([600], [0], 4, 8, 64, 64, 2, 64, torch.bfloat16),              # rows enough for one workgroup each
    ([(i * 7) % 3 for i in range(300)], [(i * 37) % 150 - 5 for i in range(300)], 1, 2, 32, 16, 2, 32,
     torch.float16),                                                # more sequences than lanes
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("fp8", [False, True])
def test_attention(case, fp8, device):
    lengths, context, *rest = case
    x = _setup(lengths, context, *rest, fp8, device)
    _check(x, lengths, context, rest[5])


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", (False, True))
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_many_small_weights_count(dtype, fp8, device):
    """64 keys of weight 1 (value 0) and thousands of weight 2^-26 (value 256): each is below half of fp16's smallest value,
    together they are the output. The logits are products of one term, so a weight is off by 2 x 18 x 2^-23 (its logit, in
    fp32) and 2^-22; its two 16-bit terms and the sums by 2^-14 together."""
    n, block, tokens = 8192, 128, 520
    x = _setup([tokens], [n - tokens], 1, 2, 16, 128, n // block, block, dtype, fp8, device)
    x["kc"].copy_(torch.zeros((), dtype=torch.float32))
    x["vc"].copy_(torch.full((), 256.0))
    if fp8:
        x["ks"].fill_(1.0)
        x["vs"].fill_(1.0)
    for page in x["table"][0, :16].tolist():  # at the head of each wave's keys, however they are shared out
        x["kc"][page, 0, ::32, 0] = 18.0
        x["vc"][page, 0, ::32] = 0.0
    x["q"].zero_()
    x["q"][..., 0] = 1.0
    x["ids"].copy_(torch.arange(n // block, dtype=torch.int32))
    got, _ = _call(x, block, scale=1.0)
    count = torch.arange(n - tokens + 1, n + 1, dtype=torch.float64) - 64
    want = 256 * count / (64 * np.exp(18.0) + count)
    bound = torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -8) + 2.0 ** -14 + 36 * 2.0 ** -23 + 2.0 ** -22
    err = (got.double().cpu() / want[:, None, None] - 1).abs()
    assert (err <= bound).all(), float(err.max())


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_selections_pages_and_scale(fp8, device):
    lengths, context = [2, 3], [250, 130]
    x = _setup(lengths, context, 2, 8, 64, 32, 4, 64, torch.bfloat16, fp8, device)
    ids = x["ids"].clone()
    ids[0, 0] = torch.tensor([3, 3, 3, 0], dtype=torch.int32)      # repeated
    ids[0, 1] = torch.tensor([-1, 99, -7, 2 ** 31 - 1], dtype=torch.int32)  # nothing
    ids[1, 0] = torch.tensor([4, 2, 3, 1], dtype=torch.int32)      # the first behind the token
    ids[2, 1] = -1
    out, lse = _check(x, lengths, context, 64, ids=ids, scale=-0.3)
    assert (out[0, 8:] == 0).all() and np.isneginf(lse[0, 8:]).all() and (out[2, 8:] == 0).all()
    _check(x, lengths, context, 64, ids=ids, scale=0.0)
    _check(x, lengths, context, 64, ids=ids[:, :, :0])
    table = x["table"].clone()
    table[0, 3], table[0, 4], table[1, 0] = -1, 1000, 2 ** 31 - 1
    _check(x, lengths, context, 64, table=table[:, :6])
    out, lse = _check(x, lengths, context, 64, table=table[:, :0])
    assert (out == 0).all()
    empty = dict(kc=x["kc"][:0], vc=x["vc"][:0])
    if fp8:
        empty.update(ks=x["ks"][:0], vs=x["vs"][:0])
    out, lse = _check(x, lengths, context, 64, **empty)
    assert (out == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_block_sizes_and_lengths_past_the_table(fp8, device):
    """A block that holds every key there is, lengths that no table holds, and more slots than LDS keeps ids of."""
    lengths, context = [1, 2], [150, 60]
    x = _setup(lengths, context, 2, 4, 32, 16, 3, 16, torch.bfloat16, fp8, device)
    ids = torch.full_like(x["ids"], -1)
    ids[..., 1] = 0
    _check(x, lengths, context, 2 ** 31 - 16, ids=ids)
    table = x["table"][:, :4].clone()  # 64 positions
    _check(x, lengths, context, 2 ** 30, ids=ids, table=table)
    want = _call(x, 2 ** 30, ids=ids, table=table)
    far = torch.tensor([2 ** 31 - 1, 2 ** 31 - 2], dtype=torch.int32, device=device)
    got = _call(x, 2 ** 30, ids=ids, table=table, context=far)
    assert torch.equal(got[0][0], want[0][0])  # (the second sequence's slots behind its tokens hold NaN)
    many = torch.randint(-3, 12, (3, 2, 1500), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    many[:, :, :1400] = torch.where(many[:, :, :1400] > 5, -1, many[:, :, :1400])
    _check(x, lengths, context, 16, ids=many.to(device))
    _check(x, lengths, context, 16, ids=many[:, :, 1350:1450].to(device))


@pytest.mark.gpu
def test_infinite_logits_and_large_values(device):
    lengths, context, block = [1, 1], [200, 40], 64
    x = _setup(lengths, context, 1, 2, 64, 16, 4, block, torch.bfloat16, False, device)
    x["q"][:] = x["q"].abs()
    page = int(x["table"][0, 1])
    x["kc"][page, 0, 3] = -float("inf")  # a visible key that no one takes
    _check(x, lengths, context, block)
    for m in range(x["table"].shape[1]):
        if int(x["table"][1, m]) >= 0:
            x["kc"][int(x["table"][1, m])] = -float("inf")  # and a row of nothing else
    out, lse = _check(x, lengths, context, block)
    assert (out[1] == 0).all() and np.isneginf(lse[1]).all()
    x = _setup(lengths, context, 1, 2, 64, 16, 4, block, torch.bfloat16, False, device)
    x["kc"] *= 300.0  # logits of some thousands: one key takes all
    _check(x, lengths, context, block)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_strided_caches_streams_and_determinism(fp8, device):
    lengths, context = [1, 2], [300, 77]
    x = _setup(lengths, context, 2, 8, 128, 16, 4, 64, torch.bfloat16, fp8, device)
    want = _call(x, 64)
    both = torch.stack([x["kc"].view(torch.uint8), x["vc"].view(torch.uint8)], 1).view(x["kc"].dtype)
    slot_first = x["vc"].view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(x["vc"].dtype)
    off = torch.empty(x["q"].numel() + 1, dtype=x["q"].dtype, device=device)[1:].view(x["q"].shape).copy_(x["q"])
    heads_first = x["q"].transpose(0, 1).contiguous().transpose(0, 1)
    for change in (dict(kc=both[:, 0], vc=both[:, 1]), dict(vc=slot_first), dict(q=off), dict(q=heads_first), {},
                   dict(cu=msa.prepare_sequences(x["cu"]))):
        got = _call(x, 64, **change)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    x["cu"] = msa.prepare_sequences(x["cu"])
    table = x["table"].to(device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _call(x, 64, table=table)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_offsets_past_32_bits(device):
    """Keys and values beyond 2^32 bytes of a cache."""
    heads, dim, page, count = 8, 256, 256, 4200  # 4.4 GB in 8 bits
    kc = torch.zeros(count, heads, page, dim, dtype=FP8, device=device)
    vc = torch.zeros(count, heads, page, dim, dtype=FP8, device=device)
    ones = torch.ones(count, heads, device=device)
    vc[-1, :, 5] = torch.arange(8, device=device)[:, None].float().to(FP8)
    kc[-1, :, 5] = 2.0
    q = torch.ones(1, 16, dim, dtype=torch.bfloat16, device=device)
    table = torch.tensor([[3, count - 1]], dtype=torch.int32, device=device)
    ids = torch.tensor([[[0, 2]]], dtype=torch.int32, device=device).expand(1, 8, 2)
    out = msa.m3_sparse_attention_paged(q, kc, vc, ids, table, cu_tensor([1], device),
                                        torch.tensor([299], dtype=torch.int32, device=device), k_scale=ones,
                                        v_scale=ones)
    # scale 1/16, logit 32 of the one key against 0 of 171 others
    weight = 1 / (1 + 171 * np.exp(-32.0))
    want = weight * np.arange(8).repeat(2)
    assert np.allclose(out[0, :, 0].double().cpu().numpy(), want, rtol=2 ** -8)


def _decode(prompt, steps, fp8, page, block, topk, device, seed=23):
    """A layer's decoding run: prompts through the packed operators and into the cache, then tokens one by one (and
    once three at a time). Returns what the packed operators give for the whole sequences and what the run gave."""
    gen = torch.Generator().manual_seed(seed)
    groups, ratio, dim, index_dim, rot = 2, 8, 128, 64, 64
    n = len(prompt)
    full = [p + steps for p in prompt]
    cu_full = cu_list(full)

    def rand(heads, d):
        return torch.randn(sum(full), heads, d, generator=gen).bfloat16().to(device)

    q, k, v = rand(groups * ratio, dim), rand(groups, dim), rand(groups, dim)
    iq, ik = rand(groups, index_dim), rand(1, index_dim)
    wq, wk = ((1 + 0.2 * torch.randn(dim, generator=gen)).bfloat16().to(device) for _ in range(2))
    wi, wj = ((1 + 0.2 * torch.randn(index_dim, generator=gen)).bfloat16().to(device) for _ in range(2))
    rope = msa.rope_table(max(full), rot, device=device)
    # the packed operators on the whole sequences
    whole = msa.prepare_sequences(cu_tensor(full, device), block_size=block)
    qn, kn = msa.m3_qk_norm_rope(q, k, wq, wk, rope, whole)
    iqn, ikn = msa.m3_qk_norm_rope(iq, ik, wi, wj, rope, whole)
    _, ids = msa.m3_index_score_topk(iqn, ikn, whole, max(full), block_size=block, topk_blocks=topk)
    want = msa.m3_sparse_attention(qn, kn, v, ids, whole, max(full), block_size=block)
    # the run
    table, count = page_table(full, page, gen)
    table = table.to(device)
    kind = FP8 if fp8 else torch.bfloat16
    kc, vc = (torch.zeros(count, groups, page, dim, dtype=kind, device=device) for _ in range(2))
    ks, vs = (torch.zeros(count, groups, device=device) if fp8 else None for _ in range(2))
    ic = torch.zeros(count, 1, page, index_dim, dtype=torch.bfloat16, device=device)
    got, got_ids = torch.zeros_like(want), torch.zeros_like(ids)
    done = [0] * n
    for size in [None, 1, 3] + [1] * (steps - 4):
        new = list(prompt) if size is None else [size] * n
        rows = torch.cat([torch.arange(c + d, c + d + m) for c, d, m in zip(cu_full, done, new)]).to(device)
        seqs = msa.prepare_sequences(cu_tensor(new, device), block_size=block)
        ctx = torch.tensor(done, dtype=torch.int32, device=device)
        msa.m3_cache_append(k[rows], v[rows], kc, vc, table, seqs, ctx, index_k=ik[rows], index_cache=ic, k_scale=ks,
                            v_scale=vs, k_weight=wk, index_weight=wj, cos_sin=rope)
        a, _ = msa.m3_qk_norm_rope(q[rows], None, wq, None, rope, seqs, context_lens=ctx)
        b, _ = msa.m3_qk_norm_rope(iq[rows], None, wi, None, rope, seqs, context_lens=ctx)
        _, sel = msa.m3_index_score_topk_paged(b, ic, table, seqs, ctx, max(full), block_size=block, topk_blocks=topk)
        got[rows] = msa.m3_sparse_attention_paged(a, kc, vc, sel, table, seqs, ctx, block_size=block, k_scale=ks,
                                                  v_scale=vs)
        got_ids[rows] = sel
        done = [d + m for d, m in zip(done, new)]
    assert done == full
    return want, ids, got, got_ids, v


@pytest.mark.gpu
@pytest.mark.parametrize("page,block", [(16, 32), (128, 64), (64, 128)])
def test_decoding_run_matches_the_packed_operators(page, block, device):
    want, ids, got, got_ids, v = _decode([333, 40, 1], 9, False, page, block, 4, device)
    assert torch.equal(ids, got_ids)
    # both round outputs of fp32 accuracy once: at most one bf16 step apart
    step = torch.maximum(want.float().abs(), torch.full_like(want.float(), 2 ** -6)) * 2 ** -7
    assert ((want.float() - got.float()).abs() <= step).all()
    assert (want == got).float().mean() > 0.98


@pytest.mark.gpu
def test_decoding_run_in_8_bits(device):
    want, ids, got, got_ids, v = _decode([333, 40, 1], 9, True, 32, 64, 4, device)
    assert torch.equal(ids, got_ids)  # the index keys are held in 16 bits
    # a key's and a value's e4m3 rounding: 2^-4 of each element, rounded again at most a few times in a page
    # (exact but below the normal range). An output is a mean of values, off by 2^-4 of max |v| from the values and by
    # at most as much again for logits of size up to 4 whose keys move by 2^-4 of each product, added in random signs
    # (sqrt(128) of 128 products): 4 x 2^-4 x 2 / sqrt(128) < 2^-4.
    assert (want.float() - got.float()).abs().max() <= 2 * 2 ** -4 * float(v.float().abs().max())
    assert (want.float() - got.float()).norm() <= 2 ** -4 * want.float().norm()


@pytest.mark.gpu
def test_captured_step_replays_at_new_lengths(device):
    """One decoding step in a graph: replayed with other lengths, rows and an absent sequence."""
    lengths, groups, ratio, dim, page, block = [1, 1, 1], 2, 4, 64, 16, 32
    totals = [120, 70, 90]
    gen = torch.Generator().manual_seed(3)
    table, count = page_table(totals, page, gen)
    table = table.to(device)
    seqs = msa.prepare_sequences(cu_tensor(lengths, device), block_size=block)
    ctx = torch.tensor([100, 30, 15], dtype=torch.int32, device=device)
    rope = msa.rope_table(128, 32, device=device)
    w = torch.ones(dim, dtype=torch.bfloat16, device=device)
    rows = torch.randn(3, groups * ratio + 4 * groups + 1, dim, generator=gen).bfloat16().to(device)
    start = [(torch.randn(count, h, page, dim, generator=gen) * 40).clamp(-400, 400).to(device) for h in (groups, groups, 1)]

    def fresh():
        return [start[0].to(FP8), start[1].to(FP8), start[2].bfloat16(), torch.full((count, groups), 2.0 ** -5, device=device),
                torch.full((count, groups), 2.0 ** -6, device=device)]

    def step(c):
        h = groups * ratio
        q, k, v, iq, ik = rows.split([h, groups, groups, 2 * groups, 1], 1)
        msa.m3_cache_append(k, v, c[0], c[1], table, seqs, ctx, index_k=ik, index_cache=c[2], k_scale=c[3], v_scale=c[4],
                            k_weight=w, index_weight=w, cos_sin=rope)
        a, b = msa.m3_qk_norm_rope(q, iq[:, :groups], w, w, rope, seqs, context_lens=ctx)
        s, sel = msa.m3_index_score_topk_paged(b, c[2], table, seqs, ctx, 128, block_size=block, topk_blocks=3)
        o, lse = msa.m3_sparse_attention_paged(a, c[0], c[1], sel, table, seqs, ctx, block_size=block, k_scale=c[3],
                                               v_scale=c[4], return_lse=True)
        return s, sel, o, lse

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fresh())
    torch.cuda.current_stream().wait_stream(side)
    held, mirror = fresh(), fresh()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(held)
    for i, lens in enumerate(([100, 30, 15], [101, 31, -1], [119, 69, 16], [0, -2, 17])):
        ctx.copy_(torch.tensor(lens, dtype=torch.int32))
        rows.copy_(torch.randn(rows.shape, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        want = step(mirror)
        assert all(torch.equal(x, y) for x, y in zip(outs, want)), i
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(held, mirror)), i


def test_refusals():
    q = torch.ones(3, 4, 32, dtype=torch.bfloat16)
    cache = torch.zeros(5, 2, 16, 32, dtype=torch.bfloat16)
    ids = torch.zeros(3, 2, 2, dtype=torch.int32)
    cu, ctx = torch.tensor([0, 3], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    table = torch.zeros(1, 2, dtype=torch.int32)
    call = msa.m3_sparse_attention_paged
    with pytest.raises(ValueError, match="expected q"):
        call(q[0], cache, cache, ids, table, cu, ctx)
    with pytest.raises(NotImplementedError, match="BF16 or FP16"):
        call(q.float(), cache.float(), cache.float(), ids, table, cu, ctx)
    with pytest.raises(ValueError, match="indices"):
        call(q, cache, cache, ids.long(), table, cu, ctx)
    with pytest.raises(ValueError, match="multiple of G"):
        call(q[:, :3], cache, cache, ids, table, cu, ctx)
    with pytest.raises(ValueError, match="k_cache must be"):
        call(q, cache, cache, ids[:, :1], table, cu, ctx)
    with pytest.raises(TypeError, match="v_cache"):
        call(q, cache.to(FP8), cache, ids, table, cu, ctx)
    with pytest.raises(ValueError, match="v_scale must be"):
        call(q, cache.to(FP8), cache.to(FP8), ids, table, cu, ctx, k_scale=torch.ones(5, 2))
    with pytest.raises(ValueError, match="8-bit cache"):
        call(q, cache, cache, ids, table, cu, ctx, v_scale=torch.ones(5, 2))
    with pytest.raises(ValueError, match="16-byte"):
        call(q, cache.transpose(2, 3).contiguous().transpose(2, 3), cache, ids, table, cu, ctx)
    with pytest.raises(ValueError, match="block_size"):
        call(q, cache, cache, ids, table, cu, ctx, block_size=-16)
    with pytest.raises(ValueError, match="scale must be finite"):
        call(q, cache, cache, ids, table, cu, ctx, scale=float("nan"))
    with pytest.raises(ValueError, match="one length per sequence"):
        call(q, cache, cache, ids, table, cu, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(TypeError, match="page_table"):
        call(q, cache, cache, ids, table.float(), cu, ctx)
    with pytest.raises(NotImplementedError, match="multiples of 16"):
        call(q, cache, cache, ids, table, cu, ctx, block_size=100)
    with pytest.raises(RuntimeError, match="ROCm device"):
        call(q, cache, cache, ids, table, cu, ctx)
