"""m3_sparse_attention_paged where queries, keys or values are not finite: against the formula in float64, at one
workgroup a row and at several."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import msa_triton_amd as msa
from msa_triton_amd import _lib
from msa_triton_amd.paged import FP8
from tests.helpers import cu_tensor

PAGE, BLOCK, SLOTS, GROUPS, RATIO, DIM = 32, 64, 6, 2, 3, 64
KEYS = BLOCK * SLOTS  # every key of a sequence is selected


def _inputs(tokens, dtype, fp8, device, seed=5):
    """One sequence of KEYS + tokens - 1 positions: its last `tokens` ones attend to all blocks in front."""
    gen = torch.Generator().manual_seed(seed)
    pages = -(-(KEYS + tokens) // PAGE)
    x = dict(q=torch.randn(tokens, GROUPS * RATIO, DIM, generator=gen).to(dtype).to(device))
    for name in ("k", "v"):
        c = torch.randn(pages, GROUPS, PAGE, DIM, generator=gen).to(dtype)
        x[name + "c"] = (c.float() * 16).clamp(-400, 400).to(FP8).to(device) if fp8 else c.to(device)
        x[name + "s"] = torch.full((pages, GROUPS), 2.0 ** -4, device=device) if fp8 else None
    x["table"] = torch.randperm(pages, generator=gen, dtype=torch.int32)[None].to(device)
    x["ids"] = torch.arange(SLOTS, dtype=torch.int32, device=device).expand(tokens, GROUPS, SLOTS).contiguous()
    x["cu"] = cu_tensor([tokens], device)
    x["ctx"] = torch.tensor([KEYS - 1], dtype=torch.int32, device=device)
    return x


def _at(x, j):
    """(page, slot) of position j."""
    return int(x["table"][0, j // PAGE]), j % PAGE


def _call(x):
    return msa.m3_sparse_attention_paged(x["q"], x["kc"], x["vc"], x["ids"], x["table"], x["cu"], x["ctx"], block_size=BLOCK,
                                         k_scale=x["ks"], v_scale=x["vs"], return_lse=True)


def _rows(x, name):
    """The sequence's KEYS first rows [G, KEYS, D] in float64."""
    c, s = x[name + "c"].float().double().cpu(), x[name + "s"]
    if s is not None:
        c = c * s.double().cpu()[:, :, None, None]
    return np.stack([c[_at(x, j)[0], :, _at(x, j)[1]].numpy() for j in range(KEYS)], 1)


def _formula(x):
    q = x["q"].double().cpu().numpy()
    k, v = _rows(x, "k"), _rows(x, "v")
    out, lse = np.zeros(q.shape), np.zeros(q.shape[:2])
    with np.errstate(all="ignore"):
        for t in range(q.shape[0]):
            for h in range(q.shape[1]):
                logit = k[h // RATIO] @ q[t, h] * DIM ** -0.5
                m = logit.max()  # (NaN if one is)
                w = np.exp(logit - m)
                lse[t, h] = m + np.log(w.sum())
                out[t, h] = (w[:, None] * v[h // RATIO]).sum(0) / w.sum()
    return out, lse


def _splits(tokens):
    size = _lib.lib().msa_attn_paged_workspace_bytes(tokens, GROUPS * RATIO, GROUPS, DIM, SLOTS, BLOCK)
    return "several" if size else "one"


# tokens of a call whose rows one workgroup each takes, and of one with several a row
WAYS = [(600, "one"), (2, "several")]
TYPES = [(torch.bfloat16, False), (torch.float16, False), (torch.bfloat16, True)]


def _compare(x, rows, exact=True):
    """The rows given against the formula: NaN and infinities where it has them (`exact`; otherwise not finite there), the
    rest as near as fp32 logits, two-term weights and one rounding give (2^-7 of the largest value covers all)."""
    out, lse = (y.double().cpu().numpy() for y in _call(x))
    few = dict(x, q=x["q"][rows])
    want, want_lse = _formula(few)
    out, lse = out[rows], lse[rows]
    odd = ~np.isfinite(want)
    if exact:
        wrong = np.argwhere(odd & (out != want) & ~(np.isnan(out) & np.isnan(want)))
        assert not len(wrong), wrong[:5].tolist()
    wrong = np.argwhere(~np.isfinite(out) != odd)
    assert not len(wrong), wrong[:5].tolist()
    assert np.abs(out[~odd] - want[~odd]).max(initial=0.0) <= 2 ** -7 * 6
    assert np.array_equal(np.isnan(lse), np.isnan(want_lse))
    ok = np.isfinite(want_lse)
    assert np.abs(lse[ok] - want_lse[ok]).max(initial=0.0) <= 2 ** -10


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,fp8", TYPES)
@pytest.mark.parametrize("tokens,ways", WAYS)
def test_nan_logits_give_nan(tokens, ways, dtype, fp8, device):
    """A query with a NaN, and the rows that see a key with one: NaN, whichever wave or workgroup has the key (positions 0, 40
    and 300 lie with different ones)."""
    assert _splits(tokens) == ways
    x = _inputs(tokens, dtype, fp8, device)
    x["q"][1, 2, 7] = float("nan")
    _compare(x, [0, 1])
    for j in (0, 40, 300):
        x = _inputs(tokens, dtype, fp8, device)
        page, slot = _at(x, j)
        x["kc"][page, 1, slot, 3] = float("nan")
        _compare(x, [0, 1])
    x["kc"][x["table"][0].long(), 0] = float("nan")  # nothing else in one group
    _compare(x, [0, 1])


def _one_key_takes_all(x, winner, j, minus_inf):
    """The key at `winner` leaves the others weights of e^-250 or less (or e^-inf); the one at `j` has values that are not
    finite in some dims."""
    x["q"][..., 0] = 8.0
    fp8 = x["ks"] is not None
    if minus_inf:
        x["kc"][..., 0] = -float("inf")
    for g in range(GROUPS):
        page, slot = _at(x, winner)
        x["kc"][page, g, slot] = torch.zeros(DIM).to(x["kc"].dtype)
        x["kc"][page, g, slot, 0] = 448.0 if fp8 else 300.0
        if fp8:
            x["ks"][page, g] = 2.0
        page, slot = _at(x, j)
        x["vc"][page, g, slot, 1] = float("nan" if fp8 else "inf")
        x["vc"][page, g, slot, 17] = float("nan" if fp8 else "-inf")
        x["vc"][page, g, slot, 40] = float("nan")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,fp8", TYPES)
@pytest.mark.parametrize("tokens,ways", WAYS)
@pytest.mark.parametrize("minus_inf", (False, True))
def test_values_of_keys_without_weight(minus_inf, tokens, ways, dtype, fp8, device):
    """They count wherever the key lies: what a row gives does not depend on which wave or workgroup has its step."""
    if minus_inf and fp8:
        pytest.skip("e4m3 has no infinity")
    for j in (0, 33, 77, 150, 200, KEYS - 1):
        x = _inputs(tokens, dtype, fp8, device)
        _one_key_takes_all(x, 170, j, minus_inf)
        _compare(x, [0, 1], exact=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,fp8", TYPES)
@pytest.mark.parametrize("tokens,ways", WAYS)
@pytest.mark.parametrize("weights", ("usual", "none", "minus_inf"))
def test_infinite_values_are_the_formulas(weights, tokens, ways, dtype, fp8, device):
    """Infinities stay themselves beside finite values, NaN comes of both signs, of a NaN and under a logit of -inf; dims
    without any are as ever."""
    if weights == "minus_inf" and fp8:
        pytest.skip("e4m3 has no infinity")
    for j, other in ((0, 1), (33, 300), (200, 40), (KEYS - 1, 0)):
        x = _inputs(tokens, dtype, fp8, device)
        if weights != "usual":
            _one_key_takes_all(x, 170, j, weights == "minus_inf")
        if not fp8:
            page, slot = _at(x, j)
            x["vc"][page, 0, slot, 3:6] = torch.tensor([float("inf"), -float("inf"), float("inf")])
            page, slot = _at(x, other)
            x["vc"][page, 0, slot, 5:8] = torch.tensor([-float("inf"), float("nan"), float("inf")])
            page, slot = _at(x, 170)
            x["vc"][page, 1, slot, 63] = float("inf")  # (of the key with the weight, where one has it)
            x["vc"][page, 1, slot, 62] = -float("inf")
        else:
            page, slot = _at(x, j)
            x["vc"][page, 0, slot, 3] = float("nan")
            x["vs"][_at(x, other)[0], 1] = float("inf")  # a scale is a factor like any other (0 x inf: NaN)
        _compare(x, [0, 1])


@pytest.mark.gpu
def test_infinite_values_of_keys_not_seen(device):
    """Behind a token, in blocks that it did not select, and in pages that are not there."""
    x = _inputs(2, torch.bfloat16, False, device)
    want = _call(x)
    page, slot = _at(x, KEYS)  # the second token's own position: behind the first one, in a block no one selected
    x["vc"][page, :, slot] = float("inf")
    got = _call(x)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    x["vc"][_at(x, 100)[0], :, 5] = float("inf")
    x["ids"][1] = torch.where(x["ids"][1] == 100 // BLOCK, -1, x["ids"][1])
    got = _call(x)
    assert torch.isinf(got[0][0]).all() and torch.isfinite(got[0][1]).all()
    x["table"][0, 100 // PAGE] = -1
    assert torch.isfinite(_call(x)[0]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_one_infinity_at_other_dims_and_head_counts(dtype, device):
    """More head tiles than one, dims that fill no tile, steps of half a block."""
    gen = torch.Generator().manual_seed(9)
    dim, page, block, ratio, keys = 80, 16, 48, 20, 150
    pages = 10
    q = torch.randn(1, ratio, dim, generator=gen).to(dtype).to(device)
    kc, vc = (torch.randn(pages, 1, page, dim, generator=gen).to(dtype).to(device) for _ in range(2))
    table = torch.randperm(pages, generator=gen, dtype=torch.int32)[None].to(device)
    vc[int(table[0, 3]), 0, 1, 77] = float("inf")  # position 49
    vc[int(table[0, 9]), 0, 5, 2] = -float("inf")  # position 149, the token's own
    ids = torch.tensor([[[3, 1, 0, 1]]], dtype=torch.int32, device=device)
    out = msa.m3_sparse_attention_paged(q, kc, vc, ids, table, cu_tensor([1], device),
                                        torch.tensor([keys - 1], dtype=torch.int32, device=device), block_size=block)
    assert (out[:, :, 77] == float("inf")).all() and (out[:, :, 2] == -float("inf")).all()
    out[:, :, 77] = out[:, :, 2] = 0
    assert torch.isfinite(out).all()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,ways", WAYS)
def test_sums_past_the_range_give_no_wrong_number(tokens, ways, device):
    """bf16 values whose weighted sum leaves fp32's range before it is divided: the mean of them, or an infinity."""
    for value in (3e38, 2e37, 1e35):
        x = _inputs(tokens, torch.bfloat16, False, device)
        x["vc"].fill_(value)
        out, _ = _call(x)
        want = float(torch.tensor(value).bfloat16())
        near = (out.double() - want).abs() <= 2 ** -8 * want
        assert (near | (out == float("inf"))).all()
    assert near.all()  # 384 x 1e35 is in range
