"""m3_window_attention_paged and m3_tree_attention_paged against float64, in both cache widths.

Tolerance, with h half a step of a type relative to the value: logits are fp32 products of exact terms, so a dot of D
terms is off by D 2^-23 sum |q||k| at most, times the scale, and by 2^-22 of itself; a weight by twice that error d of a logit
(its own and the maximum's) and its exponential's 2^-22. A weight enters the second product as two terms (2^-17 left
out) where no sequence has more than 16 rows a key head or the head dim is above 128, and is rounded once otherwise (h
of the type of that product, bf16 for 8-bit caches). The second product and its sums, over waves and workgroups, add 2^-16.
So |out - exact| <= (2 d + left out + 2^-16) max |v| + h |out|. The lse is off by d and 2^-20 of its size.
"""

from __future__ import annotations

import pytest
import torch

import msa_triton_amd as msa
from msa_triton_amd.paged import FP8
from tests.helpers import cu_list, cu_tensor
from tests.paged_helpers import page_table

pytestmark = pytest.mark.gpu


def setup(lengths, context, groups, ratio, dim, page, dtype, fp8, seed=23, width=None, device="cuda"):
    """A batch whose cache holds NaN wherever no token of it lies."""
    gen = torch.Generator().manual_seed(seed)
    totals = [n + c if c >= 0 else 0 for n, c in zip(lengths, context)]
    table, count = page_table(totals, page, gen, width=width)
    used = torch.zeros(count, page, dtype=torch.bool)
    for s, n in enumerate(totals):
        for m in range(min(-(-n // page), table.shape[1])):
            used[int(table[s, m]), :min(page, n - m * page)] = True
    x = dict(q=(torch.randn(sum(lengths), groups * ratio, dim, generator=gen) * 1.5).to(dtype), ks=None, vs=None)
    for name in ("k", "v"):
        c = torch.randn(count, groups, page, dim, generator=gen)
        if fp8:
            x[name + "s"] = torch.exp2(torch.randint(-7, -3, (count, groups), generator=gen).float()) * (
                0.7 if name == "k" else 1.3)
            c = (c / x[name + "s"][:, :, None, None]).clamp(-448, 448).to(FP8)
            c.view(torch.uint8)[~used[:, None].expand(-1, groups, -1)] = 0x7F  # NaN
            x[name + "s"][~used.any(1)] = float("nan")
        else:
            c = c.to(dtype)
            c[~used[:, None].expand(-1, groups, -1)] = float("nan")
        x[name + "c"] = c
    x["table"] = table
    x["cu"] = cu_tensor(lengths)
    x["context"] = torch.tensor(context, dtype=torch.int32)
    x["parents"] = None
    return {n: None if v is None else v.to(device) for n, v in x.items()}


def tree(lengths, seed=3, device="cuda"):
    """Parents by place, -1 for children of the context; each tree is also given entries that mean nothing else than -1."""
    gen = torch.Generator().manual_seed(seed)
    out = []
    for n in lengths:
        for i in range(n):
            back = int(torch.randint(1, 6, (1,), generator=gen))
            out.append(i - back if i - back >= 0 else (-1, i, i + 3, -7, 1 << 30)[back - 1])
    return torch.tensor(out, dtype=torch.int32, device=device)


def paths(parents, n):
    """Of each node, its ancestors and itself, from the top."""
    out = []
    for i in range(n):
        p = int(parents[i]) if parents is not None else i - 1
        out.append([*(out[p] if 0 <= p < i else []), i])
    return out


def oracle(x, lengths, context, window, sinks, scale):
    """(out, lse, how far out may be off, how far lse may be) in float64 on the GPU."""
    q = x["q"].double()
    total, heads, dim = q.shape
    pages, groups, page, _ = x["kc"].shape
    ratio = heads // groups
    fp8 = x["kc"].dtype == FP8
    two = max(lengths) * ratio <= 16 or dim > 128
    left_out = 2.0 ** -17 if two else torch.finfo(torch.bfloat16 if fp8 else x["q"].dtype).eps / 2
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((total, heads), float("-inf"), dtype=torch.float64, device=q.device)
    lse_tol = torch.zeros_like(lse)
    cu = cu_list(lengths)
    for s, (a, n, c) in enumerate(zip(cu, lengths, context)):
        if c < 0 or n == 0 or pages == 0:
            continue
        j = torch.arange(c + n, device=q.device)
        m = j // page
        held = m < x["table"].shape[1]
        ids = torch.where(held, x["table"][s][m.clamp(max=max(0, x["table"].shape[1] - 1))], -1).long() if x[
            "table"].shape[1] else torch.full_like(j, -1)
        held &= (ids >= 0) & (ids < pages)
        ids = torch.where(held, ids, 0)
        k, v = x["kc"][ids, :, j % page].double(), x["vc"][ids, :, j % page].double()  # [L, G, D]
        if fp8:
            k, v = k * x["ks"][ids].double()[..., None], v * x["vs"][ids].double()[..., None]
        seen = torch.zeros(n, c + n, dtype=torch.bool)
        own = None if x["parents"] is None else x["parents"][a:a + n].tolist()
        for i, path in enumerate(paths(own, n)):
            pos = c + len(path) - 1
            low = max(0, pos - window + 1) if window else 0
            seen[i, low:c] = True
            seen[i, :min(sinks, c)] = True
            for deep, node in enumerate(path):
                seen[i, c + node] = c + deep >= low or c + deep < sinks
        seen = seen.to(q.device) & held
        for h in range(heads):
            rows, kk, vv = q[a:a + n, h], k[:, h // ratio], v[:, h // ratio]
            kk, vv = (torch.where((seen.any(0) & held)[:, None], y, 0.0) for y in (kk, vv))
            logit = (rows @ kk.T * scale).masked_fill(~seen, float("-inf"))
            d = (dim * 2.0 ** -23 * (rows.abs() @ kk.abs().T) * abs(scale) + 2.0 ** -22 * logit.abs()).masked_fill(~seen, 0.0)
            d = d.amax(1)
            some = seen.any(1)
            lse[a:a + n, h] = torch.logsumexp(logit, 1)
            p = torch.softmax(logit, 1)
            out[a:a + n, h] = torch.where(some[:, None], p @ vv, 0.0)
            top = (vv.abs().amax(1)[None] * seen).amax(1)
            tol[a:a + n, h] = ((2 * d + 2.0 ** -22 + left_out + 2.0 ** -16) * top)[:, None]
            lse_tol[a:a + n, h] = d + 2.0 ** -20 * lse[a:a + n, h].abs().clamp(min=1.0)
    tol += torch.finfo(x["q"].dtype).eps / 2 * (out.abs() + tol)
    return out, lse, tol, lse_tol


def call(x, window, sinks, cu=None, **kw):
    args = (x["q"], x["kc"], x["vc"], x["table"], x["cu"] if cu is None else cu, x["context"])
    kw = dict(window_size=window, sink_tokens=sinks, k_scale=x["ks"], v_scale=x["vs"], return_lse=True, **kw)
    if x["parents"] is None:
        return msa.m3_window_attention_paged(*args, **kw)
    return msa.m3_tree_attention_paged(*args, x["parents"], **kw)


def check(x, lengths, context, window, sinks, scale=None, **kw):
    out, lse = call(x, window, sinks, scale=scale, **kw)
    want, want_lse, tol, lse_tol = oracle(x, lengths, context, window, sinks, x["q"].shape[2] ** -0.5 if scale is None else scale)
    assert torch.isfinite(out).all()
    part = ((out.double() - want).abs() / tol.clamp(min=1e-30)).max().item()
    assert part <= 1.0, f"out: {part:.2f} of the bound"
    none = want_lse == float("-inf")
    assert torch.equal(lse == float("-inf"), none) and not out[none].any()
    part = ((lse.double() - want_lse).abs() / lse_tol.clamp(min=1e-30))[~none]
    assert not part.numel() or part.max() <= 1.0, f"lse: {part.max():.2f} of the bound"
    return out, lse


CASES = [  # lengths, context, groups, ratio, dim, page, window, sinks, dtype, fp8
    ([1], [0], 1, 1, 64, 16, None, 0, torch.bfloat16, False),
    ([1], [20011], 4, 8, 128, 128, 4096, 4, torch.bfloat16, False),
    ([1], [20011], 1, 8, 128, 64, None, 0, torch.float16, True),       # one tile over many workgroups
    ([1] * 24, "mixed", 4, 8, 128, 64, None, 0, torch.bfloat16, False),
    ([1] * 24, "mixed", 2, 8, 128, 64, 300, 4, torch.bfloat16, True),
    ([1] * 24, "mixed", 2, 4, 96, 16, 33, 70, torch.float16, True),
    ([1, 4, 2, 0, 3], [63, 64, 65, 9, 1000], 2, 4, 64, 64, 50, 3, torch.float16, False),  # 16 rows at most
    ([1, 5, 2, 0, 3], [63, 64, 65, 9, 1000], 2, 4, 64, 64, 50, 3, torch.float16, False),  # 20
    ([40, 1, 300], [500, 0, 77], 2, 5, 128, 128, 100, 10, torch.bfloat16, False),         # a ratio of 5
    ([40, 1, 300], [500, 0, 77], 2, 5, 128, 32, None, 0, torch.bfloat16, True),
    ([129, 64], [0, 1], 1, 1, 64, 16, 16, 1, torch.float16, True),
    ([77, 3], [40, 900], 2, 3, 256, 64, 64, 2, torch.bfloat16, False),
    ([77, 3], [40, 900], 2, 3, 208, 64, 64, 2, torch.float16, True),
    ([1, 1, 1], [5, -1, 300], 2, 40, 128, 64, 31, 0, torch.bfloat16, False),  # more heads a group than a tile has rows
    ([2, 7, 1], [-1, 30, -5], 2, 2, 16, 16, 3, 200, torch.bfloat16, False),   # every cached key is a first token
    ([1] * 130, "mixed", 1, 4, 64, 16, 64, 2, torch.bfloat16, False),         # more sequences than a wave has lanes
    ([1, 0, 3] * 100, "mixed", 1, 8, 64, 16, None, 0, torch.float16, False),
]


def contexts(context, lengths):
    return [(37 * i * i + 11 * i) % 2111 if i % 9 else 0 for i in range(len(lengths))] if context == "mixed" else context


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in (len(c[0]), max(c[0]), *c[2:])))
def test_window_against_the_formula(case):
    lengths, context, g, ratio, d, page, window, sinks, dtype, fp8 = case
    context = contexts(context, lengths)
    x = setup(lengths, context, g, ratio, d, page, dtype, fp8)
    out, lse = check(x, lengths, context, window, sinks)
    again = call(x, window, sinks, msa.prepare_sequences(x["cu"]))
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


TREES = [  # lengths, context, groups, ratio, dim, page, window, sinks, dtype, fp8
    ([1], [0], 1, 1, 64, 16, None, 0, torch.bfloat16, False),
    ([2, 1, 2], [0, 7, 33], 2, 8, 128, 16, None, 0, torch.bfloat16, False),   # 16 rows
    ([15], [1999], 4, 8, 128, 128, None, 0, torch.bfloat16, False),
    ([64, 48, 0, 17, 1], [500, 0, 8, 3000, 129], 2, 8, 128, 64, None, 0, torch.bfloat16, True),
    ([64, 48, 0, 17, 1], [500, 0, 8, 3000, -1], 2, 5, 96, 64, 40, 4, torch.float16, True),
    ([130, 33], [1000, 31], 1, 4, 64, 16, 6, 33, torch.float16, False),  # windows that end inside the paths
    ([130, 33], [1000, 31], 1, 1, 256, 32, 3, 40, torch.bfloat16, False),
    ([1024], [100], 1, 2, 64, 64, 90, 1, torch.bfloat16, False),
    ([9] * 80, "mixed", 2, 2, 64, 16, None, 0, torch.float16, True),
]


@pytest.mark.parametrize("case", TREES, ids=lambda c: "-".join(str(x) for x in (len(c[0]), max(c[0]), *c[2:])))
def test_tree_against_the_formula(case):
    lengths, context, g, ratio, d, page, window, sinks, dtype, fp8 = case
    context = contexts(context, lengths)
    x = setup(lengths, context, g, ratio, d, page, dtype, fp8)
    x["parents"] = tree(lengths)
    out, lse = check(x, lengths, context, window, sinks)
    again = call(x, window, sinks, msa.prepare_sequences(x["cu"]))
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
