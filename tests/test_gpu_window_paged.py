"""m3_window_attention_paged and m3_tree_attention_paged against float64, in both cache widths.

Tolerance, with h half a step of a type relative to the value: logits are fp32 products of exact terms, so a dot of D
terms is off by D 2^-23 sum |q||k| at most, times the scale, and by 2^-22 of itself; a weight by twice that error d of a logit
(its own and the maximum's) and its exponential's 2^-22. A weight enters the second product as two terms (2^-17 left
out) where no sequence has more than 16 rows a key head, and for fp16 queries over an 8-bit cache, and is rounded once
otherwise (h of its type). The second product and its sums, over waves and workgroups, add 2^-16.
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
    two = max(lengths) * ratio <= 16
    two |= fp8 and x["q"].dtype == torch.float16
    left_out = 2.0 ** -17 if two else torch.finfo(x["q"].dtype).eps / 2
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
    ([512], [100], 1, 2, 64, 64, 90, 1, torch.bfloat16, False),
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


def test_scales_of_any_sign():
    for lengths, fp8 in (([1, 2], False), ([1, 40], False), ([2, 1], True), ([3, 40], True)):
        x = setup(lengths, [70, 300], 2, 4, 64, 16, torch.float16, fp8)
        for scale in (-0.4, 0.0, 3.0):
            check(x, lengths, [70, 300], 50, 4, scale=scale)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("new", [1, 40])
def test_pages_that_do_not_exist(new, fp8):
    """Entries of -1 and past the cache in the middle, in the window and in front of it, lengths behind the table, no table."""
    lengths, context = [new, new, new, new], [500, 333, 700, 90]
    x = setup(lengths, context, 2, 4, 64, 16, torch.bfloat16, fp8, width=50)
    x["table"][0, 3:20] = -1
    x["table"][1, 20] = x["kc"].shape[0]
    x["table"][1, 5] = 1 << 30
    x["table"][2, ::2] = -7
    x["table"][3, :] = -1
    for window, sinks in ((None, 0), (100, 4), (30, 70), (1, 0)):
        check(x, lengths, context, window, sinks)
    short = dict(x, table=x["table"][:, :21].contiguous())
    check(short, lengths, context, None, 0)
    check(short, lengths, context, 100, 4)
    none = dict(x, table=x["table"][:, :0].contiguous())
    out, lse = call(none, None, 0)
    assert not out.any() and (lse == float("-inf")).all()
    empty = dict(x, kc=x["kc"][:0], vc=x["vc"][:0], ks=x["ks"][:0] if fp8 else None, vs=x["vs"][:0] if fp8 else None)
    out, lse = call(empty, 100, 4)
    assert not out.any() and (lse == float("-inf")).all()
    far = dict(x, context=torch.tensor([2 ** 31 - 1, 333, -1, -2 ** 31], dtype=torch.int32, device="cuda"))
    out, lse = call(far, 100, 0)
    assert (lse[:new] == float("-inf")).all() and not out[:new].any() and not out[2 * new:].any()
    assert torch.isfinite(lse[new:2 * new]).all() and (lse[2 * new:] == float("-inf")).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("lengths", [[1, 3, 2], [40, 3, 70]], ids=("few", "many"))
def test_strided_caches_streams_and_a_table_of_columns(lengths, fp8):
    context = [300, 17, 64]
    x = setup(lengths, context, 2, 4, 64, 16, torch.bfloat16, fp8)
    want = call(x, 60, 3)
    moved = dict(x, table=x["table"].t().contiguous().t(), q=x["q"].transpose(0, 1).contiguous().transpose(0, 1))
    for name in ("kc", "vc"):
        c = x[name]
        both = torch.zeros(c.shape[0], c.shape[2], c.shape[1], 2 * c.shape[3], device="cuda").to(c.dtype)  # slots in front of heads
        both[..., :64] = c.transpose(1, 2)
        moved[name] = both[..., :64].transpose(1, 2)
    got = call(moved, 60, 3)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(x, 60, 3)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_past_32_bits():
    """Pages whose first value is 2^31 values and more into the cache."""
    pages, page, dim = 140_000, 128, 128
    cache = torch.zeros(pages, 1, page, dim, dtype=torch.bfloat16, device="cuda")
    assert cache.numel() > 2 ** 31
    lengths, context = [1, 20], [700, 300]
    small = setup(lengths, context, 1, 8, dim, page, torch.bfloat16, False)
    x = dict(small, kc=cache, vc=torch.zeros_like(cache), table=torch.full_like(small["table"], -1))
    at = pages - 1
    for s in range(2):
        for m in range(small["table"].shape[1]):
            p = int(small["table"][s, m])
            if p >= 0:
                x["kc"][at], x["vc"][at] = small["kc"][p], small["vc"][p]
                x["table"][s, m] = at
                at -= 3
    got, want = call(x, 500, 4), call(small, 500, 4)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("lengths,context", [([1, 1], [900, 40]), ([40, 17], [900, 40]), ([1], [20000])], ids=("few", "many", "split"))
def test_values_that_are_not_finite(lengths, context, fp8):
    """An infinity and a NaN of one key's value: the dim of every row that sees it, whatever the weight, and nothing else."""
    g, ratio, d, page = 2, 4, 64, 16
    x = setup(lengths, context, g, ratio, d, page, torch.bfloat16, fp8)
    want, want_lse, tol, lse_tol = oracle(x, lengths, context, 500, 2, d ** -0.5)
    for at, value in ((context[0] - 3, float("inf")), (0, float("-inf")), (context[0] - 450, float("nan")), (context[0] - 600, float("nan")),
                      (context[0], float("nan"))):
        if fp8 and value == value:
            value = float("nan")  # (e4m3 has no infinities)
        y = dict(x, vc=x["vc"].clone())
        p = int(x["table"][0, at // page])
        y["vc"].view(torch.uint8 if fp8 else torch.bfloat16)[p, 1, at % page, 5] = 0x7F if fp8 else value
        out, lse = call(y, 500, 2)
        pos = torch.arange(context[0], context[0] + lengths[0], device="cuda")
        sees = (pos >= at) & ((pos - at < 500) | (at < 2))
        hit = torch.zeros_like(out, dtype=torch.bool)
        hit[:lengths[0], ratio:, 5] = sees[:, None]
        assert (torch.isnan(out[hit]).all() if value != value else (out[hit] == value).all())
        assert ((out.double() - want).abs() <= tol)[~hit].all()
        assert ((lse.double() - want_lse).abs() <= lse_tol).all()


def test_a_value_under_a_weight_of_zero():
    """A key so far from the row's best that its weight is 0 in fp32, its value an infinity."""
    for lengths in ([1], [40]):
        x = setup(lengths, [300], 1, 4, 64, 16, torch.bfloat16, False)
        p = int(x["table"][0, 0])
        x["kc"][p, 0, 5] = (-100 * x["q"][0, 2].float().sign()).bfloat16()
        x["vc"][p, 0, 5, 9] = float("inf")
        out, lse = call(x, None, 0)
        assert (out[:, :, 9] == float("inf")).all() and torch.isfinite(out[:, :, :9]).all() and torch.isfinite(lse).all()


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float16, 256)])
@pytest.mark.parametrize("n", [3, 24])
@pytest.mark.parametrize("drafted", [False, True])
def test_several_values_that_are_not_finite(dtype, dim, n, drafted):
    """Infinities that meet, beside NaN, among cached tokens, under a logit of -inf and among a tree's nodes: NaN, +inf and
    -inf stand where the formula over the visible tokens has them, and the other dims are within the bound."""
    page, context, window, inf = 16, 200, 150, float("inf")
    x = setup([n], [context], 1, 4, dim, page, dtype, False)
    x["q"][:, :, 0] = x["q"][:, :, 0].abs() + 0.5
    x["parents"] = tree([n]) if drafted else None

    def put(cache, at, d, value):
        cache[x["table"][0, at // page].item(), 0, at % page, d] = value

    x["kc"], x["vc"] = x["kc"].clone(), x["vc"].clone()
    for at, d, value in ((120, 5, inf), (130, 5, -inf), (140, 6, float("nan")), (140, 7, inf), (141, 7, inf), (0, 8, -inf), (20, 10, inf),
                         (60, 11, inf), (context + 1, 12, inf), (context + 2, 12, -inf), (context + n - 1, 13, -inf)):
        put(x["vc"], at, d, value)
    put(x["kc"], 150, 0, -inf)
    put(x["vc"], 150, 9, inf)
    out, lse = call(x, window, 2)
    # (the bound's terms: of the cache with zeros for what is not finite, a logit of 0 in place of -inf)
    _, _, tol, _ = oracle(dict(x, kc=x["kc"].nan_to_num(0.0, 0.0, 0.0), vc=x["vc"].nan_to_num(0.0, 0.0, 0.0)), [n], [context], window, 2,
                          dim ** -0.5)
    own = None if x["parents"] is None else x["parents"].tolist()
    rows = x["q"].double()
    ids = x["table"][0].long()
    j = torch.arange(context + n, device="cuda")
    k, v = (x[c][ids[j // page], 0, j % page].double() for c in ("kc", "vc"))
    for i, path in enumerate(paths(own, n)):
        low = context + len(path) - window
        seen = [t for t in range(context) if t >= low or t < 2] + [context + node for node in path]
        for h in range(4):
            p = torch.softmax(k[seen] @ rows[i, h] * dim ** -0.5, 0)
            z = (p[:, None] * v[seen]).sum(0)
            for name in (torch.isnan, torch.isposinf, torch.isneginf):
                assert torch.equal(name(out[i, h]), name(z)), (i, h, name)
            clean = torch.isfinite(z)
            assert ((out[i, h].double() - z).abs() <= tol[i, h])[clean].all()


def test_keys_and_queries_that_are_not_finite():
    lengths, context = [30, 2], [100, 50]
    x = setup(lengths, context, 1, 4, 64, 16, torch.float16, False)
    want = call(x, 40, 1)
    y = dict(x, kc=x["kc"].clone())
    p = int(x["table"][0, 110 // 16])
    y["kc"][p, 0, 110 % 16, 0] = float("nan")  # seen by tokens 10 to 29 of the first sequence
    out, lse = call(y, 40, 1)
    assert torch.isnan(out[10:30]).all() and torch.isnan(lse[10:30]).all()
    rest = torch.ones(32, dtype=torch.bool)
    rest[10:30] = False
    assert torch.equal(out[rest], want[0][rest]) and torch.equal(lse[rest], want[1][rest])
    z = dict(x, q=x["q"].clone())
    z["q"][3, 1, 7] = float("inf")
    out, lse = call(z, 40, 1)
    assert not torch.isfinite(out[3, 1]).any()
    rest = torch.ones(32, 4, dtype=torch.bool)
    rest[3, 1] = False
    assert torch.equal(out[rest], want[0][rest]) and torch.equal(lse[rest], want[1][rest])


def test_a_chain_is_a_drafted_run():
    lengths, context = [9, 1, 40], [300, 5, 64]
    for fp8 in (False, True):
        x = setup(lengths, context, 2, 4, 64, 16, torch.bfloat16, fp8)
        chain = torch.cat([torch.arange(n) - 1 for n in lengths]).to(torch.int32).cuda()
        for window, sinks in ((None, 0), (20, 3)):
            a, b = call(x, window, sinks), call(dict(x, parents=chain), window, sinks)
            x["parents"] = None
            want, _, tol, _ = oracle(x, lengths, context, window, sinks, 64 ** -0.5)
            assert ((b[0].double() - want).abs() <= tol).all()
            assert window or all(torch.equal(u, w) for u, w in zip(a, b))


@pytest.mark.parametrize("lengths", [[1, 1, 1], [17, 5, 40]], ids=("single", "tree"))
def test_captured_calls_replay_at_new_lengths_and_trees(lengths):
    x = setup(lengths, [400, 200, 300], 2, 8, 64, 16, torch.bfloat16, True)
    x["context"].copy_(torch.tensor([40, 20, 30]))
    x["parents"] = tree(lengths)
    seqs = msa.prepare_sequences(x["cu"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(x, 100, 4, seqs)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, call(x, 100, 4, seqs)))
    for turn, context in enumerate(([40, 20, 30], [400, 200, 300], [0, 199, -1], [390, 1, 16])):
        x["context"].copy_(torch.tensor(context))
        x["parents"].copy_(tree(lengths, seed=turn))
        graph, held = graphs[turn % 2]
        graph.replay()
        want = call(x, 100, 4)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_a_million_sequences():
    """One call of 2^20 requests and 2^24 rows."""
    n, hq, d, page = 1 << 20, 16, 16, 16
    gen = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn(n, hq, d, generator=gen, device="cuda").bfloat16()
    kc, vc = (torch.randn(4096, 1, page, d, generator=gen, device="cuda").bfloat16() for _ in range(2))
    table = torch.randint(0, 4096, (n, 2), generator=gen, device="cuda", dtype=torch.int32)
    context = torch.randint(-1, 31, (n,), generator=gen, device="cuda", dtype=torch.int32)
    cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    out, lse = msa.m3_window_attention_paged(q, kc, vc, table, cu, context, window_size=20, sink_tokens=1, return_lse=True)
    for a in (0, 500_000, n - 20):
        part = slice(a, a + 20)
        x = dict(q=q[part], kc=kc, vc=vc, ks=None, vs=None, table=table[part], parents=None)
        want, want_lse, tol, lse_tol = oracle(x, [1] * 20, context[part].tolist(), 20, 1, d ** -0.5)
        assert ((out[part].double() - want).abs() <= tol).all()
        none = want_lse == float("-inf")
        assert torch.equal(lse[part] == float("-inf"), none)
        assert ((lse[part].double() - want_lse).abs() <= lse_tol)[~none].all()


def test_differentiating_raises():
    x = setup([2], [20], 1, 2, 64, 16, torch.bfloat16, False)
    x["q"].requires_grad_()
    for parents in (None, tree([2])):
        out, _ = call(dict(x, parents=parents), 4, 0)
        with pytest.raises(RuntimeError, match="no gradients"):
            out.float().sum().backward()
        with torch.no_grad():
            assert not call(dict(x, parents=parents), 4, 0)[0].requires_grad
