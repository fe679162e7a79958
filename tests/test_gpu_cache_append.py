"""m3_cache_append against float64: 16-bit and 8-bit caches, page ends, scales that grow, absent pages, strides.

An 8-bit byte is a single rounding of the exact value, so bytes and scales are compared for equality: the
kernel's FP64 values are some 2^-50 off, and a value that close to a rounding border does not occur by
chance in these sizes (about 1e5 values, a chance below 1e5 x 2^-45). 16-bit keys are held to the norm's bounds,
16-bit values to equality.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import msa_triton_amd as msa
from msa_triton_amd.paged import FP8
from tests.helpers import cu_list, cu_tensor
from tests.paged_helpers import page_table, place, round_e4m3, scale_for


def _turned(x, w, table, pos, eps):
    """Norm and rotation of rows [T, H, D] in float64 numpy."""
    x = x.double().cpu().numpy()
    if w is not None:
        with np.errstate(invalid="ignore"):
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * w.double().cpu().numpy()
    if table is not None:
        t = table.double().cpu().numpy()
        half = t.shape[1] // 2
        rows = np.full((len(pos), t.shape[1]), np.nan)
        for i, p in enumerate(pos):
            if 0 <= p < t.shape[0]:
                rows[i] = t[p]
        cos, sin = rows[:, None, :half], rows[:, None, half:]
        a, b = x[..., :half].copy(), x[..., half:2 * half].copy()
        with np.errstate(invalid="ignore"):
            x[..., :half], x[..., half:2 * half] = a * cos - b * sin, b * cos + a * sin
    return x


def _append_fp8(cache, scale, rows, table, lengths, context):
    """The oracle: bytes' values [P, H, page, D] and scales [P, H] after the append."""
    pages, heads, page, _ = cache.shape
    held, scale = cache.float().double().cpu().numpy(), scale.double().cpu().numpy().copy()
    for s, (a, n) in enumerate(zip(cu_list(lengths), lengths)):
        c = context[s]
        if c < 0:
            continue
        todo = {}
        for i in range(n):
            at = place(table, page, s, c + i, pages)
            if at is not None:
                todo.setdefault(at[0], []).append((at[1], a + i))
        for p, items in todo.items():
            kept = items[0][0]
            for h in range(heads):
                new = np.stack([rows[t, h] for _, t in items])
                before = scale[p, h] if kept else 0.0
                after = max(before, scale_for(np.abs(new[np.isfinite(new)]).max(initial=0.0)))
                if after != before:
                    held[p, h, :kept] = round_e4m3(held[p, h, :kept] * (before / after))
                for (slot, _), row in zip(items, new):
                    held[p, h, slot] = round_e4m3(row / after) if after else np.where(np.isfinite(row), row, np.nan)
                scale[p, h] = after
    return held, scale


def _setup(lengths, context, heads, dim, index_dim, rot, page, dtype, fp8, device, seed=11, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    total = sum(lengths)
    totals = [n + c if c >= 0 else 0 for n, c in zip(lengths, context)]
    table, count = page_table(totals, page, gen)

    def rand(*shape):
        return torch.randn(*shape, generator=gen)

    x = dict(k=(rand(total, heads, dim) * 3).to(dtype), v=(rand(total, heads, dim) * spread).to(dtype),
             ik=rand(total, 1, index_dim).to(dtype), wk=(1 + 0.2 * rand(dim)).to(dtype),
             wi=(1 + 0.2 * rand(index_dim)).to(dtype))
    if fp8:
        for name in ("k", "v"):
            scale = torch.exp2(torch.randint(-9, -4, (count, heads), generator=gen).float())
            x[name + "s"] = scale
            x[name + "c"] = rand(count, heads, page, dim).mul(60).clamp(-448, 448).to(FP8)
    else:
        x["ks"] = x["vs"] = None
        x["kc"], x["vc"] = (rand(count, heads, page, dim).to(dtype) for _ in range(2))
    x["ic"] = rand(count, 1, page, index_dim).to(dtype)
    x = {n: None if t is None else t.to(device) for n, t in x.items()}
    x["table"] = table
    x["rope"] = msa.rope_table(max(totals) + 1, rot, device=device) if rot else None
    x["cu"] = cu_tensor(lengths, device)
    x["context"] = torch.tensor(context, dtype=torch.int32, device=device)
    return x


def _call(x, **change):
    a = dict(x, **change)
    msa.m3_cache_append(a["k"], a["v"], a["kc"], a["vc"], a["table"].to(a["k"].device), a["cu"], a["context"],
                        index_k=a["ik"], index_cache=a["ic"], k_scale=a["ks"], v_scale=a["vs"], k_weight=a["wk"],
                        index_weight=a["wi"], cos_sin=a["rope"], eps=1e-5)


def _positions(lengths, context):
    return [c + i for n, c in zip(lengths, context) for i in range(n)]


def _norm_close(got, want):
    """Half a step of the type, 16 fp32 steps of the row's largest value."""
    step = torch.finfo(got.dtype).eps / 2
    got = got.double().cpu().numpy()
    bound = step * (1 + 2 ** -8) * np.abs(want) + 16 * 2.0 ** -24 * np.abs(want).max(-1, keepdims=True) + 2 ** -24 * step
    assert (np.abs(got - want) <= bound).all()


CASES = [  # lengths, context, heads, D, Di, rot, page, dtype
    ([1], [0], 1, 64, 64, 64, 16, torch.bfloat16),
    ([1, 1, 1, 1], [15, 16, 31, 200], 4, 128, 128, 64, 64, torch.bfloat16),
    ([1, 0, 5, 70], [127, 3, 126, 0], 2, 128, 64, 32, 128, torch.float16),
    ([300, 33], [0, 250], 3, 96, 96, 96, 256, torch.bfloat16),
    ([40, 3, 17], [-1, 13, -7], 2, 256, 128, 64, 16, torch.float16),
    ([21, 50], [9, 40], 2, 48, 16, 12, 32, torch.bfloat16),   # a rotation off 16-byte runs
    ([130], [60], 8, 64, 32, 0, 64, torch.bfloat16),          # no rotation
    ([(i * 7) % 3 for i in range(150)], [(i * 37) % 50 - 5 for i in range(150)], 1, 32, 16, 16, 16,
     torch.bfloat16),                                         # more sequences than lanes
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("fp8", [False, True])
def test_append(case, fp8, device):
    lengths, context, heads, dim, index_dim, rot, page, dtype = case
    x = _setup(*case, fp8, device)
    before = {n: x[n].clone() for n in ("kc", "vc", "ic")}
    old_scale = {n: None if x[n] is None else x[n].clone() for n in ("ks", "vs")}
    _call(x)
    pos = _positions(lengths, context)
    keys, index = _turned(x["k"], x["wk"], x["rope"], pos, 1e-5), _turned(x["ik"], x["wi"], x["rope"], pos, 1e-5)
    values = x["v"].double().cpu().numpy()
    written = torch.zeros(x["kc"].shape[0], page, dtype=torch.bool)
    where = []
    for s, (a, n) in enumerate(zip(cu_list(lengths), lengths)):
        for i in range(n):
            at = place(x["table"], page, s, context[s] + i, x["kc"].shape[0]) if context[s] >= 0 else None
            if at is not None:
                written[at] = True
                where.append((a + i, *at))
    t, p, slot = (torch.tensor(z, device=device) for z in zip(*where))
    tn = t.cpu().numpy()
    _norm_close(x["ic"][p, :, slot], index[tn])
    kept = ~written.to(device)
    assert torch.equal(x["ic"].transpose(1, 2)[kept], before["ic"].transpose(1, 2)[kept])
    if not fp8:
        _norm_close(x["kc"][p, :, slot], keys[tn])
        assert torch.equal(x["vc"][p, :, slot], x["v"][t])
        for n in ("kc", "vc"):
            assert torch.equal(x[n].transpose(1, 2)[kept], before[n].transpose(1, 2)[kept])
        # the bits of the norm operator
        want, _ = msa.m3_qk_norm_rope(x["k"], None, x["wk"], None, x["rope"], x["cu"], eps=1e-5,
                                      context_lens=x["context"])
        assert torch.equal(x["kc"][p, :, slot], want[t])
        return
    for n, rows in (("k", keys), ("v", values)):
        held, scale = _append_fp8(before[n + "c"], old_scale[n + "s"], rows, x["table"], lengths, context)
        assert np.array_equal(x[n + "s"].double().cpu().numpy(), scale), n
        got = x[n + "c"].float().double().cpu().numpy()
        assert np.array_equal(got, held), (n, int((got != held).sum()))


@pytest.mark.gpu
def test_token_by_token_scales_grow(device):
    """One token at a time into pages that start empty; magnitudes that double force the held tokens to be rounded again."""
    lengths, heads, dim, page = [37], 2, 64, 16
    x = _setup(lengths, [0], heads, dim, 16, 0, page, torch.bfloat16, True, device)
    size = 2.0 ** (torch.arange(37) % 13 - 20).float()
    x["v"] = (x["v"].float() * size.to(device)[:, None, None]).bfloat16()
    x["v"][5], x["v"][20] = 0, 1e-38
    table = x["table"]
    cu = cu_tensor([1], device)
    cache, scale = x["vc"].clone(), x["vs"].clone()
    held, scales = cache, scale.double().cpu().numpy()
    want_c, want_s = x["vc"].clone(), x["vs"].clone()
    for i in range(37):
        ctx = torch.tensor([i], dtype=torch.int32, device=device)
        msa.m3_cache_append(x["k"][i:i + 1], x["v"][i:i + 1], x["kc"], cache, table.to(device), cu, ctx,
                            k_scale=x["ks"], v_scale=scale)
        held, scales = _append_fp8(want_c, want_s, x["v"][i:i + 1].double().cpu().numpy(), table, [1], [i])
        want_c, want_s = torch.from_numpy(held).float().to(FP8), torch.from_numpy(scales)
        assert np.array_equal(scale.double().cpu().numpy(), scales), i
        assert np.array_equal(cache.float().double().cpu().numpy(), held), i
    # twice the same call changes nothing
    again_c, again_s = cache.clone(), scale.clone()
    msa.m3_cache_append(x["k"][36:], x["v"][36:], x["kc"], cache, table.to(device), cu,
                        torch.tensor([36], dtype=torch.int32, device=device), k_scale=x["ks"], v_scale=scale)
    assert torch.equal(again_c.view(torch.uint8), cache.view(torch.uint8)) and torch.equal(again_s, scale)


@pytest.mark.gpu
def test_not_finite_and_largest_values(device):
    x = _setup([4], [0], 1, 16, 16, 0, 16, torch.bfloat16, True, device)
    x["v"][0, 0, :4] = torch.tensor([float("inf"), -float("inf"), float("nan"), 448.0], device=device)
    x["v"][1:] = 0.25
    _call(x, wk=None, wi=None)
    p = int(x["table"][0, 0])
    got = x["vc"][p, 0, :4].float() * x["vs"][p, 0]
    assert x["vs"][p, 0] == 1.0 and torch.isnan(got[0, :3]).all() and got[0, 3] == 448
    assert (got[1:] == 0.25).all()
    x = _setup([2], [0], 1, 16, 16, 0, 16, torch.bfloat16, True, device)
    x["v"][:] = torch.finfo(torch.bfloat16).max
    x["v"][1] = 0
    x["k"][:] = 0
    _call(x, wk=None, wi=None)
    p = int(x["table"][0, 0])
    assert x["ks"][p, 0] == 0 and (x["kc"][p, 0, :2].float() == 0).all()
    assert x["vs"][p, 0] == scale_for(float(torch.finfo(torch.bfloat16).max)) and torch.isfinite(x["vc"][p, 0, :2].float()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("normed", [False, True])
def test_keys_at_scale_borders_and_out_of_range(dtype, normed, device):
    """Rotated keys whose largest value is 448 x 2^k to the last bit, or next to it; rows that are zero, huge, tiny, infinite
    or NaN beside ordinary ones; a rotation that is none."""
    page, heads, dim = 16, 5, 32
    x = _setup([page], [0], heads, dim, 16, 0, page, dtype, True, device)
    x["wk"] = torch.ones(dim, dtype=dtype, device=device) if normed else None
    x["wi"] = x["ik"] = x["ic"] = None
    gen = torch.Generator().manual_seed(5)
    x["k"] = torch.randn(page, heads, dim, generator=gen).to(dtype).to(device)
    step = 1 + torch.finfo(dtype).eps
    x["k"][3, 0, 7] = 448.0 / 64
    x["k"][3, 1, 20] = -448.0 / 64 * step
    x["k"][2, 2], x["k"][5, 2] = 0, 1e-7
    big = 60000.0 if dtype == torch.float16 else 3e38
    x["k"][4, 3] = big
    x["k"][6, 4, 0], x["k"][7, 4, 1], x["k"][8, 4, 2] = float("inf"), float("nan"), -float("inf")
    for turn in ("none", "scaled", "real"):
        if turn == "none":
            rope = torch.cat([torch.ones(page, 8), torch.zeros(page, 8)], 1)
        elif turn == "scaled":
            rope = torch.randn(page, 16, generator=gen) * 5
        else:
            rope = msa.rope_table(page - 1, 16)  # and no row for the last position
        x["rope"] = rope.to(device)
        x["kc"].view(torch.uint8).fill_(0)
        x["ks"].fill_(0.25)
        _call(x)
        rows = _turned(x["k"], x["wk"], x["rope"], list(range(page)), 1e-5)
        with np.errstate(invalid="ignore", over="ignore"):
            held, scale = _append_fp8(torch.zeros_like(x["kc"], device="cpu"), torch.full_like(x["ks"], 0.25, device="cpu"),
                                      rows, x["table"], [page], [0])
        p = int(x["table"][0, 0])
        assert np.array_equal(x["ks"].double().cpu().numpy(), scale), turn
        assert np.array_equal(x["kc"][p].float().double().cpu().numpy(), held[p], equal_nan=True), turn


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_missing_pages_strided_caches_and_views(fp8, device):
    lengths, context = [40, 9], [3, 14]
    x = _setup(lengths, context, 2, 64, 32, 32, 16, torch.bfloat16, fp8, device)
    x["table"][0, 1] = 10_000  # outside the cache
    x["table"] = x["table"][:, :2].clone()  # and too narrow for the longest sequence
    y = {n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in x.items()}
    both = torch.empty((y["kc"].shape[0], 2, *y["kc"].shape[1:]), dtype=y["kc"].dtype, device=device)
    both[:, 0], both[:, 1] = y["kc"], y["vc"]
    total = sum(lengths)
    fused = torch.cat([y["k"], y["v"]], 1).view(total, 2, 2, 64)
    before = x["kc"].clone()
    _call(x)
    _call(y, kc=both[:, 0], vc=both[:, 1], k=fused[:, 0], v=fused[:, 1], cu=msa.prepare_sequences(y["cu"]))
    for a, b in ((x["kc"], both[:, 0]), (x["vc"], both[:, 1])):
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
    # only the pages that exist were touched
    live = torch.tensor(sorted({int(p) for p in x["table"].flatten() if 0 <= p < x["kc"].shape[0]}))
    rest = torch.ones(x["kc"].shape[0], dtype=torch.bool)
    rest[live] = False
    rest = rest.to(device)
    assert torch.equal(before[rest].view(torch.uint8), x["kc"][rest].view(torch.uint8))
    assert not torch.equal(before.view(torch.uint8), x["kc"].view(torch.uint8))


@pytest.mark.gpu
def test_offsets_past_32_bits(device):
    """Pages beyond 2^32 bytes of a cache."""
    heads, dim, page, count = 8, 256, 256, 4200  # 4.4 GB in 8 bits
    kc = torch.zeros(count, heads, page, dim, dtype=FP8, device=device)
    ks, vs = (torch.zeros(count, heads, device=device) for _ in range(2))
    k = torch.randn(3, heads, dim, device=device).bfloat16()
    table = torch.tensor([[count - 1]], dtype=torch.int32, device=device)
    msa.m3_cache_append(k, k, kc, kc.clone(), table, cu_tensor([3], device),
                        torch.tensor([253], dtype=torch.int32, device=device), k_scale=ks, v_scale=vs)
    scale = 2.0 ** np.ceil(np.log2(k.float().abs().amax((0, 2)).double().cpu().numpy() / 448))
    # slots before the new ones were empty pages' zeros: the old scale was 0
    assert np.array_equal(ks[-1].double().cpu().numpy(), scale)
    want = round_e4m3(k.double().cpu().numpy() / scale[None, :, None])
    got = kc[-1, :, 253:].float().double().cpu().numpy().transpose(1, 0, 2)
    assert np.array_equal(got, want) and (kc[:-1].view(torch.uint8).flatten()[::4097] == 0).all()


@pytest.mark.gpu
def test_graph_replay_with_new_lengths(device):
    """A captured step writes where the lengths and tables point when it is replayed."""
    x = _setup([1, 1, 1], [4, 30, -1], 2, 64, 64, 64, 16, torch.bfloat16, True, device)
    x["cu"] = msa.prepare_sequences(x["cu"])
    x["rope"] = msa.rope_table(64, 64, device=device)
    table = x["table"].to(device)
    x["table"] = table
    graph = torch.cuda.CUDAGraph()
    y = {n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in x.items()}
    _call(x)
    x = {n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in y.items()}
    with torch.cuda.graph(graph):
        _call(x)
    for step in range(3):
        graph.replay()
        torch.cuda.synchronize()
        _call(y)
        for n in ("kc", "vc", "ic", "ks", "vs"):
            assert torch.equal(x[n].view(torch.uint8), y[n].view(torch.uint8)), (step, n)
        for z in (x, y):
            z["context"].copy_(torch.tensor([5 + step, 31, -1 - step], dtype=torch.int32))
            z["k"].copy_(torch.randn(z["k"].shape, generator=torch.Generator().manual_seed(step)))


def test_refusals():
    k = torch.ones(3, 2, 32, dtype=torch.bfloat16)
    cache = torch.zeros(5, 2, 16, 32, dtype=torch.bfloat16)
    cu, ctx = torch.tensor([0, 3], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    table = torch.zeros(1, 2, dtype=torch.int32)
    call = msa.m3_cache_append
    with pytest.raises(ValueError, match="one shape"):
        call(k, k[:, :1], cache, cache, table, cu, ctx)
    with pytest.raises(NotImplementedError, match="BF16 or FP16"):
        call(k.float(), k.float(), cache, cache, table, cu, ctx)
    with pytest.raises(TypeError, match="BF16 or FP16"):
        call(k.double(), k.double(), cache, cache, table, cu, ctx)
    with pytest.raises(ValueError, match="k_cache must be"):
        call(k, k, cache[:, :1], cache, table, cu, ctx)
    with pytest.raises(TypeError, match="v_cache"):
        call(k, k, cache, cache.half(), table, cu, ctx)
    with pytest.raises(ValueError, match="power of two"):
        call(k, k, cache[:, :, :12], cache[:, :, :12], table, cu, ctx)
    with pytest.raises(ValueError, match="16-byte"):
        bad = torch.zeros(5 * 2 * 16 * 32 + 1, dtype=torch.bfloat16)[1:].view(5, 2, 16, 32)
        call(k, k, bad, cache, table, cu, ctx)
    with pytest.raises(ValueError, match="one shape"):
        call(k, k, cache, cache[:4], table, cu, ctx)
    with pytest.raises(ValueError, match="8-bit cache"):
        call(k, k, cache, cache, table, cu, ctx, k_scale=torch.ones(5, 2))
    with pytest.raises(ValueError, match="k_scale must be"):
        call(k, k, cache.to(FP8), cache.to(FP8), table, cu, ctx)
    with pytest.raises(ValueError, match="go together"):
        call(k, k, cache, cache, table, cu, ctx, index_k=k[:, :1])
    with pytest.raises(ValueError, match="index_k"):
        call(k, k, cache, cache, table, cu, ctx, index_k=k, index_cache=cache)
    with pytest.raises(ValueError, match="pages of k_cache"):
        call(k, k, cache, cache, table, cu, ctx, index_k=k[:, :1], index_cache=cache[:4, :1])
    with pytest.raises(ValueError, match="without index_k"):
        call(k, k, cache, cache, table, cu, ctx, index_weight=k[0, 0])
    with pytest.raises(ValueError, match="k_weight"):
        call(k, k, cache, cache, table, cu, ctx, k_weight=torch.ones(8))
    with pytest.raises(ValueError, match="rotary_dim"):
        call(k, k, cache, cache, table, cu, ctx, cos_sin=msa.rope_table(4, 64))
    with pytest.raises(ValueError, match="eps"):
        call(k, k, cache, cache, table, cu, ctx, eps=-1.0)
    with pytest.raises(TypeError, match="page_table"):
        call(k, k, cache, cache, table.long(), cu, ctx)
    with pytest.raises(ValueError, match="page_table"):
        call(k, k, cache, cache, table[0], cu, ctx)
    with pytest.raises(ValueError, match="int32 metadata"):
        call(k, k, cache, cache, torch.zeros(1, 1, dtype=torch.int32).expand(1, 2 ** 27), cu, ctx)
    with pytest.raises(TypeError, match="context_lens"):
        call(k, k, cache, cache, table, cu, None)
    with pytest.raises(ValueError, match="end at total_tokens"):
        call(k, k, cache, cache, table, torch.tensor([0, 2], dtype=torch.int32), ctx)
    with pytest.raises(NotImplementedError, match="multiples of 16"):
        call(k[:, :, :24].contiguous(), k[:, :, :24].contiguous(), cache[..., :24], cache[..., :24], table, cu, ctx)
    with pytest.raises(RuntimeError, match="ROCm device"):
        call(k, k, cache, cache, table, cu, ctx)
