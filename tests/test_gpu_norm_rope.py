"""m3_qk_norm_rope against a float64 formula: outputs, gradients, strides, positions, refusals.

Tolerances: arithmetic is fp32 (2^-24 a step, relative). A row passes a sum of D squares, a square root
and a division, two products and a rotation: 16 steps of 2^-24 cover it with room (the sum's error is a few steps
for D <= 512 in runs of 16 and a tree), in units of the larger of the value and its rotation partner; then
half a step of the output type. A weight's gradient is a sum of N terms in fp32 runs of at most 64 x 32 rows: its
error is below N_run 2^-24 sum |terms|.
"""

from __future__ import annotations

import pytest
import torch
import torch.utils.checkpoint

import msa_triton_amd as msa
from tests.helpers import cu_tensor

DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _positions(lengths, context):
    return torch.cat([torch.arange(c, c + n) for n, c in zip(lengths, context)])


def _reference(x, w, table, pos, eps):
    """float64, differentiable."""
    n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    if table is None:
        return n
    half = table.shape[1] // 2
    rows = torch.full((pos.numel(), table.shape[1]), float("nan"), dtype=torch.float64, device=x.device)
    known = (pos >= 0) & (pos < table.shape[0])
    rows[known] = table.double()[pos[known]]
    cos, sin = rows[:, None, :half], rows[:, None, half:]
    a, b = n[..., :half], n[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, n[..., 2 * half:]], -1)


def _close(got, want, scale=None, steps=16.0, what=""):
    """|got - want| <= half a step of the type of |want| + steps 2^-24 scale."""
    want = want.detach()
    half_step = torch.finfo(got.dtype).eps / 2
    size = want.abs() if scale is None else torch.maximum(want.abs(), scale)
    tiny = torch.finfo(got.dtype).smallest_normal * half_step
    bound = half_step * (1 + 2 ** -8) * want.abs() + steps * 2 ** -24 * size + tiny
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all() and (err <= bound).all(), f"{what}: {float((err / bound).max()):.3f} of the bound"


def _pair_scale(y, rot):
    """The larger magnitude of each element and its rotation partner."""
    y = y.detach().abs()
    if not rot:
        return y
    half = rot // 2
    a, b = y[..., :half], y[..., half:rot]
    m = a + b
    return torch.cat([m, m, y[..., rot:]], -1)


CASES = [  # lengths, context, hq, hkv, D, rot, dtype, weight dtype
    ([1], None, 1, 1, 64, 64, torch.bfloat16, None),
    ([5, 0, 130, 1], None, 4, 2, 128, 64, torch.bfloat16, None),
    ([1] * 33, "far", 8, 1, 128, 128, torch.float16, None),
    ([77, 3], "far", 6, 3, 96, 32, torch.float32, None),
    ([700], None, 32, 4, 128, 64, torch.bfloat16, torch.float32),
    ([19, 40], None, 3, 3, 80, 32, torch.float16, torch.float32),
    ([31], None, 2, 1, 256, 128, torch.bfloat16, None),
    ([9], None, 2, 2, 512, 64, torch.float32, None),
    ([33], None, 2, 1, 50, 20, torch.bfloat16, None),     # no 16-byte runs
    ([17], None, 1, 2, 7, 2, torch.float32, None),        # odd dims
    ([1100, 1029], None, 1, 1, 64, 0, torch.float16, None),  # no rotation
    ([4000], None, 40, 1, 64, 32, torch.bfloat16, None),
]


def _inputs(case, device, seed=3):
    lengths, context, hq, hkv, dim, rot, dtype, wdtype = case
    gen = torch.Generator().manual_seed(seed)
    total = sum(lengths)

    def rand(*shape):
        return torch.randn(*shape, generator=gen)

    q = (rand(total, hq, dim) * (0.2 + 3 * torch.rand(hq, 1, generator=gen))).to(dtype).to(device)
    k = rand(total, hkv, dim).to(dtype).to(device)
    wq, wk = ((1 + 0.3 * rand(dim)).to(wdtype or dtype).to(device) for _ in range(2))
    ctx = None
    if context == "far":
        ctx = [0 if i % 3 else 900_000 + 17 * i for i in range(len(lengths))]
    pos = _positions(lengths, ctx or [0] * len(lengths)).to(device)
    table = msa.rope_table(int(pos.max()) + 1, rot, base=5e6, device=device) if rot else None
    dq, dk = rand(total, hq, dim).to(dtype).to(device), rand(total, hkv, dim).to(dtype).to(device)
    ctx = None if ctx is None else torch.tensor(ctx, dtype=torch.int32, device=device)
    return q, k, wq, wk, table, pos, ctx, dq, dk


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_and_gradients(case, device):
    lengths, rot = case[0], case[5]
    q, k, wq, wk, table, pos, ctx, dq, dk = _inputs(case, device)
    cu = cu_tensor(lengths, device)
    leaves = [x.clone().requires_grad_() for x in (q, k, wq, wk)]
    outs = msa.m3_qk_norm_rope(*leaves, table, cu, eps=1e-5, context_lens=ctx)
    grads = torch.autograd.grad(outs, leaves, (dq, dk))
    for i, (x, w, dy) in enumerate(((q, wq, dq), (k, wk, dk))):
        a, b = x.double().requires_grad_(), w.double().requires_grad_()
        y = _reference(a, b, table, pos, 1e-5)
        _close(outs[i].detach(), y, _pair_scale(y, rot), what=f"out {i}")
        da, db = torch.autograd.grad(y, (a, b), dy.double())
        # dx = r (dm w - n mean(dm w n)): the difference of two terms, so in units of the row's largest r |dm w|
        # (a sum over D of products: 2 more steps a level of its tree, below 32 in all)
        n = a.detach() / torch.sqrt((a.detach() ** 2).mean(-1, keepdim=True) + 1e-5)
        r = 1 / torch.sqrt((a.detach() ** 2).mean(-1, keepdim=True) + 1e-5)
        big = dy.double().abs().amax(-1, keepdim=True) * b.detach().abs().max() * 2
        scale = r * big * (1 + n.abs() * n.abs().amax(-1, keepdim=True))
        _close(grads[i], da, scale.expand_as(da), steps=32, what=f"dx {i}")
        # dw: fp32 runs; the terms' sizes add up to the bound, at most 2048 terms one after the other
        terms = (2 * dy.double().abs().amax(-1, keepdim=True) * n.abs()).sum((0, 1))
        rows = x.shape[0] * x.shape[1]
        _close(grads[2 + i], db, terms, steps=16 + min(rows, 64), what=f"dw {i}")


@pytest.mark.gpu
def test_gradient_against_differences(device):
    case = ([6], None, 2, 1, 32, 16, torch.float32, None)
    q, k, wq, wk, table, pos, ctx, dq, dk = _inputs(case, device)
    cu = cu_tensor(case[0], device)
    leaves = [x.clone().requires_grad_() for x in (q, k, wq, wk)]
    outs = msa.m3_qk_norm_rope(*leaves, table, cu)
    grads = torch.autograd.grad(outs, leaves, (dq, dk))

    def loss(args):
        y = [_reference(a.double(), b.double(), table, pos, 1e-6) for a, b in ((args[0], args[2]), (args[1], args[3]))]
        return float((y[0] * dq.double()).sum() + (y[1] * dk.double()).sum())

    base = [x.double() for x in (q, k, wq, wk)]
    for i, at in ((0, (2, 1, 3)), (0, (5, 0, 20)), (1, (0, 0, 12)), (2, (9,)), (3, (31,))):
        h = 1e-4
        up, down = [x.clone() for x in base], [x.clone() for x in base]
        up[i][at] += h
        down[i][at] -= h
        slope = (loss(up) - loss(down)) / (2 * h)
        # the central difference is off by h^2 / 6 of a third derivative (below 1e3 here), the kernel by fp32 steps
        assert abs(float(grads[i][at]) - slope) <= 1e-5 + 1e-4 * abs(slope)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_one_side(dtype, device):
    gen = torch.Generator().manual_seed(5)
    total, hq, hkv, dim = 45, 6, 2, 64
    fused = torch.randn(total, (hq + 2 * hkv) * dim, generator=gen).to(dtype).to(device)
    q = fused[:, :hq * dim].view(total, hq, dim)
    k = fused[:, hq * dim:(hq + hkv) * dim].view(total, hkv, dim)
    w = (1 + 0.1 * torch.randn(dim, generator=gen)).to(dtype).to(device)
    table = msa.rope_table(64, 32, device=device)
    cu = cu_tensor([20, 25], device)
    want = msa.m3_qk_norm_rope(q.contiguous(), k.contiguous(), w, w, table, cu)
    got = msa.m3_qk_norm_rope(q, k, w, w, table, cu)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one, none = msa.m3_qk_norm_rope(q, None, w, None, table, msa.prepare_sequences(cu))
    assert none is None and torch.equal(one, want[0])
    heads_last = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(msa.m3_qk_norm_rope(heads_last, None, w, None, table, cu)[0], want[0])
    dims_first = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(msa.m3_qk_norm_rope(dims_first, None, w, None, table, cu)[0], want[0])
    # rows off 16-byte boundaries take single elements: the same formula, other sums
    off = torch.empty(total * hq * dim + 1, dtype=dtype, device=device)[1:].view(total, hq, dim).copy_(q)
    y = _reference(q.double(), w.double(), table, _positions([20, 25], [0, 0]).to(device), 1e-6)
    _close(msa.m3_qk_norm_rope(off, None, w, None, table, cu)[0], y, _pair_scale(y, 32))


@pytest.mark.gpu
def test_positions_outside_the_table_are_nan(device):
    q = torch.randn(7, 2, 32, device=device)
    w = torch.ones(32, device=device)
    table = msa.rope_table(10, 16, device=device)
    cu = cu_tensor([3, 2, 2], device)
    ctx = torch.tensor([0, -5, 9], dtype=torch.int32, device=device)
    out, _ = msa.m3_qk_norm_rope(q, None, w, None, table, cu, context_lens=ctx)
    bad = torch.tensor([False, False, False, True, True, False, True], device=device)
    assert torch.isnan(out[bad][..., :16]).all() and torch.isfinite(out[~bad]).all()
    assert torch.isfinite(out[..., 16:]).all()


@pytest.mark.gpu
def test_zero_rows_infinities_and_empty_packs(device):
    x = torch.zeros(4, 1, 64, dtype=torch.bfloat16, device=device)
    x[1] = float("inf")
    x[2, 0, 5] = float("nan")
    x[3] = 1e-20
    w = torch.ones(64, dtype=torch.bfloat16, device=device)
    cu = cu_tensor([4], device)
    leaf = x.clone().requires_grad_()
    out, _ = msa.m3_qk_norm_rope(leaf, None, w, None, None, cu)
    out.backward(torch.ones_like(out))
    assert (out[0] == 0).all() and torch.isnan(out[1]).all() and torch.isnan(out[2, 0, 5])
    assert torch.isfinite(out[3]).all() and torch.isfinite(leaf.grad[[0, 3]]).all()
    e = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=device, requires_grad=True)
    we = w.clone().requires_grad_()
    q0, k0 = msa.m3_qk_norm_rope(e, e, we, w, None, torch.zeros(2, dtype=torch.int32, device=device))
    assert q0.shape == k0.shape == (0, 2, 64)
    (q0.float().sum() + k0.float().sum()).backward()
    assert (we.grad == 0).all()


@pytest.mark.gpu
def test_partial_gradients_and_determinism(device):
    case = ([300, 211], None, 8, 2, 128, 64, torch.bfloat16, None)
    q, k, wq, wk, table, pos, ctx, dq, dk = _inputs(case, device)
    cu = msa.prepare_sequences(cu_tensor(case[0], device))
    leaves = [x.clone().requires_grad_() for x in (q, k, wq, wk)]
    full = torch.autograd.grad(msa.m3_qk_norm_rope(*leaves, table, cu), leaves, (dq, dk))
    again = torch.autograd.grad(msa.m3_qk_norm_rope(*leaves, table, cu), leaves, (dq, dk))
    assert all(torch.equal(a, b) for a, b in zip(full, again))
    for i in range(4):
        args = [x.clone().requires_grad_(j == i) for j, x in enumerate((q, k, wq, wk))]
        outs = msa.m3_qk_norm_rope(*args, table, cu)
        (one,) = torch.autograd.grad(outs[i % 2], args[i], (dq, dk)[i % 2])
        assert torch.equal(one, full[i])
    outs = msa.m3_qk_norm_rope(*leaves, table, cu)
    got = torch.autograd.grad(outs[0], leaves, dq, allow_unused=True)
    assert torch.equal(got[0], full[0]) and torch.equal(got[2], full[2]) and got[1] is None and got[3] is None
    with pytest.raises(RuntimeError, match="once_differentiable"):
        outs = msa.m3_qk_norm_rope(*leaves, table, cu)
        (g,) = torch.autograd.grad(outs[0], leaves[0], dq.clone().requires_grad_(), create_graph=True)
        g.float().sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("way", ("checkpoint", "offload"))
def test_saved_tensors_that_move(way, device):
    """Checkpointing recomputes what the backward reads and offloading copies it: other tensors at other addresses."""
    case = ([300, 211], "far", 8, 2, 128, 64, torch.bfloat16, None)
    q, k, wq, wk, table, pos, ctx, dq, dk = _inputs(case, device)
    cu = msa.prepare_sequences(cu_tensor(case[0], device))
    leaves = [x.clone().requires_grad_() for x in (q, k, wq, wk)]

    def layer(q, k, wq, wk):
        # (weights and inputs that nothing but the saved state keeps; a transposed one comes back in another layout)
        return msa.m3_qk_norm_rope(q * 2, (k * 2).transpose(1, 2).contiguous().transpose(1, 2), wq * 1.5, wk * 1.5, table,
                                   cu, context_lens=ctx)

    want = torch.autograd.grad(layer(*leaves), leaves, (dq, dk))
    if way == "checkpoint":
        outs = torch.utils.checkpoint.checkpoint(layer, *leaves, use_reentrant=False)
    else:
        with torch.autograd.graph.save_on_cpu():
            outs = layer(*leaves)
    noise = [torch.full_like(q, float("nan")) for _ in range(4)]  # takes the place of what was freed
    got = torch.autograd.grad(outs, leaves, (dq, dk))
    del noise
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_graph_replays(device):
    case = ([64, 33], None, 4, 2, 64, 64, torch.bfloat16, None)
    q, k, wq, wk, table, pos, ctx, dq, dk = _inputs(case, device)
    cu = msa.prepare_sequences(cu_tensor(case[0], device))
    leaves = [x.clone().requires_grad_() for x in (q, k, wq, wk)]

    def step():
        outs = msa.m3_qk_norm_rope(*leaves, table, cu)
        return (*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, (dq, dk)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        with torch.no_grad():
            leaves[0].copy_(torch.randn_like(leaves[0]))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_rope_table_and_refusals():
    t = msa.rope_table(1_000_001, 8, base=10000.0)[1_000_000].double()
    angle = 1_000_000.0 * 10000.0 ** (-torch.arange(4, dtype=torch.float64) / 4)
    assert (t - torch.cat([angle.cos(), angle.sin()])).abs().max() <= 2 ** -24
    assert msa.rope_table(0, 2).shape == (0, 2)
    for bad in ((-1, 8), (4, 7), (4, 0)):
        with pytest.raises(ValueError):
            msa.rope_table(*bad)
    q, k, w = torch.ones(3, 4, 16), torch.ones(3, 2, 16), torch.ones(16)
    cu = torch.tensor([0, 3], dtype=torch.int32)
    table = msa.rope_table(8, 16)
    call = msa.m3_qk_norm_rope
    with pytest.raises(ValueError, match="rank-3"):
        call(q[0], k, w, w, table, cu)
    with pytest.raises(ValueError, match="expected q"):
        call(q, k[:2], w, w, table, cu)
    with pytest.raises(TypeError, match="dtype"):
        call(q.double(), k.double(), w, w, table, cu)
    with pytest.raises(ValueError, match="share dtype"):
        call(q, k.bfloat16(), w, w, table, cu)
    with pytest.raises(ValueError, match="q_weight"):
        call(q, k, w[:8], w, table, cu)
    with pytest.raises(ValueError, match="q_weight"):
        call(q, k, w.double(), w, table, cu)
    with pytest.raises(ValueError, match="k_weight"):
        call(q, k, w, None, table, cu)
    with pytest.raises(ValueError, match="k_weight without k"):
        call(q, None, w, w, table, cu)
    with pytest.raises(ValueError, match="share a dtype"):
        call(q.bfloat16(), k.bfloat16(), w, w.bfloat16(), table, cu)
    with pytest.raises(ValueError, match="cos_sin"):
        call(q, k, w, w, table.double(), cu)
    with pytest.raises(ValueError, match="rotary_dim"):
        call(q, k, w, w, msa.rope_table(8, 32), cu)
    with pytest.raises(ValueError, match="eps"):
        call(q, k, w, w, table, cu, eps=float("nan"))
    with pytest.raises(ValueError, match="end at total_tokens"):
        call(q, k, w, w, table, torch.tensor([0, 2], dtype=torch.int32))
    with pytest.raises(TypeError, match="context_lens"):
        call(q, k, w, w, table, cu, context_lens=torch.zeros(1))
    with pytest.raises(ValueError, match="one length per sequence"):
        call(q, k, w, w, table, cu, context_lens=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(NotImplementedError, match="512"):
        call(torch.ones(3, 1, 520), None, torch.ones(520), None, None, cu)
    with pytest.raises(RuntimeError, match="ROCm device"):
        call(q, k, w, w, table, cu)
