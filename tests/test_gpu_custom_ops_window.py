"""torch.library registration of the window and tree operators: fake kernels, ``opcheck``, and a compiled layer and serving step
bit for bit the eager operators'."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import msa_triton_amd as msa
from msa_triton_amd import custom_ops as C
from msa_triton_amd.paged import FP8
from tests.helpers import cu_tensor


def test_registered_with_fake_kernels():
    ops = torch.ops.msa_mi355x
    with FakeTensorMode():
        def t(*shape, dtype=torch.bfloat16):
            return torch.empty(*shape, dtype=dtype, device="cuda")

        cu, ctx, pages = t(3, dtype=torch.int32), t(2, dtype=torch.int32), t(2, 5, dtype=torch.int32)
        q, k = t(7, 6, 32), t(7, 2, 32)
        out, lse, lo = ops.window_attention(q, k, k, cu, 7, 3, 1, 0.2, True)
        assert out.shape == lo.shape == q.shape and lse.shape == (7, 6) and lse.dtype == torch.float32
        assert ops.window_attention(q, k, k, cu, 7, None, 0, 0.2, False)[2].shape == (0,)
        assert ops.window_attention(q.float(), k.float(), k.float(), cu, 7, None, 0, 0.2, True)[2].shape == (0,)
        g = ops.window_attention_backward(q, k, k, cu, 7, 3, 1, 0.2, out, lo, lse, out, True, False, True)
        assert [tuple(x.shape) for x in g] == [(7, 6, 32), (0,), (7, 2, 32)]
        kc, ks = t(9, 2, 16, 32, dtype=FP8), t(9, 2, dtype=torch.float32)
        for parents in (None, t(7, dtype=torch.int32)):
            o, s = ops.window_attention_paged(q, kc, kc, pages, cu, ctx, parents, 4, 0, 0.2, ks, ks)
            assert o.shape == q.shape and o.dtype == q.dtype and s.shape == (7, 6)


def _packed(dtype):
    gen = torch.Generator().manual_seed(9)
    return [torch.randn(50, h, 64, generator=gen).to(dtype).cuda() for h in (4, 2, 2)], cu_tensor([20, 30], "cuda")


def _cache(fp8):
    gen = torch.Generator().manual_seed(10)
    q = torch.randn(5, 4, 32, generator=gen).bfloat16().cuda()
    c = [torch.randn(8, 2, 16, 32, generator=gen).cuda().to(FP8 if fp8 else torch.bfloat16) for _ in range(2)]
    scale = torch.full((8, 2), 0.5, device="cuda") if fp8 else None
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    return (q, *c, table, cu_tensor([3, 2], "cuda"), torch.tensor([20, 5], dtype=torch.int32, device="cuda")), dict(k_scale=scale,
                                                                                                                   v_scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_opcheck_and_gradients(dtype):
    x, cu = _packed(dtype)
    leaves = [y.requires_grad_() for y in x]
    torch.library.opcheck(torch.ops.msa_mi355x.window_attention, (*leaves, cu, 30, 9, 2, 0.125, True))
    out, lse = C.m3_window_attention(*leaves, cu, 30, window_size=9, sink_tokens=2, return_lse=True)
    want, want_lse = msa.m3_window_attention(*leaves, cu, 30, window_size=9, sink_tokens=2, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse) and not lse.requires_grad
    do = torch.randn_like(out)
    a, b = torch.autograd.grad(out, leaves, do), torch.autograd.grad(want, leaves, do)
    assert all(torch.equal(u, w) for u, w in zip(a, b))
    with pytest.raises(ValueError, match="max_seqlen"):
        C.m3_window_attention(*leaves, cu, 29, window_size=9)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_opcheck_of_the_paged_op(fp8):
    x, scales = _cache(fp8)
    parents = torch.tensor([-1, 0, 0, -1, 0], dtype=torch.int32, device="cuda")
    for p in (None, parents) if not fp8 else ():  # (opcheck multiplies its inputs: no 8-bit ones)
        torch.library.opcheck(torch.ops.msa_mi355x.window_attention_paged, (*x, p, 9, 2, 0.2, scales["k_scale"], scales["v_scale"]))
    a = C.m3_window_attention_paged(*x, window_size=9, sink_tokens=2, return_lse=True, **scales)
    b = msa.m3_window_attention_paged(*x, window_size=9, sink_tokens=2, return_lse=True, **scales)
    c = C.m3_tree_attention_paged(*x, parents, return_lse=True, **scales)
    d = msa.m3_tree_attention_paged(*x, parents, return_lse=True, **scales)
    assert all(torch.equal(u, w) for u, w in zip((*a, *c), (*b, *d)))


@pytest.mark.gpu
def test_compiled_layer_and_step():
    x, cu = _packed(torch.bfloat16)
    leaves = [y.requires_grad_() for y in x]

    def layer(q, k, v, ops):
        return (ops.m3_window_attention(q * 2, k, v, cu, 30, window_size=9, sink_tokens=2) * 0.5).float().pow(2).sum()

    got = torch.compile(lambda *y: layer(*y, C), backend="aot_eager", fullgraph=True)(*leaves)
    want = layer(*leaves, msa)
    assert torch.equal(got, want)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, leaves), torch.autograd.grad(want, leaves)))
    y, scales = _cache(True)
    with torch.no_grad():
        step = torch.compile(lambda q: C.m3_window_attention_paged(q, *y[1:], window_size=9, **scales), backend="aot_eager",
                             fullgraph=True)
        assert torch.equal(step(y[0]), msa.m3_window_attention_paged(*y, window_size=9, **scales))
