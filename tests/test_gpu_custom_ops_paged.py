"""torch.library registration of the norm and the paged operators: ``opcheck`` of each op, a compiled training
layer with the norm and a compiled decoding step, both bit for bit the eager operators'."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import msa_triton_amd as msa
from msa_triton_amd import custom_ops as C
from msa_triton_amd.paged import FP8
from tests.helpers import cu_tensor
from tests.paged_helpers import page_table

NAMES = ("qk_norm_rope", "qk_norm_rope_backward", "cache_append", "index_score_topk_paged", "sparse_attention_paged")


def test_registered_with_fake_kernels():
    ops = torch.ops.msa_mi355x
    assert all(hasattr(ops, n) for n in NAMES)
    with FakeTensorMode():
        def t(*shape, dtype=torch.bfloat16):
            return torch.empty(*shape, dtype=dtype, device="cuda")

        cu, ctx, pages = t(3, dtype=torch.int32), t(2, dtype=torch.int32), t(2, 5, dtype=torch.int32)
        q, k, w, rope = t(7, 6, 32), t(7, 2, 32), t(32), t(100, 16, dtype=torch.float32)
        a, b = ops.qk_norm_rope(q, k, w, w, rope, cu, None, 1e-6)
        assert a.shape == q.shape and b.shape == k.shape and a.dtype == q.dtype
        assert ops.qk_norm_rope(q, None, w, None, None, cu, ctx, 1e-6)[1].shape == (0,)
        g = ops.qk_norm_rope_backward(q, k, w, w, rope, cu, None, 1e-6, a, b, True, False, True, False)
        assert [tuple(x.shape) for x in g] == [(7, 6, 32), (0,), (32,), (0,)]
        kc, ks, ic = t(9, 2, 16, 32, dtype=FP8), t(9, 2, dtype=torch.float32), t(9, 1, 16, 64)
        assert ops.cache_append(k, k, kc, kc, pages, cu, ctx, t(7, 1, 64), ic, ks, ks, w, t(64), rope, 1e-6) is None
        s, i = ops.index_score_topk_paged(t(7, 2, 64), ic, pages, cu, ctx, 70, 32, 1.0, 4, 1)
        assert s.shape == (7, 2, 3) and s.dtype == torch.float32 and i.shape == (7, 2, 4) and i.dtype == torch.int32
        o, lse = ops.sparse_attention_paged(q, kc, kc, i, pages, cu, ctx, 32, 0.1, ks, ks)
        assert o.shape == q.shape and lse.shape == (7, 6) and lse.dtype == torch.float32


def _inputs(device, fp8=True, seed=4):
    gen = torch.Generator().manual_seed(seed)
    lengths, context, groups, ratio, dim, page = [3, 0, 2], [40, 5, 70], 2, 2, 32, 16
    table, count = page_table([n + c for n, c in zip(lengths, context)], page, gen)

    def rand(*shape):
        return torch.randn(*shape, generator=gen).bfloat16().to(device)

    total = sum(lengths)
    kind = FP8 if fp8 else torch.bfloat16
    scale = torch.full((count, groups), 2.0 ** -6, device=device) if fp8 else None
    x = dict(q=rand(total, groups * ratio, dim), k=rand(total, groups, dim), v=rand(total, groups, dim),
             iq=rand(total, groups, dim), ik=rand(total, 1, dim), w=rand(dim).abs() + 0.5,
             kc=(rand(count, groups, page, dim) * (40 if fp8 else 1)).to(kind),
             vc=(rand(count, groups, page, dim) * (40 if fp8 else 1)).to(kind), ic=rand(count, 1, page, dim), ks=scale,
             vs=None if scale is None else scale.clone(), table=table.to(device), cu=cu_tensor(lengths, device),
             ctx=torch.tensor(context, dtype=torch.int32, device=device), rope=msa.rope_table(128, 16, device=device))
    return x


@pytest.mark.gpu
def test_opcheck_each_op(device):
    x = _inputs(device, fp8=False)  # opcheck compares with arithmetic that torch has not for 8-bit types
    q, k, wq, wk = (x[n].clone().requires_grad_() for n in ("q", "k", "w", "w"))
    ops = torch.ops.msa_mi355x
    torch.library.opcheck(ops.qk_norm_rope.default, (q, k, wq, wk, x["rope"], x["cu"], x["ctx"], 1e-6))
    torch.library.opcheck(ops.cache_append.default,
                          (x["k"], x["v"], x["kc"], x["vc"], x["table"], x["cu"], x["ctx"], x["ik"], x["ic"], None, None, x["w"],
                           x["w"], x["rope"], 1e-6))
    torch.library.opcheck(ops.index_score_topk_paged.default,
                          (x["iq"], x["ic"], x["table"], x["cu"], x["ctx"], 80, 16, 1.0, 3, 1))
    _, ids = msa.m3_index_score_topk_paged(x["iq"], x["ic"], x["table"], x["cu"], x["ctx"], 80, block_size=16, topk_blocks=3)
    torch.library.opcheck(ops.sparse_attention_paged.default,
                          (x["q"], x["kc"], x["vc"], ids, x["table"], x["cu"], x["ctx"], 16, 0.2, x["ks"], x["vs"]))


@pytest.mark.gpu
def test_compiled_layer_with_the_norm(device):
    lengths, block = [150, 0, 90], 32
    gen = torch.Generator().manual_seed(8)
    cu = cu_tensor(lengths, device)
    total = sum(lengths)
    q, k, v = (torch.randn(total, h, 64, generator=gen).bfloat16().to(device) for h in (4, 2, 2))
    w = (1 + 0.1 * torch.randn(64, generator=gen)).bfloat16().to(device)
    g = torch.randn(total, 4, 64, generator=gen).bfloat16().to(device)
    rope = msa.rope_table(max(lengths), 32, device=device)

    def layer(ops, q, k, v, wq, wk):
        a, b = ops.m3_qk_norm_rope(q, k, wq, wk, rope, cu)
        scores = ops.m3_index_score(b[:, :2], b[:, :1], cu, max(lengths), block_size=block)
        ids = ops.m3_topk(scores.detach(), cu, block_size=block, topk_blocks=3, local_blocks=1)
        return ops.m3_sparse_attention(a, b, v, ids, cu, max(lengths), block_size=block)

    def run(fn):
        leaves = [x.clone().requires_grad_() for x in (q, k, v, w, w)]
        out = fn(*leaves)
        (out.float() * g.float()).sum().backward()
        return [out.detach(), *(x.grad for x in leaves)]

    eager = run(lambda *a: layer(msa, *a))
    compiled = run(torch.compile(lambda *a: layer(C, *a), backend="aot_eager", fullgraph=True))
    assert all(torch.equal(a, b) for a, b in zip(eager, compiled))


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_compiled_decoding_step(fp8, device):
    def step(ops, x, kc, vc, ic, ks, vs):
        ops.m3_cache_append(x["k"], x["v"], kc, vc, x["table"], x["cu"], x["ctx"], index_k=x["ik"], index_cache=ic,
                            k_scale=ks, v_scale=vs, k_weight=x["w"], index_weight=x["w"], cos_sin=x["rope"])
        a, _ = ops.m3_qk_norm_rope(x["q"], None, x["w"], None, x["rope"], x["cu"], context_lens=x["ctx"])
        s, ids = ops.m3_index_score_topk_paged(x["iq"], ic, x["table"], x["cu"], x["ctx"], 80, block_size=16, topk_blocks=3)
        return s, ids, ops.m3_sparse_attention_paged(a, kc, vc, ids, x["table"], x["cu"], x["ctx"], block_size=16,
                                                     k_scale=ks, v_scale=vs)

    x, y = _inputs(device, fp8), _inputs(device, fp8)
    names = ("kc", "vc", "ic", "ks", "vs")
    want = step(msa, x, *(x[n] for n in names))
    with torch.no_grad():
        got = torch.compile(lambda *a: step(C, y, *a), backend="aot_eager", fullgraph=True)(*(y[n] for n in names))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    for n in names:
        assert x[n] is None or torch.equal(x[n].view(torch.uint8), y[n].view(torch.uint8)), n
