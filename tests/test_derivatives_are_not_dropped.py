"""No operator returns outputs whose derivative was asked for and silently left out. On the CPU, with C calls that do
nothing: what is tested is the path that a call takes."""

from __future__ import annotations

import contextlib

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import msa_triton_amd as msa
from msa_triton_amd import _lib, custom_ops


class _Calls:
    """Every C entry point: workspaces of 0 bytes, status 0."""

    def __getattr__(self, name):
        return lambda *args: 0


@pytest.fixture
def no_kernels(monkeypatch):
    monkeypatch.setattr(_lib, "lib", _Calls)
    monkeypatch.setattr(_lib, "require_gpu", lambda tensor, what: None)
    monkeypatch.setattr(_lib, "stream_of", lambda device: 0)
    monkeypatch.setattr(_lib, "on_device", lambda device: contextlib.nullcontext())


def _norm_inputs():
    x = [torch.randn(3, 4, 16), torch.randn(3, 2, 16), torch.ones(16), torch.ones(16)]
    return x, (msa.rope_table(8, 16), torch.tensor([0, 3], dtype=torch.int32))


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("grad", (False, True))
@pytest.mark.parametrize("ops", (msa, custom_ops), ids=("eager", "library"))
def test_norm_in_forward_mode(ops, which, grad, no_kernels):
    x, rest = _norm_inputs()
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        ops.m3_qk_norm_rope(*x, *rest)  # (no tangent: as outside)
        x[which] = forward_ad.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(NotImplementedError, match="jvp"):
            ops.m3_qk_norm_rope(*x, *rest)


@pytest.mark.parametrize("name,which", [("score", 0), ("score", 1), ("attention", 0), ("attention", 1), ("attention", 2),
                                        ("kl", 0), ("kl", 1)])
def test_library_ops_in_forward_mode(name, which, no_kernels):
    """The registered operators would run below autograd and leave the tangent out."""
    cu, ids = torch.tensor([0, 3], dtype=torch.int32), torch.zeros(3, 2, 1, dtype=torch.int32)
    q, k = torch.randn(3, 4, 16), torch.randn(3, 2, 16)
    x = [q[:, :2], k[:, :1]] if name != "attention" else [q, k, k.clone()]
    call = dict(score=lambda a, b: custom_ops.m3_index_score(a, b, cu, 3),
                attention=lambda a, b, c: custom_ops.m3_sparse_attention(a, b, c, ids, cu, 3),
                kl=lambda a, b: custom_ops.m3_indexer_kl(a, b, q, k, ids, cu, 3))[name]
    with forward_ad.dual_level(), torch.no_grad():
        x[which] = forward_ad.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(NotImplementedError, match="jvp"):
            call(*x)


def _paged(name, ops):
    """(tensors that may be differentiated, a call of them) of a paged operator."""
    cu, ctx = torch.tensor([0, 3], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    table, ids = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(3, 2, 1, dtype=torch.int32)
    kc, vc, ic = (torch.zeros(2, h, 16, 16, dtype=torch.bfloat16) for h in (2, 2, 1))
    q, k, v, ik = (torch.ones(3, h, 16, dtype=torch.bfloat16) for h in (4, 2, 2, 1))
    w = torch.ones(16, dtype=torch.bfloat16)
    if name == "append":
        return [k, v, ik, w, w.clone(), kc], lambda k, v, ik, wk, wi, kc: ops.m3_cache_append(
            k, v, kc, vc, table, cu, ctx, index_k=ik, index_cache=ic, k_weight=wk, index_weight=wi)
    if name == "score":
        return [q[:, :2].clone(), ic], lambda iq, ic: ops.m3_index_score_topk_paged(iq, ic, table, cu, ctx, 16, topk_blocks=1)
    return [q, kc, vc], lambda q, kc, vc: ops.m3_sparse_attention_paged(q, kc, vc, ids, table, cu, ctx, return_lse=True)


PAGED = [(name, i) for name, n in (("append", 6), ("score", 2), ("attention", 3)) for i in range(n)]


@pytest.mark.parametrize("name,which", PAGED)
@pytest.mark.parametrize("ops", (msa, custom_ops), ids=("eager", "library"))
def test_paged_operators_and_gradients(ops, name, which, no_kernels):
    x, call = _paged(name, ops)
    plain = call(*x)
    assert name == "append" or not any(y.requires_grad for y in plain)
    x[which].requires_grad_()
    with torch.no_grad():
        call(*x)
    if name == "append":
        with pytest.raises(RuntimeError, match="no gradients"):
            call(*x)
        call(*(y.detach() for y in x))
        return
    outs = call(*x)
    assert outs[0].requires_grad and [y.shape for y in outs] == [y.shape for y in plain]
    with pytest.raises(RuntimeError, match="no gradients|no autograd formula"):
        outs[0].float().sum().backward()


@pytest.mark.parametrize("name,which", PAGED)
@pytest.mark.parametrize("ops", (msa, custom_ops), ids=("eager", "library"))
def test_paged_operators_in_forward_mode(ops, name, which, no_kernels):
    x, call = _paged(name, ops)
    with forward_ad.dual_level(), torch.no_grad():
        call(*x)
        x[which] = forward_ad.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(NotImplementedError, match="jvp"):
            call(*x)


@pytest.mark.parametrize("ops", (msa, custom_ops), ids=("eager", "library"))
def test_a_backward_pass_notices_an_append(ops, no_kernels):
    """Caches and scales that a graph has saved and an append then wrote."""
    cu, ctx = torch.tensor([0, 1], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    table = torch.zeros(1, 2, dtype=torch.int32)
    k, ik = torch.ones(1, 2, 16, dtype=torch.bfloat16), torch.ones(1, 1, 16, dtype=torch.bfloat16)
    kc, vc = (torch.zeros(2, 2, 16, 16, dtype=torch.bfloat16).to(torch.float8_e4m3fn) for _ in range(2))
    ic, ks, vs = torch.zeros(2, 1, 16, 16, dtype=torch.bfloat16), torch.ones(2, 2), torch.ones(2, 2)
    q = torch.ones(16, dtype=torch.bfloat16, requires_grad=True)
    uses = [(q * ic).sum(), (q[:2] * ks).sum(), (q[:2] * vs).sum()]
    before = [x._version for x in (kc, vc)]
    ops.m3_cache_append(k, k, kc, vc, table, cu, ctx, index_k=ik, index_cache=ic, k_scale=ks, v_scale=vs)
    for y in uses:
        with pytest.raises(RuntimeError, match="inplace operation"):
            y.backward()
    assert all(x._version > b for x, b in zip((kc, vc), before))
    with torch.inference_mode():
        ops.m3_cache_append(k, k, kc.clone(), vc.clone(), table, cu, ctx, index_k=ik, index_cache=ic.clone(), k_scale=ks.clone(),
                            v_scale=vs.clone())
