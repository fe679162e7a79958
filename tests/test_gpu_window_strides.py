"""Packed window attention on views whose heads lie far apart."""

from __future__ import annotations

import struct

import pytest
import torch

import msa_triton_amd as msa
from msa_triton_amd import _lib
from msa_triton_amd.window_attention import _backward, _forward, aligned_rows
from tests.helpers import cu_tensor

pytestmark = pytest.mark.gpu

FAR = 1 << 26  # elements from one head to the next: 32 of them are 2^31


def far_heads(x):
    """The same values as a view whose heads lie FAR apart."""
    tokens, heads, dim = x.shape
    held = torch.empty(heads * FAR, dtype=x.dtype, device=x.device)
    view = held.as_strided((tokens, heads, dim), (dim, FAR, 1))
    view.copy_(x)
    return view


@pytest.mark.parametrize("q_heads,groups", [(64, 8), (64, 64)])
def test_heads_more_than_2_to_the_31_values_apart(q_heads, groups):
    """Through the C entry points, whose header bounds the heads of one key head: the same bits as contiguous tensors give."""
    tokens, dim, window, sinks, scale = 150, 64, 40, 3, 0.125
    gen = torch.Generator(device="cuda").manual_seed(6)
    q, do = (torch.randn(tokens, q_heads, dim, generator=gen, device="cuda").bfloat16() for _ in range(2))
    k, v = (torch.randn(tokens, groups, dim, generator=gen, device="cuda").bfloat16() for _ in range(2))
    cu = cu_tensor([tokens], "cuda")
    want = _forward(q, k, v, cu, 1, window, sinks, scale, True, True)
    out, lse, lo = want
    want_grads = _backward(q, k, v, cu, 1, tokens, window, sinks, scale, out, lo, lse, do, True, True, True)

    # (keys and values of 8 heads stay below 2^31 whatever their stride)
    far = [far_heads(x) for x in (q, k, v, do)]
    assert max((x.shape[1] - 1) * x.stride(1) for x in far) > 1 << 31
    strides = [s for x in far for s in x.stride()[:2]]
    code, lib, stream = _lib.DTYPE_CODE[q.dtype], _lib.lib(), _lib.stream_of(q.device)
    got = [torch.full_like(x, float("nan")) for x in (out, lo, lse)]
    qp, kp, vp, gp = (x.data_ptr() for x in far)
    status = lib.msa_window_attn_fwd(qp, kp, vp, code, struct.pack("6q", *strides[:6]), cu.data_ptr(), 1, tokens, q_heads, groups, dim,
                                     window, sinks, scale, got[0].data_ptr(), got[1].data_ptr(), got[2].data_ptr(), stream)
    assert status == 0
    assert all(torch.equal(a, b) for a, b in zip(got, (out, lo, lse)))

    size = lib.msa_window_attn_bwd_workspace_bytes(code, tokens, 1, tokens, q_heads, groups, dim, window, sinks)
    workspace = torch.empty(size, dtype=torch.uint8, device="cuda")
    grads = [torch.full_like(x, float("nan")) for x in want_grads]
    status = lib.msa_window_attn_bwd(qp, kp, vp, code, struct.pack("8q", *strides), cu.data_ptr(), 1, tokens, tokens, q_heads, groups, dim,
                                     window, sinks, scale, out.data_ptr(), lo.data_ptr(), lse.data_ptr(), gp,
                                     *(x.data_ptr() for x in grads), workspace.data_ptr(), size, stream)
    assert status == 0
    assert all(torch.equal(a, b) for a, b in zip(grads, want_grads))


@pytest.mark.parametrize("q_heads,groups,far", [(64, 4, "kv"), (64, 8, "qkv"), (40, 40, "qkv"), (64, 2, "qkv")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_heads_in_front_through_the_operator(q_heads, groups, far, dtype):
    """Keys and values of far heads are read in place whatever the heads that share them; queries where a key head's lie near
    enough, and copied otherwise (64 over 2)."""
    tokens, dim, ratio = 90, 64, q_heads // groups
    gen = torch.Generator(device="cuda").manual_seed(9)
    q, do = (torch.randn(tokens, q_heads, dim, generator=gen, device="cuda").to(dtype) for _ in range(2))
    k, v = (torch.randn(tokens, groups, dim, generator=gen, device="cuda").to(dtype) for _ in range(2))
    cu = cu_tensor([tokens], "cuda")

    def run(*leaves, grad):
        leaves = [x.detach().requires_grad_() for x in leaves]
        out, lse = msa.m3_window_attention(*leaves, cu, tokens, window_size=30, sink_tokens=2, return_lse=True)
        return out.detach(), lse, *torch.autograd.grad(out, leaves, grad)

    want = run(q, k, v, grad=do)
    k, v = far_heads(k), far_heads(v)
    assert aligned_rows(k)[0] is k and aligned_rows(v)[0] is v
    if "q" in far:
        q, do = far_heads(q), far_heads(do)
        assert (aligned_rows(q, ratio)[0] is q) == (ratio < 16)
    assert all(torch.equal(a, b) for a, b in zip(run(q, k, v, grad=do), want))
