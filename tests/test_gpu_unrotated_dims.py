"""Dims past rotary_dim pass unchanged: one that is not finite changes no other. Rotary dims of 32 are read 16 bytes at a
time, 20 value by value; 0 has no rotation at all."""

from __future__ import annotations

import pytest
import torch

import msa_triton_amd as msa
from msa_triton_amd.paged import FP8
from tests.helpers import cu_tensor

D, TOKENS = 64, 5
ODD = (float("inf"), -float("inf"), float("nan"))


def _but(x, dim):
    return torch.cat([x[..., :dim], x[..., dim + 1:]], -1)


def _table(rot, device):
    return msa.rope_table(16, rot, device=device) if rot else None


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16, torch.float32))
@pytest.mark.parametrize("rot", (0, 20, 32))
@pytest.mark.parametrize("dim", (33, 48, 63))
def test_norm_forward(dim, rot, dtype, device):
    gen = torch.Generator().manual_seed(2)
    x, w = torch.randn(TOKENS, 2, D, generator=gen).to(dtype).to(device), torch.ones(D, dtype=dtype, device=device)
    cu = msa.prepare_sequences(cu_tensor([TOKENS], device))
    want, _ = msa.m3_qk_norm_rope(x, None, w, None, _table(rot, device), cu)
    for odd in ODD:
        v = w.clone()
        v[dim] = odd
        got, _ = msa.m3_qk_norm_rope(x, None, v, None, _table(rot, device), cu)
        assert torch.equal(_but(got, dim), _but(want, dim)) and not torch.isfinite(got[..., dim]).any()
    y = x.clone()
    y[2, 1, dim] = float("inf")  # 1 / rms = 0: the row is 0, and 0 x inf there
    got, _ = msa.m3_qk_norm_rope(y, None, w, None, _table(rot, device), cu)
    assert (_but(got[2, 1], dim) == 0).all() and torch.isnan(got[2, 1, dim])
    got[2, 1] = want[2, 1]
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16, torch.float32))
@pytest.mark.parametrize("rot", (0, 20, 32))
@pytest.mark.parametrize("dim", (33, 48, 63))
def test_norm_backward(dim, rot, dtype, device):
    """An incoming gradient: the weight's gradient of that dim alone, and the rows of the inputs' that it belongs to."""
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(TOKENS, 2, D, generator=gen).to(dtype).to(device).requires_grad_()
    w = torch.ones(D, dtype=dtype, device=device).requires_grad_()
    g = torch.randn(TOKENS, 2, D, generator=gen).to(dtype).to(device)
    cu = msa.prepare_sequences(cu_tensor([TOKENS], device))

    def grads(g):
        out, _ = msa.m3_qk_norm_rope(x, None, w, None, _table(rot, device), cu)
        return torch.autograd.grad(out, (x, w), g)

    dx, dw = grads(g)
    for odd in ODD:
        h = g.clone()
        h[3, 0, dim] = odd
        ex, ew = grads(h)
        assert torch.equal(_but(ew, dim), _but(dw, dim)) and not torch.isfinite(ew[dim])
        ex[3, 0] = dx[3, 0]
        assert torch.equal(ex, dx)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", (False, True))
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("rot", (20, 32))
@pytest.mark.parametrize("dim", (33, 48, 63))
def test_append(dim, rot, dtype, fp8, device):
    """Keys that are rotated and not normed: the value that is not finite is stored as such (NaN in 8 bits), the scale and
    all others as if it were 0."""
    gen = torch.Generator().manual_seed(2)
    k, v = (torch.randn(TOKENS, 2, D, generator=gen).to(dtype).to(device) for _ in range(2))
    ik = torch.randn(TOKENS, 1, D, generator=gen).to(dtype).to(device)
    cu = msa.prepare_sequences(cu_tensor([TOKENS], device))
    ctx, pages = torch.tensor([3], dtype=torch.int32, device=device), torch.zeros(1, 1, dtype=torch.int32, device=device)

    def run(odd):
        a, b = k.clone(), ik.clone()
        a[2, 1, dim] = b[4, 0, dim] = odd
        kc, vc = (torch.zeros(1, 2, 16, D, device=device).to(FP8 if fp8 else dtype) for _ in range(2))
        ic = torch.zeros(1, 1, 16, D, dtype=dtype, device=device)
        ks, vs = (torch.full((1, 2), 2.0 ** -20, device=device) if fp8 else None for _ in range(2))
        msa.m3_cache_append(a, v, kc, vc, pages, cu, ctx, index_k=b, index_cache=ic, k_scale=ks, v_scale=vs,
                            cos_sin=_table(rot, device))
        return kc.float(), vc.float(), ic.float(), ks

    want = run(0.0)
    for odd in ODD:
        got = run(odd)
        for x, y, at in ((got[0], want[0], (0, 1, 5, dim)), (got[2], want[2], (0, 0, 7, dim))):
            there = x[at]
            if fp8 and at[1] == 1:
                assert torch.isnan(there)
            else:
                assert torch.isnan(there) if odd != odd else there == odd
            x[at] = y[at]
            assert torch.equal(x, y)
        assert torch.equal(got[1], want[1]) and (got[3] is None or torch.equal(got[3], want[3]))
