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
