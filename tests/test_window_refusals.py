"""What the window operators refuse, on the CPU: arguments are checked before any device work."""

from __future__ import annotations

import pytest
import torch

import msa_triton_amd as msa
from tests.helpers import cu_tensor


def _packed(tokens=6, hq=4, g=2, d=16, dtype=torch.bfloat16):
    return torch.zeros(tokens, hq, d, dtype=dtype), torch.zeros(tokens, g, d, dtype=dtype), torch.zeros(tokens, g, d, dtype=dtype)


def _call(q, k, v, cu=None, most=6, **kw):
    kw.setdefault("window_size", 3)
    return msa.m3_window_attention(q, k, v, cu_tensor([4, 2]) if cu is None else cu, most, **kw)


@pytest.mark.parametrize("kw,error", [
    (dict(window_size=0), ValueError), (dict(window_size=-1), ValueError), (dict(window_size=2.0), ValueError),
    (dict(window_size=True), ValueError), (dict(sink_tokens=-1), ValueError), (dict(sink_tokens=None), ValueError),
    (dict(sink_tokens=1.5), ValueError), (dict(scale=float("inf")), ValueError), (dict(scale=float("nan")), ValueError),
    (dict(most=3), ValueError), (dict(most=0), ValueError), (dict(most=6.0), ValueError),
    (dict(cu=torch.tensor([0, 4, 6])), TypeError), (dict(cu=cu_tensor([4, 3])), ValueError),
    (dict(cu=torch.tensor([0, 5, 4, 6], dtype=torch.int32)), ValueError), (dict(cu=[0, 4, 6]), TypeError),
    (dict(cu=msa.prepare_sequences(cu_tensor([4, 3]))), ValueError),
], ids=str)
def test_arguments(kw, error):
    with pytest.raises(error):
        _call(*_packed(), **kw)


def test_window_is_a_keyword_that_must_be_given():
    q, k, v = _packed()
    with pytest.raises(TypeError):
        msa.m3_window_attention(q, k, v, cu_tensor([6]), 6)


def test_shapes_and_types():
    q, k, v = _packed()
    for bad in ((q[0], k, v), (q, k[0], v), (q, k, v[:, :1]), (q[:5], k, v), (q[..., :8], k, v), (q[:, :3], k, v),
                (q[:, :0], k, v), (q, k[:, :0], v[:, :0]), (q[..., :0], k[..., :0], v[..., :0])):
        with pytest.raises(ValueError):
            _call(*bad)
    for bad in ((q.float(), k, v), (q, k, v.half()), (q.double(), k.double(), v.double())):
        with pytest.raises(TypeError):
            _call(*bad)
    with pytest.raises(ValueError):
        _call(q, k.to("meta"), v.to("meta"))


@pytest.mark.parametrize("d,dtype", [(12, torch.bfloat16), (264, torch.float16), (4, torch.float32), (12, torch.float32), (264, torch.float32)])
def test_head_dims_that_no_kernel_takes(d, dtype):
    with pytest.raises(NotImplementedError):
        _call(*_packed(d=d, dtype=dtype))


def test_there_is_no_cpu_path():
    for window in (3, None, 1 << 40):
        with pytest.raises(RuntimeError, match="no CPU execution path"):
            _call(*_packed(), window_size=window, sink_tokens=1 << 40)


def _paged(tokens=3, hq=4, g=2, d=16, page=16, pages=4, dtype=torch.bfloat16, cache=None, scales=False):
    cache = cache or dtype
    x = dict(q=torch.zeros(tokens, hq, d, dtype=dtype), k_cache=torch.zeros(pages, g, page, d).to(cache),
             v_cache=torch.zeros(pages, g, page, d).to(cache), page_table=torch.zeros(2, 2, dtype=torch.int32),
             cu_seqlens=cu_tensor([1, tokens - 1]), context_lens=torch.zeros(2, dtype=torch.int32), window_size=3)
    if scales:
        x |= dict(k_scale=torch.ones(pages, g), v_scale=torch.ones(pages, g))
    return x


def _serve(tree, **x):
    if tree:
        x.setdefault("parents", torch.full((x["q"].shape[0],), -1, dtype=torch.int32))
    return (msa.m3_tree_attention_paged if tree else msa.m3_window_attention_paged)(**x)


@pytest.mark.parametrize("tree", [False, True])
def test_paged_arguments(tree):
    x = _paged()
    fp8 = torch.float8_e4m3fn
    for change, error in [
        (dict(window_size=0), ValueError), (dict(sink_tokens=-2), ValueError), (dict(scale=float("nan")), ValueError),
        (dict(q=x["q"].float()), NotImplementedError), (dict(q=x["q"].double()), TypeError), (dict(q=x["q"][0]), ValueError),
        (dict(q=x["q"][:, :3]), ValueError), (dict(q=x["q"][:2]), ValueError), (dict(q=x["q"].half()), TypeError),
        (dict(k_cache=x["k_cache"][0]), ValueError), (dict(k_cache=x["k_cache"][:, :, :8]), ValueError),
        (dict(v_cache=x["v_cache"][:3]), ValueError), (dict(k_cache=x["k_cache"].transpose(2, 3)), ValueError),
        (dict(k_scale=torch.ones(4, 2)), ValueError), (dict(page_table=x["page_table"].long()), TypeError),
        (dict(page_table=x["page_table"][:1]), ValueError), (dict(context_lens=None), TypeError),
        (dict(context_lens=x["context_lens"].long()), TypeError), (dict(context_lens=x["context_lens"][:1]), ValueError),
        (dict(cu_seqlens=cu_tensor([1, 3])), ValueError), (dict(cu_seqlens=torch.tensor([0, 1, 3])), TypeError),
    ]:
        with pytest.raises(error):
            _serve(tree, **dict(x, **change))
    for x in (_paged(cache=fp8), dict(_paged(cache=fp8, scales=True), k_scale=torch.ones(4, 2).half()),
              dict(_paged(cache=fp8, scales=True), v_scale=torch.ones(4, 1))):
        with pytest.raises(ValueError):
            _serve(tree, **x)
    for x in (_paged(d=24), _paged(d=272)):
        with pytest.raises(NotImplementedError):
            _serve(tree, **x)
    with pytest.raises(RuntimeError, match="no CPU execution path"):
        _serve(tree, **_paged(cache=fp8, scales=True))


def test_parents():
    x = _paged()
    for parents, error in ((None, TypeError), ([-1, -1, 0], TypeError), (torch.zeros(3), TypeError),
                           (torch.zeros(3, dtype=torch.int64), TypeError), (torch.zeros(2, dtype=torch.int32), ValueError),
                           (torch.zeros(3, 1, dtype=torch.int32), ValueError),
                           (torch.zeros(3, dtype=torch.int32, device="meta"), ValueError)):
        with pytest.raises(error):
            _serve(True, **x, parents=parents)
    with pytest.raises(NotImplementedError, match="512 nodes"):
        _serve(True, **_paged(tokens=514))


def test_backward_workspace_is_bounded():
    """Beyond delta: parts of sums of at most 256 MiB for each of the two kinds, whatever the window and the first tokens."""
    from msa_triton_amd import _lib

    size = _lib.lib().msa_window_attn_bwd_workspace_bytes
    for code in (0, 1, 2):
        for tokens, seqs, longest in ((1, 1, 1), (1280, 2, 768), (32768, 1, 32768), (32768, 500, 9000), (1 << 20, 10000, 3000),
                                      (1 << 20, 1, 1 << 20)):
            for hq, g, d in ((8, 2, 64), (32, 4, 128), (64, 8, 256), (128, 1, 80)):
                for window in (0, 1, 100, 4096, 1 << 30):
                    for sinks in (0, 1, 4, 130, 5000, 2147483647):
                        got = size(code, tokens, seqs, longest, hq, g, d, window, sinks)
                        delta = 4 * (tokens * hq + 3)
                        assert 4 * tokens * hq <= got <= delta + (2 << 28), (code, tokens, seqs, longest, hq, g, d, window, sinks)
