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


@pytest.mark.parametrize("d,dtype", [(12, torch.bfloat16), (264, torch.float16), (6, torch.float32), (260, torch.float32)])
def test_head_dims_that_no_kernel_takes(d, dtype):
    with pytest.raises(NotImplementedError):
        _call(*_packed(d=d, dtype=dtype))


def test_there_is_no_cpu_path():
    for window in (3, None, 1 << 40):
        with pytest.raises(RuntimeError, match="no CPU execution path"):
            _call(*_packed(), window_size=window, sink_tokens=1 << 40)
