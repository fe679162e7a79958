"""An incoming gradient that is an infinity: dk and dv have infinities and NaN where the formula has them, in every type.

ds_ij = p_ij (dO_i . v_j - dO_i . out_i). With one infinity in dO_i at dim c the first product has the sign of v_jc and the second that of
out_ic: ds is an infinity for keys whose value has the other sign than the output, NaN for those that have the same.
"""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_window_attention import inputs, run, visible

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,d,window,sinks", [(20, 64, None, 0), (140, 128, 30, 2), (70, 256, 9, 0), (70, 8, 9, 0)])
@pytest.mark.parametrize("value", [float("inf"), float("-inf")])
def test_an_infinity(dtype, n, d, window, sinks, value):
    hq, g, scale = 4, 2, d ** -0.5
    q, k, v, do = inputs([n], hq, g, d, dtype)
    hits = [(3, 0, 1), (n // 2, 1, 0), (n - 1, 2, d - 1)]
    for hit in hits:
        do[hit] = value
    _, _, dq, dk, dv = run(q, k, v, [n], do, window, sinks)
    seen = visible(n, window, sinks, "cuda")
    q, k, v, do = (x.double() for x in (q, k, v, do))
    want = [torch.zeros_like(x) for x in (q, k, v)]
    for h in range(hq):
        kk, vv, y = k[:, h // 2], v[:, h // 2], do[:, h]
        p = torch.softmax((q[:, h] @ kk.T * scale).masked_fill(~seen, float("-inf")), 1)
        delta = (y * (p @ vv)).sum(1, keepdim=True)
        ds = p * ((y[:, None] * vv).sum(2) - delta)
        over = seen[:, :, None]
        want[0][:, h] = torch.where(over, ds[:, :, None] * kk, 0.0).sum(1)
        want[1][:, h // 2] += torch.where(over, ds[:, :, None] * q[:, None, h], 0.0).sum(0)
        want[2][:, h // 2] += torch.where(over, p[:, :, None] * y[:, None], 0.0).sum(0)
    assert torch.isinf(want[1]).any() and torch.isnan(want[1]).any()
    for name, got, exact in zip(("dq", "dk", "dv"), (dq, dk, dv), want):
        for kind in (torch.isnan, torch.isposinf, torch.isneginf):
            assert torch.equal(kind(got), kind(exact)), (name, kind.__name__)
