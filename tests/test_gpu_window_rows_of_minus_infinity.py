"""Rows whose visible logits are all -inf, beside values and keys that are not finite and that these rows do not see.

Such a row has an output of 0 and a log sum of -inf, weights of 0 and so a dq of 0, whatever the rest of its tile holds.
"""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_window_attention import inputs, run
from tests.test_gpu_window_paged import call, oracle, setup

pytestmark = pytest.mark.gpu

INF = float("inf")


PAGED = [  # new tokens, cached tokens, ratio, dim
    (3, 40, 4, 64),       # 16 rows a tile
    (3, 20000, 4, 64),    # the same, shared by several workgroups
    (40, 40, 1, 64),      # 64 rows
    (40, 40, 4, 128),     # 128 rows
    (40, 20000, 4, 128),  # the same, shared
    (40, 20000, 4, 256),
    (300, 3000, 8, 64),   # shared, and joined four rows a wave
    (300, 3000, 8, 256),
]


@pytest.mark.parametrize("dtype,fp8", [(torch.bfloat16, False), (torch.float16, False), (torch.bfloat16, True)])
@pytest.mark.parametrize("new,context,ratio,dim", PAGED)
@pytest.mark.parametrize("drafted", [False, True])
def test_over_a_paged_cache(new, context, ratio, dim, dtype, fp8, drafted):
    """The third new token's value is not finite, in one dim; the first one does not see it, as no node but itself does in a tree
    of which all nodes are children of the context."""
    page = 64
    x = setup([new], [context], 1, ratio, dim, page, dtype, fp8)
    if drafted:
        x["parents"] = torch.full((new,), -1, dtype=torch.int32, device="cuda")
    k = x["kc"].float()
    k[..., 0] = k[..., 0].abs() + 0.5
    x["kc"] = k.to(x["kc"].dtype)
    want, want_lse, tol, lse_tol = oracle(x, [new], [context], 0, 0, dim ** -0.5)
    x["q"] = x["q"].clone()
    x["q"][0, 0, 0] = -INF
    third = context + 2
    at = int(x["table"][0, third // page]), 0, third % page, 3
    sees = slice(2, 3) if drafted else slice(2, new)
    for value in (INF, float("nan")):
        x["vc"] = x["vc"].clone()
        x["vc"].view(torch.uint8 if fp8 else dtype)[at] = 0x7F if fp8 else value
        out, lse = call(x, None, 0)
        assert not out[0, 0].any() and lse[0, 0] == -INF, out[0, 0]
        other = torch.ones_like(out, dtype=torch.bool)
        other[0, 0] = False
        assert ((lse.double() - want_lse).abs() <= lse_tol)[other[..., 0]].all()
        other[sees, :, 3] = False
        assert ((out.double() - want).abs() <= tol)[other].all()
        hit = out[sees, :, 3]
        assert torch.isnan(hit).all() if fp8 or value != value else (hit == INF).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(8, 0), (None, 0), (5, 3)])
def test_gradients_of_queries(dtype, dim, window, sinks):
    """The key that is not finite is later than the row, or in front of its window."""
    n, row = 70, 20
    q, k, v, do = inputs([n], 2, 1, dim, dtype)
    k[..., 0] = k[..., 0].abs() + 0.5
    q[row, 1, 0] = -INF
    want = run(q, k, v, [n], do, window, sinks)
    assert not want[0][row, 1].any() and (want[1][row, 1] == -INF) and not want[2][row, 1].any()
    for at in (row + 5, n - 1, *([row - 9] if window else [])):
        for value in (INF, float("nan")):
            y = k.clone()
            y[at, 0, 3] = value
            out, lse, dq, _, _ = run(q, y, v, [n], do, window, sinks)
            assert not out[row, 1].any() and lse[row, 1] == -INF
            assert not dq[row, 1].any(), (at, value, dq[row, 1])
