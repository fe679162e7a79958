"""Values whose weighted sums leave fp32's range before they are divided: the outputs are means of them, and finite."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_window_attention import against, inputs, run
from tests.test_gpu_window_paged import check, setup

pytestmark = pytest.mark.gpu

SIZES = (3e38, 2e36, 1e34)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 256)])
@pytest.mark.parametrize("size", SIZES)
def test_packed(dtype, dim, size):
    lengths, window = [700, 3], 300
    q, k, v, do = inputs(lengths, 4, 2, dim, dtype)
    q = q * 3  # (weights of all sizes)
    v = torch.where(v < 0, -size, size * 0.75).to(dtype)
    against(run(q, k, v, lengths, None, window, 3), q, k, v, lengths, window, 3, dim ** -0.5, None)
    # as it is saved for a backward pass (whose sums over dims are past the range)
    out = run(q, k, v, lengths, do, window, 3)[0]
    assert torch.isfinite(out).all()
    assert ((out.double() - run(q, k, v, lengths, None, window, 3)[0].double()).abs() <= 2.0 ** -6 * size).all()


@pytest.mark.parametrize("dtype,fp8", [(torch.bfloat16, False), (torch.bfloat16, True)])
@pytest.mark.parametrize("new,context,ratio", [(1, 500, 4), (3, 20000, 4), (40, 300, 4), (40, 20000, 4), (300, 3000, 8)])
@pytest.mark.parametrize("size", SIZES)
def test_over_a_paged_cache(new, context, ratio, dtype, fp8, size):
    """(8-bit values reach 448: their scale is the large one)"""
    x = setup([new], [context], 1, ratio, 64, 64, dtype, fp8)
    if fp8:
        x["vs"] = torch.where(torch.isnan(x["vs"]), x["vs"], size / 448)
        there = x["vc"].float()
        x["vc"] = torch.where(there < 0, -448.0, torch.where(there >= 0, 320.0, there)).to(x["vc"].dtype)
    else:
        x["vc"] = torch.where(x["vc"] < 0, -size, torch.where(x["vc"] >= 0, 0.75 * size, x["vc"])).to(dtype)
    check(x, [new], [context], None, 0)
    check(x, [new], [context], 200, 3)
