"""Window attention with scales next to the least normal number: every visible key has one weight, and the log sum counts them."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_window_attention import against, inputs, run
from tests.test_gpu_window_paged import check, setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [1e-37, 1e-38, -1e-38, 1e-40])
@pytest.mark.parametrize("new,context", [(1, 300), (3, 20000), (40, 300), (40, 20000), (600, 3000)])
@pytest.mark.parametrize("dtype,fp8", [(torch.bfloat16, False), (torch.float16, True)])
def test_over_a_paged_cache(new, context, scale, dtype, fp8):
    x = setup([new], [context], 1, 4, 64, 64, dtype, fp8)
    check(x, [new], [context], None, 0, scale=scale)
    check(x, [new], [context], 100, 4, scale=scale)


@pytest.mark.parametrize("scale", [1e-37, 1e-38, -1e-38, 1e-40])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_packed(dtype, scale):
    q, k, v, _ = inputs([90, 33], 4, 2, 64, dtype)
    against(run(q, k, v, [90, 33], None, 40, 3, scale=scale), q, k, v, [90, 33], 40, 3, scale, None)
