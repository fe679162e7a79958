"""Top-k rows of 1025 to 4096 blocks: up to 64 slots by threshold and sort, more pick by pick; random rows, rows of few
distinct values (ties in block order), infinities and NaN, and rows whose causal prefix ends early."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import msa_triton_amd as msa
from oracle import msa_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("blocks,slots,local", [(1025, 1, 1), (1025, 24, 2), (2048, 25, 0), (2048, 64, 64), (2049, 16, 1),
                                                (3001, 64, 3), (4096, 7, 1), (4096, 64, 0), (4096, 65, 1), (1500, 200, 2)])
def test_rows_of_many_blocks(blocks, slots, local, device):
    gen = torch.Generator().manual_seed(blocks * 100 + slots)
    total, groups = blocks, 2  # blocks of one token: every length of causal prefix
    scores = torch.randn(total, groups, blocks, generator=gen)
    scores[::3] = torch.randint(0, 4, scores[::3].shape, generator=gen).float()
    scores[1::7, :, ::2] = -float("inf")
    scores[2::11, :, 5] = float("nan")
    scores[4::13, :, 9::100] = float("inf")
    cu = torch.tensor([0, total], dtype=torch.int32, device=device)
    got = msa.m3_topk(scores.to(device), cu, block_size=1, topk_blocks=slots, local_blocks=local).cpu().numpy()
    rows = np.unique(np.concatenate([np.arange(0, total, 61), np.arange(70), np.arange(total - 70, total),
                                     np.arange(2, total, 97)]))
    want = O.topk_rows(scores[rows].numpy(), rows, block_size=1, topk_blocks=slots, local_blocks=local)
    np.testing.assert_array_equal(got[rows], want)
