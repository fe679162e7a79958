"""Scales of the window operators: scale * log2(e) is held in fp32, where it has to be finite."""

from __future__ import annotations

import struct

import pytest
import torch

import msa_triton_amd as msa
from msa_triton_amd import _lib
from tests.helpers import cu_tensor
from tests.test_window_refusals import _paged, _serve


@pytest.mark.parametrize("scale", [2.4e38, -3e38, 1e39, 1e300])
def test_scales_past_fp32_are_refused(scale):
    q, k = torch.zeros(6, 4, 16), torch.zeros(6, 2, 16)
    with pytest.raises(ValueError, match="scale"):
        msa.m3_window_attention(q, k, k, cu_tensor([6]), 6, window_size=None, scale=scale)
    for tree in (False, True):
        with pytest.raises(ValueError, match="scale"):
            _serve(tree, **_paged(), scale=scale)


def test_c_entry_points():
    """(no tokens: arguments are checked, nothing is launched and no address is read)"""
    p, strides = 4096, struct.pack("8q", *[64] * 8)
    for scale, status in ((2e38, 0), (-2e38, 0), (1e-300, 0), (2.4e38, 1), (-1e39, 1), (float("inf"), 1), (float("nan"), 1)):
        lib = _lib.lib()
        assert lib.msa_window_attn_fwd(p, p, p, 2, strides, p, 1, 0, 4, 2, 64, 0, 0, scale, p, None, None, None) == status
        assert lib.msa_window_attn_bwd(p, p, p, 2, strides, p, 1, 0, 0, 4, 2, 64, 0, 0, scale, p, None, p, p, p, p, p, p, 0, None) == status
        assert lib.msa_window_attn_paged(p, p, p, 2, 0, None, None, strides, None, p, 1, 1, 1, 16, p, 1, 0, p, 0, 4, 2, 64, 0, 0, scale, p, 0, p,
                                         None, None) == status
