"""The package's names: those bound on first use like the others."""

import subprocess
import sys

import pytest

import msa_triton_amd as msa


def test_all_names_resolve_and_unknown_ones_do_not():
    for name in msa.__all__:
        assert callable(getattr(msa, name)) and name in dir(msa)
    assert msa.m3_cache_append is msa.m3_cache_append
    with pytest.raises(AttributeError, match="no attribute 'm3_nothing'"):
        msa.m3_nothing


def test_names_in_a_fresh_process():
    code = ("from msa_triton_amd import *; from msa_triton_amd import m3_qk_norm_rope as f; import msa_triton_amd as m;"
            "assert f is m3_qk_norm_rope is m.m3_qk_norm_rope and m3_sparse_attention_paged.__name__ in m.__all__")
    subprocess.run([sys.executable, "-c", code], check=True, timeout=120)
