"""Refusals of the paged cache's operators at the ends of their arguments (no GPU needed)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from conftest import package, submodule
from test_paged_host import attention_args, i32


@pytest.fixture(scope="module")
def ops():
    return package().ops


@pytest.mark.parametrize("scale", [2.4e38, -2.4e38, 3.4e38])
def test_attention_entry_refuses_scales_that_overflow(scale):
    lib = submodule("_lib")
    assert lib.load().bd_paged_attention(ctypes.byref(attention_args(scale=scale)), None) == 1


def test_attention_wrapper_refuses_scales_that_are_no_numbers_of_fp32(ops):
    cache = torch.zeros((3, 16, 2, 64), dtype=torch.float16)
    good = dict(q=torch.zeros((5, 4, 64)), k_cache=cache, v_cache=cache.clone(), table=torch.zeros((2, 3), dtype=torch.int32),
                context=i32(3, 4), starts=i32(0, 2, 5))
    for scale in (float("nan"), float("inf"), -float("inf"), 1e39, -2.4e38):
        with pytest.raises(ValueError, match="scale must be"):
            ops.paged_attention(**good, scale=scale)
    for scale in (1e38, 0.0, -0.5, None):
        with pytest.raises(ValueError, match="CUDA tensors"):
            ops.paged_attention(**good, scale=scale)
