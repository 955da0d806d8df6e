"""Refusals of the paged cache's operators at the ends of their arguments (no GPU needed)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from conftest import package, submodule
from test_paged_host import ADDR, attention_args, i32, store_args, strides


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


@pytest.mark.parametrize("k, v", [((2048, 128, 0), (2048, 128, 64)), ((2048, 128, 64), (2048, 0, 64)), ((0, 128, 64), (2048, 128, 64)),
                                  ((2048, 64, 64), (2048, 128, 64)), ((2048, 128, 56), (2048, 128, 64)),
                                  ((1920, 128, 64), (2048, 128, 64))])
def test_store_entry_refuses_caches_whose_slots_share_elements(k, v):
    """[8 pages][16 slots][2 heads][64 columns]; the second cache lies behind the first."""
    args = store_args(k_strides=strides(*k), v_cache=ADDR + 2 * 8 * 2048, v_strides=strides(*v))
    assert submodule("_lib").load().bd_paged_store(*args) == 1


@pytest.mark.parametrize("offset", [0, 16, -16, 112, -112])
def test_store_entry_refuses_caches_over_one_another(offset):
    assert submodule("_lib").load().bd_paged_store(*store_args(k_cache=4096, v_cache=4096 + offset)) == 1


# byte sizes of the call of attention_args(): q and out 3 x 256 x 2, a cache 8 x 2048 x 2, the table 2 x 4 x 4
Q, CACHE, OUT = 1536, 32768, 1536


@pytest.mark.parametrize("name, place, size", [("q", 0x100000, Q), ("k_cache", 0x200000, CACHE), ("v_cache", 0x300000, CACHE),
                                               ("table", 0x400000, 32), ("context", 0x500000, 8), ("starts", 0x600000, 12),
                                               ("workspace", 0x10000000, 1 << 26)])
@pytest.mark.parametrize("where", ["same", "last", "first"])
def test_attention_entry_refuses_an_output_over_what_is_read(name, place, size, where):
    lib = submodule("_lib")
    places = dict(q=0x100000, k_cache=0x200000, v_cache=0x300000, table=0x400000, context=0x500000, starts=0x600000,
                  workspace=0x10000000, workspace_bytes=1 << 26)
    out = {"same": place, "last": place + (size - 1) // 16 * 16, "first": place - OUT + 16}[where]
    args = attention_args(**places, out=out)
    assert lib.load().bd_paged_attention(ctypes.byref(args), None) == 1


def test_sizes_that_depend_on_the_device_are_kept_by_device(monkeypatch):
    """Two GPUs of different SM counts in one process: each has the workspace of its own."""
    lib = submodule("_lib")

    class Fake:
        sms = 0

        def bd_paged_attention_workspace_bytes(self, head_dim):
            return head_dim * self.sms

    fake = Fake()
    monkeypatch.setattr(lib, "load", lambda: fake)
    monkeypatch.setattr(lib, "_SIZES", {})
    for device, sms in ((0, 100), (1, 148), (0, 100), (1, 148)):
        fake.sms = sms
        assert lib.size("bd_paged_attention_workspace_bytes", 128, device=device) == 128 * sms


def test_attention_asks_for_the_workspace_of_its_device(ops):
    import inspect

    assert 'size("bd_paged_attention_workspace_bytes", head_dim, device=index)' in inspect.getsource(ops.paged_attention)


def test_launch_accounting_has_the_sources_constants(ops):
    import re
    from pathlib import Path

    csrc = Path(submodule("_lib").__file__).parent / "csrc"
    plan, attention, shared = ((csrc / f"{n}").read_text() for n in ("paged.cu", "paged_attention.cu", "paged_attention.cuh"))
    assert int(re.search(r"kPlanRows = (\d+);", plan)[1]) == ops._PLAN_ROWS
    assert int(re.search(r"kOneKernelPairs = (\d+);", attention)[1]) == ops._ONE_KERNEL_PAIRS
    narrow, wide = re.search(r"head_dim == 64 \? (\d+) : (\d+)\);", shared).groups()
    assert {64: int(narrow), 128: int(wide)} == ops._FEW_ROWS
