"""Refusals of the paged cache's operators, before any device work (no GPU needed)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from conftest import package, submodule

ADDR = 256  # never dereferenced: every call below is refused on the host


@pytest.fixture(scope="module")
def ops():
    return package().ops


def strides(*values):
    return (ctypes.c_int64 * 3)(*values)


def plan_args(**change):
    names = ("context", "count", "requests", "page_size", "pool", "table", "ld", "width", "owned_in", "owned_out", "free",
             "capacity", "top_in", "top_out", "starts", "positions", "slots", "rows", "flags", "stream")
    values = dict(zip(names, (ADDR, ADDR, 2, 16, 8, ADDR, 4, 4, ADDR, ADDR, ADDR, 8, ADDR, ADDR, ADDR, ADDR, ADDR, 3,
                              None, None)))
    values.update(change)
    return [values[n] for n in names]


@pytest.mark.parametrize("change", [dict(requests=0), dict(page_size=12), dict(page_size=4), dict(page_size=512),
                                    dict(pool=0), dict(pool=1 << 28), dict(width=0), dict(ld=3), dict(width=1 << 28, ld=1 << 28),
                                    dict(capacity=-1), dict(rows=-1), dict(context=None), dict(count=None),
                                    dict(table=None), dict(owned_in=None), dict(owned_out=None), dict(free=None),
                                    dict(top_in=None), dict(top_out=None), dict(starts=None), dict(positions=None),
                                    dict(slots=None)])
def test_plan_entry_refuses(change):
    assert submodule("_lib").load().bd_page_plan(*plan_args(**change)) == 1


def store_args(**change):
    names = ("k", "k_row", "k_head", "v", "v_row", "v_head", "row_type", "slots", "rows", "kv_heads", "head_dim", "page_size",
             "pool", "k_cache", "k_strides", "v_cache", "v_strides", "cache_type", "flags", "stream")
    values = dict(zip(names, (ADDR, 128, 64, ADDR, 128, 64, 0, ADDR, 3, 2, 64, 16, 8, ADDR, strides(2048, 128, 64), ADDR,
                              strides(2048, 128, 64), 0, None, None)))
    values.update(change)
    return [values[n] for n in names]


@pytest.mark.parametrize("change, status", [
    (dict(rows=-1), 1), (dict(kv_heads=0), 1), (dict(head_dim=60), 1), (dict(head_dim=0), 1), (dict(page_size=7), 1),
    (dict(row_type=3), 1), (dict(cache_type=2), 1), (dict(k=None), 1), (dict(slots=None), 1), (dict(v_cache=None), 1),
    (dict(k=ADDR + 2), 2), (dict(v_cache=ADDR + 8), 2), (dict(k_row=127), 2), (dict(v_head=60), 2),
    (dict(k_strides=strides(2048, 132, 64)), 2), (dict(v_strides=strides(-2048, 128, 64)), 2), (dict(rows=0), 0),
])
def test_store_entry_refuses(change, status):
    assert submodule("_lib").load().bd_paged_store(*store_args(**change)) == status


def attention_args(**change):
    lib = submodule("_lib")
    values = dict(q=ADDR, q_row=256, q_head=64, row_type=0, k_cache=ADDR, v_cache=ADDR, k_strides=(2048, 128, 64),
                  v_strides=(2048, 128, 64), cache_type=0, page_size=16, pool_pages=8, table=ADDR, table_ld=4,
                  table_width=4, context=ADDR, starts=ADDR, requests=2, rows=3, heads=4, kv_heads=2, head_dim=64, causal=1,
                  window=0, longest=0, scale=0.125, out=ADDR, zero_fill=0, workspace=ADDR, workspace_bytes=1 << 30,
                  flags=None)
    values.update(change)
    return lib.PagedAttentionArgs(**values)


@pytest.mark.parametrize("change, status", [
    (dict(rows=-1), 1), (dict(requests=-1), 1), (dict(heads=5), 1), (dict(kv_heads=0), 1), (dict(heads=0), 1),
    (dict(head_dim=96), 1), (dict(page_size=24), 1), (dict(pool_pages=0), 1), (dict(table_width=0), 1),
    (dict(table_ld=3), 1), (dict(window=-1), 1), (dict(longest=-1), 1), (dict(scale=float("nan")), 1),
    (dict(scale=float("inf")), 1), (dict(row_type=2, cache_type=1), 1), (dict(row_type=0, cache_type=1), 1),
    (dict(row_type=7), 1), (dict(q=None), 1), (dict(out=None), 1), (dict(k_cache=None), 1), (dict(table=None), 1),
    (dict(context=None), 1), (dict(starts=None), 1), (dict(q=ADDR + 4), 2), (dict(q_row=252), 2), (dict(out=ADDR + 2), 2),
    (dict(k_strides=(2048, 130, 64)), 2), (dict(v_strides=(2048, 128, -64)), 2), (dict(workspace=None), 4),
    (dict(workspace_bytes=1024), 4), (dict(rows=0), 0),
])
def test_attention_entry_refuses(change, status):
    lib = submodule("_lib")
    assert lib.load().bd_paged_attention(ctypes.byref(attention_args(**change)), None) == status


def i32(*values):
    return torch.tensor(values, dtype=torch.int32)


def test_plan_wrapper_refuses(ops):
    table = torch.full((2, 4), -1, dtype=torch.int32)
    good = dict(context=i32(1, 2), count=i32(1, 1), table=table, owned=i32(0, 0), free=i32(0, 1, 2), top=i32(3),
                page_size=16, rows=2, pool_pages=3)

    def refused(message, **change):
        with pytest.raises(ValueError, match=message):
            ops.page_plan(**{**good, **change})

    refused("at least one request", context=torch.zeros(0, dtype=torch.int32))
    refused("at least one request", context=torch.zeros((2, 1), dtype=torch.int32))
    refused("context must be", context=torch.zeros(2, dtype=torch.int64))
    refused("count must be", count=i32(1))
    refused("owned must be", owned=i32(1, 2, 3))
    refused("top must be", top=i32(1, 2))
    refused("free must be", free=torch.zeros(3))
    refused("owned_out must be", owned_out=i32(1))
    refused("top_out must be", top_out=torch.zeros(1))
    refused("table must be", table=table.long())
    refused("table must be", table=table.t())
    refused("table must be", table=table[:1])
    refused("page_size must be", page_size=10)
    refused("rows must not", rows=-1)
    refused("CUDA tensors")


def test_store_wrapper_refuses(ops):
    cache = torch.zeros((3, 16, 2, 64), dtype=torch.float16)
    rows = torch.zeros((5, 2, 64))
    good = dict(k=rows, v=rows, slots=i32(0, 1, 2, 3, 4), k_cache=cache, v_cache=cache.clone())

    def refused(message, **change):
        with pytest.raises(ValueError, match=message):
            ops.paged_store(**{**good, **change})

    refused("caches must be", k_cache=cache.float())
    refused("caches must be", v_cache=cache[:2])
    refused("page_size must be", k_cache=cache[:, :12], v_cache=cache[:, :12])
    refused("unit stride within a head", k_cache=cache.transpose(2, 3).contiguous().transpose(2, 3))
    refused("k and v must be", k=rows[:, :1], v=rows[:, :1])
    refused("k and v must be", k=rows.double(), v=rows.double())
    refused("k and v must be", v=rows.half())
    refused("k and v need unit", k=torch.zeros((5, 64, 2)).transpose(1, 2))
    refused("slots must be", slots=i32(0, 1))
    refused("CUDA tensors")


def test_attention_wrapper_refuses(ops):
    cache = torch.zeros((3, 16, 2, 64), dtype=torch.float16)
    q = torch.zeros((5, 4, 64))
    good = dict(q=q, k_cache=cache, v_cache=cache.clone(), table=torch.zeros((2, 3), dtype=torch.int32),
                context=i32(3, 4), starts=i32(0, 2, 5))

    def refused(message, **change):
        with pytest.raises(ValueError, match=message):
            ops.paged_attention(**{**good, **change})

    refused("q must be", q=q.bfloat16())
    refused("q must be", q=q[0])
    refused("head_dim must be", q=torch.zeros((5, 4, 128)))
    refused("head_dim must be", q=torch.zeros((5, 3, 64)))
    refused("head_dim must be", q=torch.zeros((5, 4, 32)), k_cache=cache[..., :32], v_cache=cache[..., :32])
    refused("q needs unit", q=torch.zeros((5, 64, 4)).transpose(1, 2))
    refused("starts must be", starts=i32(0, 5))
    refused("context must be", context=torch.zeros(2))
    refused("table must be", table=torch.zeros((1, 3), dtype=torch.int32))
    refused("window must be", window=0)
    refused("longest must be", longest=0)
    refused("CUDA tensors")


def test_flag_messages_of_the_paged_cache():
    lib = submodule("_lib")
    for bit, message in ((lib.FLAG_BAD_LENGTH, "out of range"), (lib.FLAG_NO_PAGES, "out of free"),
                         (lib.FLAG_NO_PAGES | lib.FLAG_BAD_PAGE, "out of free"), (lib.FLAG_BAD_PAGE, "outside the pool")):
        with pytest.raises(ValueError, match=message):
            lib.raise_flags(bit)
