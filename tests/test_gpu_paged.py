"""The paged cache on the GPU: page plan, store and attention against plain 64-bit
implementations, and the three of them together (needs a B200)."""

from __future__ import annotations

import math

import pytest
import torch

from conftest import package, submodule

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module")
def ops():
    return package().ops


def dev32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------ plan


def plain_plan(context, count, table, owned, stack, top, page, rows, pool):
    """The plan in plain Python, on lists; returns everything that it changes."""
    table, owned, stack = [list(r) for r in table], list(owned), list(stack)
    free = stack[:top]
    need = [-(-(c + n) // page) for c, n in zip(context, count)]
    for b in range(len(context)):
        for j in range(need[b], owned[b]):
            free.append(table[b][j])
            table[b][j] = -1
        owned[b] = min(owned[b], need[b])
    short, available, wanted, used = False, len(free), 0, 0
    stack[:len(free)] = free
    for b in range(len(context)):
        lack = max(0, need[b] - owned[b])
        wanted += lack
        if lack and wanted > available:
            short = True
            continue
        for _ in range(lack):
            table[b][owned[b]] = free[available - 1 - used]
            owned[b] += 1
            used += 1
    starts, positions, slots = [0], [], []
    for b in range(len(context)):
        for t in range(count[b]):
            p = context[b] + t
            positions.append(p)
            slots.append(table[b][p // page] * page + p % page if p // page < owned[b] else -1)
        starts.append(len(positions))
    positions, slots = positions[:rows], slots[:rows]
    tail = [-1] * (rows - len(positions))
    return table, owned, stack, available - used, starts, positions + tail, slots + tail, short


def plan_case(seed, requests, width, page, pool_extra, rows_extra, finish=0.0):
    g = torch.Generator().manual_seed(seed)

    def rand(n):
        return int(torch.randint(0, n + 1, (1,), generator=g))

    owned = [rand(width) for _ in range(requests)]
    context, count = [], []
    for b in range(requests):
        if finish and float(torch.rand(1, generator=g)) < finish:
            context.append(0)
            count.append(0)
            continue
        length = rand(width * page)
        n = rand(min(length, 3 * page))
        context.append(length - n)
        count.append(n)
    need = [-(-(c + n) // page) for c, n in zip(context, count)]
    pool = max(1, sum(max(a, b) for a, b in zip(owned, need)) + pool_extra)  # a pool has a page
    ids = torch.randperm(pool, generator=g).tolist()
    table, at = [], 0
    for b in range(requests):
        table.append(ids[at:at + owned[b]] + [-1] * (width - owned[b]))
        at += owned[b]
    stack = ids[at:]
    return dict(context=context, count=count, table=table, owned=owned, stack=stack + [-7] * at, top=len(stack), page=page,
                rows=sum(count) + rows_extra, pool=pool)


def run_plan(ops, c, in_place=True):
    table, owned = dev32(c["table"]), dev32(c["owned"])
    free, top = dev32(c["stack"]), dev32([c["top"]])
    flags = ops.Flags(DEV)
    more = {} if in_place else dict(owned_out=torch.empty_like(owned), top_out=torch.empty_like(top))
    plan = ops.page_plan(dev32(c["context"]), dev32(c["count"]), table, owned, free, top, c["page"], c["rows"], c["pool"],
                         flags=flags, **more)
    if not in_place:
        assert owned.tolist() == c["owned"] and top.tolist() == [c["top"]]
        owned, top = more["owned_out"], more["top_out"]
    return table, owned, free, top, plan, int(flags.tensor.item())


def check_plan(ops, c, in_place=True):
    lib = submodule("_lib")
    table, owned, free, top, plan, flag = run_plan(ops, c, in_place)
    w_table, w_owned, w_stack, w_top, starts, positions, slots, short = plain_plan(
        c["context"], c["count"], c["table"], c["owned"], c["stack"], c["top"], c["page"], c["rows"], c["pool"])
    assert plan.starts.tolist() == starts
    assert plan.positions.tolist() == positions
    assert plan.slots.tolist() == slots
    assert table.tolist() == w_table and owned.tolist() == w_owned and top.tolist() == [w_top]
    assert free.tolist()[:w_top] == w_stack[:w_top]
    assert flag == (lib.FLAG_NO_PAGES if short else 0) | (lib.FLAG_BAD_LENGTH if sum(c["count"]) > c["rows"] else 0)


@pytest.mark.parametrize("requests, width, page, pool_extra, rows_extra", [
    (1, 1, 8, 0, 0), (1, 4, 16, 3, 5), (2, 3, 256, 0, 1), (33, 7, 16, 11, 0), (100, 40, 8, 5, 17), (1025, 3, 16, 4, 100),
    (2500, 2, 8, 0, 0), (7, 300, 32, 9, 3000), (1, 900, 8, 2, 0),
])
@pytest.mark.parametrize("in_place", [True, False])
def test_plan_takes_and_gives_pages(ops, requests, width, page, pool_extra, rows_extra, in_place):
    for finish in (0.0, 0.4):
        check_plan(ops, plan_case(requests * 7 + page, requests, width, page, pool_extra, rows_extra, finish), in_place)


def test_plan_of_growing_requests_is_a_fixed_point(ops):
    c = plan_case(5, 20, 9, 16, 4, 3)
    table, owned, free, top, plan, _ = run_plan(ops, c)
    again = ops.page_plan(dev32(c["context"]), dev32(c["count"]), table, owned, free, top, 16, c["rows"], c["pool"])
    assert all(torch.equal(x, y) for x, y in zip(plan, again))


def test_plan_without_enough_pages_serves_the_first(ops):
    c = dict(context=[0, 16, 0, 3], count=[40, 5, 10, 2], table=[[-1] * 4, [5, -1, -1, -1], [-1] * 4, [6, -1, -1, -1]],
             owned=[0, 1, 0, 1], stack=[0, 1, 2, 3], top=4, page=16, rows=57, pool=8)
    check_plan(ops, c)
    check_plan(ops, {**c, "top": 3, "stack": [0, 1, 2, -9]})  # the second and third request get nothing
    check_plan(ops, {**c, "top": 0, "stack": [-9] * 4})
    with pytest.raises(ValueError, match="out of free cache pages"):
        ops.page_plan(dev32(c["context"]), dev32(c["count"]), dev32(c["table"]), dev32(c["owned"]), dev32([0]), dev32([1]),
                      16, 57, 8)


def test_plan_with_too_few_rows_flags_and_stays_inside(ops):
    for rows_extra in (-3, -40):
        check_plan(ops, plan_case(11, 30, 6, 16, 2, rows_extra))
    many = plan_case(12, 100, 60, 64, 2, 0)
    assert many["rows"] > 4096
    check_plan(ops, {**many, "rows": many["rows"] - 9})
    check_plan(ops, {**many, "rows": 4097})


def test_plan_of_more_tokens_than_32_bits_count(ops):
    """Lengths that each fit and together do not: flagged, and nothing outside the rows is written."""
    lib = submodule("_lib")
    requests, width, page, rows = 140_000, 64, 256, 5000
    table = torch.full((requests, width), -1, dtype=torch.int32, device=DEV)
    count = torch.full((requests,), width * page, dtype=torch.int32, device=DEV)
    context, owned = torch.zeros_like(count), torch.zeros_like(count)
    free, top, flags = torch.arange(70, dtype=torch.int32, device=DEV), dev32([70]), ops.Flags(DEV)
    plan = ops.page_plan(context, count, table, owned, free, top, page, rows, 70, flags=flags)
    assert int(flags.tensor.item()) == lib.FLAG_BAD_LENGTH | lib.FLAG_NO_PAGES
    starts = plan.starts.tolist()
    assert starts == [min(b * width * page, 2 ** 31 - 1) for b in range(requests + 1)]
    # the first request has the 64 pages that it needs, from the top of the stack
    assert table[0].tolist() == list(range(69, 5, -1)) and not (table[1:] >= 0).any() and int(top) == 6
    assert plan.positions.tolist() == list(range(rows))
    assert plan.slots.tolist() == [(69 - r // page) * page + r % page for r in range(rows)]


@pytest.mark.parametrize("context, count", [([-1, 3], [2, 2]), ([3, 1], [2, -5]), ([60, 1], [5, 1]),
                                            ([2 ** 31 - 1, 1], [2 ** 31 - 1, 1])])
def test_plan_leaves_out_requests_with_bad_lengths(ops, context, count):
    lib = submodule("_lib")
    table, flags = dev32([[0, 1, -1, -1], [2, -1, -1, -1]]), ops.Flags(DEV)
    owned, top = dev32([2, 1]), dev32([3])
    plan = ops.page_plan(dev32(context), dev32(count), table, owned, dev32([3, 4, 5]), top, 16, 8, 6, flags=flags)
    assert int(flags.tensor.item()) == lib.FLAG_BAD_LENGTH
    bad = [b for b in range(2) if context[b] < 0 or count[b] < 0 or context[b] + count[b] > 64]
    assert len(bad) == 1 and plan.starts.tolist()[-1] == count[1 - bad[0]]
    assert table.tolist()[bad[0]] == [[0, 1, -1, -1], [2, -1, -1, -1]][bad[0]]
    assert owned.tolist()[bad[0]] == [2, 1][bad[0]]


def test_plan_refuses_bad_pages_and_stacks(ops):
    lib = submodule("_lib")

    def flag(table, stack, top, owned=(1,)):
        flags = ops.Flags(DEV)
        plan = ops.page_plan(dev32([10]), dev32([20]), dev32([table]), dev32(list(owned)), dev32(stack), dev32([top]), 16, 20,
                             4, flags=flags)
        return int(flags.tensor.item()), plan.slots.tolist()

    assert flag([0, -1], [1, 2], 2) == (0, [10 + i for i in range(6)] + [32 + i for i in range(14)])
    got, slots = flag([9, -1], [1, 2], 2)
    assert got == lib.FLAG_BAD_PAGE and slots == [-1] * 6 + [32 + i for i in range(14)]
    got, slots = flag([0, -1], [1, 4], 2)
    assert got == lib.FLAG_BAD_PAGE and slots == [10 + i for i in range(6)] + [-1] * 14
    assert flag([0, -1], [1, 2], 5)[0] & lib.FLAG_BAD_LENGTH
    assert flag([0, -1], [1, 2], -2)[0] & lib.FLAG_BAD_LENGTH
    assert flag([0, -1], [1, 2], 2, owned=(3,))[0] & lib.FLAG_BAD_LENGTH


# ------------------------------------------------------------------ store


@pytest.mark.parametrize("cache_type", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("row_type", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows, kv_heads, head_dim, page, heads_first", [
    (1, 1, 64, 8, False), (5, 3, 128, 16, True), (67, 8, 128, 64, False), (700, 5, 72, 256, True), (3, 2, 8, 8, False)])
def test_store_rounds_rows_into_slots(ops, row_type, cache_type, rows, kv_heads, head_dim, page, heads_first):
    g = torch.Generator(device=DEV).manual_seed(rows)
    pages = rows // page + 3
    shape = (pages, kv_heads, page, head_dim) if heads_first else (pages, page, kv_heads, head_dim)
    caches = [torch.randn(shape, generator=g, device=DEV).to(cache_type) for _ in range(2)]
    caches = [c.transpose(1, 2) if heads_first else c for c in caches]
    fused = (torch.randn((rows, 2 * kv_heads * head_dim + 16), generator=g, device=DEV) * 4).to(row_type)
    width = kv_heads * head_dim
    k, v = (fused[:, s:s + width].unflatten(1, (kv_heads, head_dim)) for s in (0, width + 16))
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:rows].to(torch.int32)
    slots[rows // 3::5] = -1
    want = [c.clone() for c in caches]
    for w, x in zip(want, (k, v)):
        for r in range(rows):
            s = int(slots[r])
            if s >= 0:
                w[s // page, s % page] = x[r].double().to(cache_type)  # one rounding from the exact value
    ops.paged_store(k, v, slots, *caches)
    for c, w in zip(caches, want):
        assert torch.equal(c.contiguous().view(torch.int16), w.contiguous().view(torch.int16))


def test_store_reports_overflow_and_bad_slots(ops):
    lib = submodule("_lib")
    cache = torch.zeros((2, 8, 1, 64), dtype=torch.float16, device=DEV)
    k = torch.ones((3, 1, 64), device=DEV)

    def flag(k, v, slots):
        flags = ops.Flags(DEV)
        ops.paged_store(k, v, dev32(slots), cache, cache.clone(), flags=flags)
        return int(flags.tensor.item())

    assert flag(k, k, [0, 5, 15]) == 0
    assert flag(k, k, [0, 16, -5]) == lib.FLAG_BAD_PAGE
    assert flag(k, k, [0, 2 ** 31 - 1, 3]) == lib.FLAG_BAD_PAGE
    for value in (65520.0, math.inf, math.nan):
        big = k.clone()
        big[1, 0, 63] = value
        assert flag(k, big, [0, 5, 15]) == lib.FLAG_CACHE_OVERFLOW
        assert flag(big, k, [0, 5, 15]) == lib.FLAG_CACHE_OVERFLOW
        assert flag(big, k, [0, -1, 15]) == 0  # not stored
    big[1, 0, 63] = 65504.0
    assert flag(big, big, [0, 5, 15]) == 0
    with pytest.raises(ValueError, match="cache storage overflow"):
        ops.paged_store(k * 1e6, k, dev32([0, 1, 2]), cache, cache.clone())
    ops.paged_store(k[:0], k[:0], dev32([]), cache, cache)


# ------------------------------------------------------------------ attention


class Batch:
    """Requests of given (context, count) over a paged cache with random pages."""

    def __init__(self, lengths, heads, kv_heads, head_dim, page, row_type=torch.float32, seed=0, heads_first=False,
                 spread=1.0, extra_rows=0, extra_width=1):
        cache_type = torch.bfloat16 if row_type == torch.bfloat16 else torch.float16
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.lengths, self.heads, self.kv_heads, self.head_dim, self.page = lengths, heads, kv_heads, head_dim, page
        need = [-(-(c + n) // page) for c, n in lengths]
        pool = sum(need) + 3
        ids = torch.randperm(pool, generator=g, device=DEV).tolist()
        width = max(need + [1]) + extra_width
        rows, at = [], 0
        for n in need:
            rows.append(ids[at:at + n] + [-1] * (width - n))
            at += n
        self.table = dev32(rows).reshape(len(lengths), width)
        shape = (pool, kv_heads, page, head_dim) if heads_first else (pool, page, kv_heads, head_dim)
        caches = [torch.randn(shape, generator=g, device=DEV).to(cache_type) for _ in range(2)]
        self.k, self.v = (c.transpose(1, 2) if heads_first else c for c in caches)
        self.context = dev32([c for c, _ in lengths])
        starts = [0]
        for _, n in lengths:
            starts.append(starts[-1] + n)
        self.starts = dev32(starts)
        total = starts[-1] + extra_rows
        fused = torch.randn((total, heads * head_dim + 8), generator=g, device=DEV) * spread
        self.q = fused.to(row_type)[:, :heads * head_dim].unflatten(1, (heads, head_dim))

    def run(self, ops, **how):
        return ops.paged_attention(self.q, self.k, self.v, self.table, self.context, self.starts, **how)

    def expected(self, causal=True, window=None, scale=None):
        """(output, bound of its error) per element in 64 bits: see the derivation at check()."""
        d, u, group = self.head_dim, HALF_STEP[self.q.dtype], self.heads // self.kv_heads
        scale = d ** -0.5 if scale is None else scale
        out = torch.zeros(self.q.shape, dtype=torch.float64, device=DEV)
        bound = torch.zeros_like(out)
        row = 0
        for b, (context, count) in enumerate(self.lengths):
            length = context + count
            if count == 0:
                continue
            at = torch.arange(length, device=DEV)
            page = self.table[b, (at // self.page)].long()
            k = self.k[page, at % self.page].double().repeat_interleave(group, 1)  # [s, heads, d]
            v = self.v[page, at % self.page].double().repeat_interleave(group, 1)
            q = self.q[row:row + count].double()
            gap = (context + torch.arange(count, device=DEV))[:, None] - at
            seen = torch.ones_like(gap, dtype=torch.bool)
            if causal:
                seen &= gap >= 0
            if window:
                seen &= gap.abs() < window
            for h in range(self.heads):
                kh = torch.where(seen.any(0)[:, None], k[:, h], 0.0)
                vh = torch.where(seen.any(0)[:, None], v[:, h], 0.0)
                s = (q[:, h] @ kh.T) * scale
                size = (q[:, h].abs() @ kh.abs().T) * abs(scale)
                s = torch.where(seen, s, -math.inf)
                p = torch.softmax(s, -1)
                out[row:row + count, h] = p @ vh
                reach = torch.where(seen, size, 0.0).amax(-1, keepdim=True)
                a = p @ vh.abs()
                # exponent: d exact products added in fp32 (one unit each), the scale, log2 e and the
                # maximum's subtraction rounded, ex2 within 2^-22; for fp32 rows the halves' 2^-21
                delta = (d + 12) * 2.0 ** -23 * reach + 2.0 ** -21
                if self.q.dtype == torch.float32:
                    delta = delta + 2.0 ** -20 * reach
                    weight = 2.0 ** -21
                    floor = length * 2.0 ** -24 * vh.abs().amax()
                else:
                    weight, floor = u, 0.0
                # P rounded once, sums of length / 16 + 16 steps and the joins in fp32, then the output's rounding
                sums = 2 * (length / 16 + 64) * 2.0 ** -23
                bound[row:row + count, h] = u * out[row:row + count, h].abs() + a * (weight + 2 * delta + sums) * 1.1 + floor
            row += count
        return out, bound


def check(ops, batch, causal=True, window=None, scale=None, **how):
    """Each element within its bound (rounding and accumulation, as derived in
    ``expected``); the whole within the rounding of P and of the output: each at most half
    a step, so at most their sum in the 2-norm for independent signs of the terms
    (fp32 rows: 2^-18, the exponent's error at the sizes used here)."""
    got = batch.run(ops, causal=causal, window=window, scale=scale, **how).double()
    want, bound = batch.expected(causal, window, scale)
    err = (got - want).abs()
    assert bool(torch.isfinite(got).all())
    assert bool((err <= bound).all()), (float((err / bound.clamp(min=1e-300)).max()), int((err > bound).sum()))
    if want.norm() > 0 and batch.q.dtype != torch.float32:
        assert float(err.norm() / want.norm()) <= 2 * HALF_STEP[batch.q.dtype]
    elif want.norm() > 0:
        assert float(err.norm() / want.norm()) <= 2.0 ** -18
    return got


TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("row_type", TYPES)
@pytest.mark.parametrize("heads, kv_heads, head_dim", [(1, 1, 64), (4, 1, 128), (6, 2, 64), (10, 2, 128), (8, 8, 64),
                                                       (32, 8, 128), (16, 1, 64)])
def test_attention_of_small_batches(ops, row_type, heads, kv_heads, head_dim):
    lengths = [(0, 1), (5, 0), (63, 1), (64, 1), (0, 17), (31, 3), (200, 16), (1, 2)]
    batch = Batch(lengths, heads, kv_heads, head_dim, 16, row_type, seed=heads)
    check(ops, batch)
    check(ops, batch, causal=False)
    check(ops, batch, window=7)
    check(ops, batch, causal=False, window=5, longest=17)


@pytest.mark.parametrize("row_type", TYPES)
@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
def test_attention_with_every_page_size(ops, row_type, page):
    lengths = [(page - 1, 1), (page, 1), (3 * page + 5, 20), (0, page + 1), (2 * page - 7, 150)]
    for heads_first in (False, True):
        batch = Batch(lengths, 4, 2, 128, page, row_type, seed=page, heads_first=heads_first)
        check(ops, batch)
        check(ops, batch, window=page + 3)


@pytest.mark.parametrize("row_type", TYPES)
@pytest.mark.parametrize("lengths", [[(4096, 16)], [(20000, 1)], [(0, 700)], [(1500, 333), (0, 1), (800, 129)],
                                     [(i * 37 % 500, 1 + i % 3) for i in range(150)],
                                     [(1000 + 11 * i, 17) for i in range(9)], [(0, 0), (0, 0), (9000, 5)]])
@pytest.mark.parametrize("causal, window", [(True, None), (False, None), (True, 100), (False, 1000)])
def test_attention_of_long_and_ragged_batches(ops, row_type, lengths, causal, window):
    check(ops, Batch(lengths, 8, 2, 128, 16, row_type, seed=3), causal=causal, window=window)
    check(ops, Batch(lengths, 6, 2, 64, 32, row_type, seed=4), causal=causal, window=window,
          longest=max(n for _, n in lengths))


@pytest.mark.parametrize("row_type", TYPES)
def test_attention_of_sharp_and_flat_weights_and_scales(ops, row_type):
    lengths = [(300, 20), (40, 1)]
    for spread, scale in ((20.0, None), (0.0, None), (1.0, 0.5), (1.0, -0.125), (1.0, 0.0), (1e-3, 40.0)):
        check(ops, Batch(lengths, 4, 2, 64, 16, row_type, seed=9, spread=spread), scale=scale)


def test_fp32_rows_of_any_size_keep_their_precision(ops):
    lengths = [(500, 16)]
    for size in (1e-30, 1e-6, 1e6, 1e30):
        batch = Batch(lengths, 4, 2, 128, 16, torch.float32, seed=10, spread=size)
        check(ops, batch, causal=False, scale=0.1 / size)


def test_attention_out_rows_of_no_request(ops):
    batch = Batch([(10, 3), (0, 2)], 4, 2, 64, 16, extra_rows=4)
    fresh = batch.run(ops)
    assert torch.count_nonzero(fresh[5:]) == 0 and torch.count_nonzero(fresh[:5]) > 0
    out = torch.full_like(fresh, 7.0)
    assert batch.run(ops, out=out).data_ptr() == out.data_ptr()
    assert torch.equal(out[:5], fresh[:5]) and bool((out[5:] == 7.0).all())
    none = ops.paged_attention(batch.q, batch.k, batch.v, batch.table[:0], batch.context[:0], dev32([0]))
    assert torch.count_nonzero(none) == 0
    assert ops.paged_attention(batch.q[:0], batch.k, batch.v, batch.table, batch.context, dev32([0, 0, 0])).shape[0] == 0


def test_attention_refuses_what_it_cannot_write(ops):
    """An output over the queries (they are read again for some rows) and flags elsewhere."""
    batch = Batch([(30, 5), (7, 2)], 4, 2, 64, 16, torch.float16, seed=25)
    buffer = torch.zeros((2, *batch.q.shape), dtype=torch.float16, device=DEV)
    buffer[0] = batch.q
    batch.q = buffer[0]
    for out in (buffer[0], buffer.flatten()[64:64 + batch.q.numel()].view(batch.q.shape)):
        with pytest.raises(ValueError, match="must not overlap"):
            batch.run(ops, out=out)
    assert torch.equal(batch.run(ops, out=buffer[1]), batch.run(ops))
    with pytest.raises(ValueError, match="flags must be"):
        batch.run(ops, flags=ops.Flags(torch.device("cpu")))


@pytest.mark.parametrize("row_type", TYPES)
@pytest.mark.parametrize("count", [5, 90, 300])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_a_row_does_not_see_never_reaches_it(ops, row_type, count, value):
    window = 40
    batch = Batch([(150, count), (70, 1)], 4, 2, 64, 16, row_type, seed=11)
    want = batch.run(ops, window=window)
    # everything outside the requests' visible keys: stale rows of their pages, other pages
    live = torch.zeros(batch.k.shape[:2], dtype=torch.bool, device=DEV)
    for b, (context, n) in enumerate(batch.lengths):
        for p in range(max(0, context - window + 1), context + n):
            live[batch.table[b, p // 16].long(), p % 16] = True
    k, v = batch.k.clone(), batch.v.clone()
    batch.k[~live], batch.v[~live] = value, value
    assert torch.equal(batch.run(ops, window=window), want)
    # a token's own key: later tokens of its window see it, earlier ones must not
    spot = 150 + count // 2
    batch.k, batch.v = k, v
    batch.v[batch.table[0, spot // 16].long(), spot % 16, 1, 5] = value
    got = batch.run(ops, window=window)
    first = count // 2
    hit = torch.zeros(got.shape, dtype=torch.bool, device=DEV)
    hit[first:min(count, first + window), 2:, 5] = True
    tolerance = 2 * HALF_STEP[row_type] if row_type != torch.float32 else 2.0 ** -18
    clean = ~hit
    assert bool(torch.isfinite(got[clean]).all())
    assert float((got[clean].double() - want[clean].double()).norm() / want[clean].double().norm()) <= 2 * tolerance
    assert not bool(torch.isfinite(got[hit]).any())


def test_pages_of_no_seen_key_may_be_gone(ops):
    batch = Batch([(500, 3), (64, 1)], 4, 2, 64, 16, torch.float16, seed=12)
    want = batch.run(ops, window=50)
    batch.table[0, :(500 - 49) // 16] = -1
    assert torch.equal(batch.run(ops, window=50), want)
    with pytest.raises(ValueError, match="outside the pool"):
        batch.run(ops, window=80)
    batch.table[0, 0] = 10 ** 6
    with pytest.raises(ValueError, match="outside the pool"):
        batch.run(ops)


def test_requests_that_do_not_fit_are_left_out(ops):
    batch = Batch([(40, 3), (20, 5), (33, 2)], 4, 2, 64, 16, torch.bfloat16, seed=13)
    want = batch.run(ops)
    lib = submodule("_lib")

    def flag(**change):
        flags = ops.Flags(DEV)
        args = dict(q=batch.q, k_cache=batch.k, v_cache=batch.v, table=batch.table, context=batch.context,
                    starts=batch.starts, flags=flags)
        args.update(change)
        return ops.paged_attention(**args), int(flags.tensor.item())

    got, value = flag(longest=4)
    assert value == lib.FLAG_BAD_LENGTH
    assert torch.equal(got[:3], want[:3]) and torch.equal(got[8:], want[8:]) and torch.count_nonzero(got[3:8]) == 0
    for context in ([40, -1, 33], [40, 10 ** 6, 33], [40, 2 ** 31 - 1, 33]):
        got, value = flag(context=dev32(context))
        assert value == lib.FLAG_BAD_LENGTH
        assert torch.equal(got[:3], want[:3]) and torch.equal(got[8:], want[8:]) and torch.count_nonzero(got[3:8]) == 0
    got, value = flag(starts=dev32([0, 3, 8, 1000]))
    assert value == lib.FLAG_BAD_LENGTH and torch.equal(got[:8], want[:8]) and torch.count_nonzero(got[8:]) == 0
    got, value = flag(starts=dev32([-5, 3, 8, 10]))
    assert value == lib.FLAG_BAD_LENGTH and torch.equal(got[3:], want[3:])
    got, value = flag(starts=dev32([0, 3, 2, 10]))
    assert value == lib.FLAG_BAD_LENGTH and torch.equal(got[:2], want[:2])


def test_attention_repeats_bit_for_bit(ops):
    for row_type in TYPES:
        batch = Batch([(5000, 16), (10, 1), (300, 200)], 8, 2, 128, 16, row_type, seed=14)
        first = batch.run(ops)
        for _ in range(3):
            assert torch.equal(batch.run(ops), first)


@pytest.mark.parametrize("row_type", TYPES)
@pytest.mark.parametrize("requests, heads, kv_heads, head_dim, counts", [
    (32, 16, 8, 64, (1, 40, 3)), (33, 16, 8, 64, (1, 40, 3)), (40, 24, 8, 128, (0, 1, 17, 100)), (400, 2, 1, 64, (1, 0, 70)),
    (900, 2, 1, 64, (1, 1, 33, 2))])
def test_attention_of_many_requests(ops, row_type, requests, heads, kv_heads, head_dim, counts):
    """Short and long requests side by side, on either side of 32 requests, 256 (request,
    kv head) pairs and a block's threads, where the split of the work takes another way."""
    lengths = [((37 * b) % 211, counts[b % len(counts)]) for b in range(requests)]
    check(ops, Batch(lengths, heads, kv_heads, head_dim, 16, row_type, seed=19))


@pytest.mark.parametrize("row_type", TYPES)
@pytest.mark.parametrize("order", [(0, 1, 2), (0, 2, 1), (1, 0, 2), (1, 2, 0), (2, 0, 1), (2, 1, 0)])
@pytest.mark.parametrize("count", [3, 40])
def test_caches_in_any_order_of_their_axes(ops, row_type, order, count):
    """Pages, slots and heads lie in any order, keys and values in one buffer: the store
    and the attention see the same cache."""
    batch = Batch([(150, count), (9, count)], 6, 2, 64, 16, row_type, seed=20)
    want = batch.run(ops)
    shape = [batch.k.shape[i] for i in order]
    both = torch.zeros((*shape[:2], 2, shape[2], 64), dtype=batch.k.dtype, device=DEV)
    back = [order.index(i) for i in range(3)] + [3]
    k, v = (both[:, :, i].permute(back) for i in range(2))
    rows = batch.k.flatten(0, 1), batch.v.flatten(0, 1)
    ops.paged_store(*rows, torch.arange(rows[0].shape[0], dtype=torch.int32, device=DEV), k, v)
    assert torch.equal(k, batch.k) and torch.equal(v, batch.v)
    batch.k, batch.v = k, v
    assert torch.equal(batch.run(ops), want)


@pytest.mark.parametrize("row_type", TYPES)
def test_longest_bounds_the_requests(ops, row_type):
    """A bound that holds changes no value; a request beyond it is left out, with a flag."""
    lib = submodule("_lib")
    batch = Batch([(70, 5), (300, 90), (20, 1)], 8, 2, 64, 32, row_type, seed=21)
    want, bound = batch.expected()
    for longest in (90, 91, 2 ** 31 - 1, 2 ** 40):
        assert bool(((batch.run(ops, longest=longest).double() - want).abs() <= bound).all())
    for longest in (1, 5, 89):
        flags = ops.Flags(DEV)
        got = batch.run(ops, longest=longest, flags=flags)
        assert int(flags.tensor.item()) == lib.FLAG_BAD_LENGTH
        row = 0
        for _, count in batch.lengths:
            here = slice(row, row + count)
            if count <= longest:
                assert bool(((got[here].double() - want[here]).abs() <= bound[here]).all())
            else:
                assert not got[here].any()
            row += count


@pytest.mark.parametrize("row_type", TYPES)
def test_many_calls_in_a_row_end_alike(ops, row_type):
    """Calls of every kernel queued one behind the other: none runs out of its waits."""
    batches = [Batch([(500, 1000), (0, 900)], 16, 4, 128, 64, row_type, seed=22),
               Batch([(900, 17)] * 9, 16, 4, 64, 16, row_type, seed=23), Batch([(4000, 1)] * 40, 16, 8, 64, 16, row_type, seed=24)]
    flags = ops.Flags(DEV)
    first = [batch.run(ops, flags=flags) for batch in batches]
    for i in range(60):
        for batch, want in zip(batches, first):
            got = batch.run(ops, flags=flags)
            if i % 20 == 19:
                assert torch.equal(got, want)
    flags.check()


def test_calls_on_streams_and_in_graphs_do_not_meet(ops):
    """Two captured graphs replayed at once on their own streams, with lengths changed
    between replays, beside eager calls of the same operators."""
    batches = [Batch([(3000, 16), (700, 4)], 8, 2, 128, 16, torch.float16, seed=s) for s in (15, 16)]
    flags = [ops.Flags(DEV) for _ in batches]
    streams, graphs, outs = [], [], []
    for batch, flag in zip(batches, flags):
        stream = torch.cuda.Stream(DEV)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            batch.run(ops, flags=flag)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(batch.run(ops, flags=flag))
        streams.append(stream)
        graphs.append(graph)
    torch.cuda.synchronize()
    for contexts in ((3000, 700), (17, 690), (2999, 0)):
        for batch in batches:
            batch.context.copy_(dev32(contexts))
            batch.lengths = [(contexts[0], 16), (contexts[1], 4)]
        torch.cuda.synchronize()
        for _ in range(5):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        eager = [batch.run(ops) for batch in batches]
        torch.cuda.synchronize()
        for batch, out, e in zip(batches, outs, eager):
            assert torch.equal(out, e)
            want, bound = batch.expected()
            assert bool(((out.double() - want).abs() <= bound).all())
    for flag in flags:
        flag.check()


def test_long_cache_offsets_pass_32_bits(ops):
    """A pool of more than 2^32 elements, its last pages in use."""
    pages, page, kv_heads, d = 2 ** 17 + 40, 256, 1, 128
    if torch.cuda.mem_get_info(DEV)[0] < 5 * pages * page * kv_heads * d:
        pytest.skip("not enough free memory")
    small = Batch([(700, 5)], 4, 1, d, page, torch.bfloat16, seed=17)
    k = torch.empty((pages, page, kv_heads, d), dtype=torch.bfloat16, device=DEV)
    v = torch.empty_like(k)
    far = dev32([[pages - 1 - i for i in range(small.table.shape[1])]])
    for i in range(3):
        k[pages - 1 - i], v[pages - 1 - i] = small.k[small.table[0, i].long()], small.v[small.table[0, i].long()]
    got = ops.paged_attention(small.q, k, v, far, small.context, small.starts)
    assert torch.equal(got, small.run(ops))
    rows = torch.randn((3, 1, d), device=DEV)
    slots = dev32([pages * page - 1, (pages - 2) * page, 0])
    ops.paged_store(rows, rows, slots, k, v)
    assert torch.equal(k.flatten(0, 1)[slots.long()], rows.to(torch.bfloat16))


# ------------------------------------------------------------------ together


def test_a_batch_served_over_pages_equals_each_request_alone(ops):
    """Plan, store and attend step by step, requests joining, growing and finishing,
    against attention over each request's own contiguous keys."""
    heads, kv_heads, d, page, pool = 8, 2, 128, 16, 40
    g = torch.Generator(device=DEV).manual_seed(18)
    k_cache = torch.zeros((pool, page, kv_heads, d), dtype=torch.float16, device=DEV)
    v_cache = torch.zeros_like(k_cache)
    table = torch.full((3, 12), -1, dtype=torch.int32, device=DEV)
    owned, free, top = dev32([0, 0, 0]), torch.arange(pool, dtype=torch.int32, device=DEV), dev32([pool])
    history = [[torch.zeros((0, kv_heads, d), device=DEV)] * 2 for _ in range(3)]
    lengths = [0, 0, 0]
    steps = [([20, 1, 0], ()), ([1, 1, 70], ()), ([16, 16, 16], ()), ([0, 1, 1], (1,)), ([5, 33, 0], (0,)), ([1, 1, 1], ())]
    for counts, finished in steps:
        for b in finished:
            lengths[b], history[b] = 0, [torch.zeros((0, kv_heads, d), device=DEV)] * 2
        if finished:
            done = [0 if b in finished else lengths[b] for b in range(3)]
            ops.page_plan(dev32(done), dev32([0, 0, 0]), table, owned, free, top, page, 0, pool)
            assert all(int(owned[b]) == 0 for b in finished)
        total = sum(counts)
        q = torch.randn((total, heads, d), generator=g, device=DEV)
        kv = torch.randn((total, 2 * kv_heads, d), generator=g, device=DEV)
        k, v = kv[:, :kv_heads], kv[:, kv_heads:]
        plan = ops.page_plan(dev32(lengths), dev32(counts), table, owned, free, top, page, total, pool)
        ops.paged_store(k, v, plan.slots, k_cache, v_cache)
        got = ops.paged_attention(q, k_cache, v_cache, table, dev32(lengths), plan.starts)
        row = 0
        for b, n in enumerate(counts):
            history[b] = [torch.cat((x, y[row:row + n].half().float())) for x, y in zip(history[b], (k, v))]
            if n:
                keys, values = (x.double().repeat_interleave(heads // kv_heads, 1) for x in history[b])
                s = torch.einsum("thd,shd->hts", q[row:row + n].double(), keys) * d ** -0.5
                late = torch.arange(keys.shape[0], device=DEV) > lengths[b] + torch.arange(n, device=DEV)[:, None]
                want = torch.einsum("hts,shd->thd", torch.softmax(s.masked_fill(late, -math.inf), -1), values)
                assert float((got[row:row + n].double() - want).norm() / want.norm()) <= 2.0 ** -18
            row += n
            lengths[b] += n
        used = sum(-(-n // page) for n in lengths)
        assert int(top) == pool - used
        held = [p for b in range(3) for p in table[b, :int(owned[b])].tolist()] + free[:int(top)].tolist()
        assert sorted(held) == list(range(pool))
