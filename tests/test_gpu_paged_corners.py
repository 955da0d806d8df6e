"""Corners of the paged cache on the GPU: small weights beside a large one, values at the
types' limits, values that are not finite, lengths that do not fit (needs a B200)."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from conftest import package, submodule
from test_gpu_paged import DEV, HALF_STEP, TYPES, Batch, check, dev32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    return package().ops


# ------------------------------------------------------------------ small weights


def exact(batch, scale=None, window=None):
    """Causal attention in 64 bits: (output, sum of weight x |v|, largest weight, sum of |q k|
    x scale at its largest), per row and head."""
    scale = batch.head_dim ** -0.5 if scale is None else scale
    group, row = batch.heads // batch.kv_heads, 0
    out = torch.zeros(batch.q.shape, dtype=torch.float64, device=DEV)
    size, peak, reach = torch.zeros_like(out), torch.zeros_like(out), torch.zeros_like(out)
    for b, (context, count) in enumerate(batch.lengths):
        at = torch.arange(context + count, device=DEV)
        page = batch.table[b, at // batch.page].long()
        k, v = batch.k[page, at % batch.page].double(), batch.v[page, at % batch.page].double()
        gap = (context + torch.arange(count, device=DEV))[:, None] - at
        hidden = (gap < 0) | (gap >= (window or 2 ** 40))
        here = slice(row, row + count)
        for h in range(batch.heads):
            q, kh, vh = batch.q[here, h].double(), k[:, h // group], v[:, h // group]
            p = torch.softmax((q @ kh.T * scale).masked_fill(hidden, -math.inf), -1)
            out[here, h], size[here, h] = p @ vh, p @ vh.abs()
            peak[here, h] = p.amax(-1, keepdim=True)
            reach[here, h] = (q.abs() @ kh.abs().T * abs(scale)).masked_fill(hidden, 0.0).amax(-1, keepdim=True)
        row += count
    return out, size, peak, reach


def small_weights_bound(batch, out, size, peak, reach):
    """Error of the weights and sums.  The exponent: head_dim products added in fp32, the scale,
    log2 e and the maximum's subtraction rounded, ex2 within 2^-22, and for fp32 rows the
    halves' 2^-21 each of a product.  A weight's rounding: 2^-21 for fp32 rows, half a step of
    the cache's type for others; where that type is fp16, at most half its smallest step, 2^-25,
    of weights scaled so that the largest is 2^11 or more (fp32 rows 2^15): 2^-36 (2^-40) of the
    largest, a key.
    Sums of length / 16 + 64 steps in fp32, and the output's rounding."""
    u, d, f32 = HALF_STEP[batch.q.dtype], batch.head_dim, batch.q.dtype == torch.float32
    length = max(a + b for a, b in batch.lengths)
    delta = (d + 12) * 2.0 ** -23 * reach + 2.0 ** -21 + (2.0 ** -20 * reach if f32 else 0.0)
    sums = 2 * (length / 16 + 64) * 2.0 ** -23
    step = {torch.float32: 2.0 ** -40, torch.float16: 2.0 ** -36, torch.bfloat16: 0.0}[batch.q.dtype]
    lost = length * step * peak * batch.v.abs().amax().double()
    return u * out.abs() + size * ((2.0 ** -21 if f32 else u) + 2 * delta + sums) * 1.1 + lost


@pytest.mark.parametrize("row_type", TYPES)
@pytest.mark.parametrize("requests, keys, count, head_dim", [(160, 8192, 1, 128), (160, 8192, 1, 64), (80, 16384, 20, 128),
                                                             (80, 16384, 40, 64), (2, 100_000, 20, 128)])
@pytest.mark.parametrize("nats", [11.0, 15.0, 18.5])
def test_many_small_weights_beside_a_large_one(ops, row_type, requests, keys, count, head_dim, nats):
    """A first key that draws nearly all of a row's weight and holds little, the others each
    `nats` below it: together they are the output.  With 80 and more pairs an item
    stays whole in one CTA and one running maximum."""
    kv_heads = 2 if requests == 80 else 1
    batch = Batch([(keys - count, count)] * requests, kv_heads, kv_heads, head_dim, 64, row_type, seed=int(nats))
    q = batch.q.clone() * 0.05
    q[..., 0] = 8.0
    batch.q = q
    batch.k.mul_(0.05)
    batch.k[..., 0] = 0.0
    batch.v.add_(0.5)
    first = batch.table[:, 0].long()
    batch.k[first, 0] = 0.0
    batch.k[first, 0, :, 0] = nats * head_dim ** 0.5 / 8.0
    batch.v[first, 0] = 0.0
    want, *how = exact(batch)
    err = (batch.run(ops).double() - want).abs()
    bound = small_weights_bound(batch, want, *how)
    assert bool((err <= bound).all()), (float((err / bound).max()), float(err.norm() / want.norm()))


@pytest.mark.parametrize("count, head_dim", [(1, 128), (16, 128), (70, 64)])
@pytest.mark.parametrize("big", [1e3, 1e5, 1e6, 3e38])
def test_fp32_rows_with_one_large_value(ops, count, head_dim, big):
    """The keys hold nothing where the rows are large, so the rows' small values decide.  A value's
    halves are off by 2^-22 of it or by half of fp16's smallest step, at the row's largest value
    scaled to 2^14 or more: 2^-25 / 2^14 of that value, on each of the row's products."""
    batch = Batch([(300, count), (40, 2)], 4, 2, head_dim, 16, torch.float32, seed=31)
    q = batch.q.clone()
    q[..., 5] = big
    batch.q = q
    batch.k[..., 5] = 0.0
    want, size, peak, reach = exact(batch)
    err = (batch.run(ops).double() - want).abs()
    halves = 2.0 ** -39 * big * batch.k.double().abs().sum(-1).amax() * head_dim ** -0.5
    if big > 1e30:  # their products are all lost: only the mean over the keys of flat weights is left
        assert bool(torch.isfinite(err).all())
    else:
        assert bool((err <= small_weights_bound(batch, want, size, peak, reach) + 2.2 * halves * size).all())


# ------------------------------------------------------------------ values that are not finite


def matches_exact(ops, batch, **how):
    """Finite where the definition is, within the bound, and not a number where it is not."""
    got, (want, *rest) = batch.run(ops, **how).double(), exact(batch)
    real = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isfinite(got), real)
    bound = torch.nan_to_num(small_weights_bound(batch, *(torch.nan_to_num(x, posinf=1.0, neginf=1.0) for x in (want, *rest))))
    assert bool(((got - want).abs() <= bound)[real].all())
    return real


@pytest.mark.parametrize("row_type", TYPES)
@pytest.mark.parametrize("count, head_dim", [(1, 128), (5, 64), (20, 128), (90, 64), (300, 128)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_keys_that_are_not_finite(ops, row_type, count, head_dim, value):
    """A key of a later token must not reach earlier ones; where it is seen, a score of -inf
    only removes the key and one of +inf or NaN leaves no number."""
    batch = Batch([(150, count), (0, 1), (70, 2)], 4, 2, head_dim, 16, row_type, seed=41)
    spot = 150 + count // 2
    batch.k[batch.table[0, spot // 16].long(), spot % 16, 1, 3] = value
    batch.k[batch.table[2, 0].long(), 7, 0, 0] = value  # key 7 of the last request
    real = matches_exact(ops, batch)
    assert bool(real[:count // 2].all()) and bool(real[:, :2][:count + 1].all())
    if math.isnan(value):
        assert not bool(real[count // 2:count, 2:].any())


@pytest.mark.parametrize("row_type", TYPES)
@pytest.mark.parametrize("count, head_dim", [(1, 128), (3, 64), (20, 128), (90, 64)])
def test_a_row_whose_scores_are_all_minus_infinity_is_not_a_number(ops, row_type, count, head_dim):
    """As the softmax of its definition is, split over CTAs or not."""
    batch = Batch([(0, count), (700, 2)], 4, 2, head_dim, 16, row_type, seed=42)
    q = batch.q.clone()
    q[:count, :, 0] = 2.0
    batch.q = q
    length = torch.arange(count, device=DEV)
    batch.k[batch.table[0, length // 16].long(), length % 16, 0, 0] = -math.inf
    real = matches_exact(ops, batch)
    assert not bool(real[:count, :2].any()) and bool(real[:count, 2:].all()) and bool(real[count:].all())


@pytest.mark.parametrize("row_type, count, keys", [(torch.float32, 64, 250_000), (torch.float16, 256, 200_000),
                                                   (torch.bfloat16, 256, 200_000), (torch.float16, 3, 20_000)])
def test_a_request_that_is_not_finite_spoils_no_other(ops, row_type, count, keys):
    """All rows of a request are not numbers, over more keys than a wait of the kernels lasts when
    they are done one by one; the requests share their pages and all but those rows stay as they were."""
    requests, page = 160, 256
    batch = Batch([(keys - count, count)], 1, 1, 64, page, row_type, seed=43)
    table = batch.table.expand(requests, -1).contiguous()
    context = batch.context.expand(requests).contiguous()
    starts = torch.arange(requests + 1, dtype=torch.int32, device=DEV) * count
    q = torch.randn((requests * count, 1, 64), device=DEV).to(row_type)
    flags = ops.Flags(DEV)
    want = ops.paged_attention(q, batch.k, batch.v, table, context, starts, flags=flags)
    q[:count, 0, 9] = math.nan  # this request is whole in the first CTA
    got = ops.paged_attention(q, batch.k, batch.v, table, context, starts, flags=flags)
    flags.check()
    assert torch.equal(got[count:], want[count:])
    assert bool(torch.isnan(got[:count]).all()) and bool(torch.isfinite(want).all())


# ------------------------------------------------------------------ lengths that do not fit


@pytest.mark.parametrize("row_type", TYPES)
@pytest.mark.parametrize("heads_each, context", [(1, 20), (1, 3000), (20, 300)])
@pytest.mark.parametrize("starts", [[0, 1000, 8, 10], [0, 3, 1000, 8, 10, 5], [9, 20, 3, 5], [-4, 2, 1000, 6, 7], [4, 2, 10, 10, 3],
                                    [0, 3, 3, 10, 6]])
def test_refused_rows_do_not_touch_those_of_others(ops, row_type, heads_each, context, starts):
    """Row offsets that do not ascend: each request that fits has its rows, whole items and
    joined ones alike, and all rows that no such request claims are zero or stay."""
    lib, rows, requests = submodule("_lib"), 10, len(starts) - 1
    batch = Batch([(context, rows)] * requests, 2 * heads_each, 2, 64, 16, row_type, seed=51)
    q = batch.q[:rows]
    out = torch.full((rows, 2 * heads_each, 64), 7.0, dtype=row_type, device=DEV)
    want, claims = torch.zeros_like(out), [0] * rows
    for b in range(requests):
        s, e = starts[b], starts[b + 1]
        if 0 <= s <= e <= rows:
            alone = ops.paged_attention(q[s:e], batch.k, batch.v, batch.table[b:b + 1], batch.context[:1], dev32([0, e - s]))
            want[s:e] = alone
            for r in range(s, e):
                claims[r] += 1
    assert max(claims) == 1
    args = (q, batch.k, batch.v, batch.table, batch.context, dev32(starts))
    free = torch.tensor(claims, device=DEV) == 0
    u = HALF_STEP[row_type]
    for _ in range(20):
        flags = ops.Flags(DEV)
        got, kept = ops.paged_attention(*args, flags=flags), ops.paged_attention(*args, out=out.clone(), flags=flags)
        assert int(flags.tensor.item()) == lib.FLAG_BAD_LENGTH
        assert not got[free].any() and bool((kept[free] == 7.0).all())
        # another batch splits the work elsewhere: each side is within a rounding of P, O and the output
        for x in (got, kept):
            assert float((x[~free].double() - want[~free].double()).norm()) <= 4 * max(u, 2.0 ** -20) * float(want.double().norm())


# ------------------------------------------------------------------ plan


@pytest.mark.parametrize("page", [-1, 6, 2 ** 31 - 1, -2 ** 31])
def test_plan_reports_a_bad_page_that_is_given_back(ops, page):
    """By the step that gives it back, not only by one that would take it."""
    lib, flags = submodule("_lib"), ops.Flags(DEV)
    table, owned, free, top = dev32([[0, page, -1], [1, 2, -1]]), dev32([2, 2]), dev32([3, 4, 5, -9]), dev32([3])
    ops.page_plan(dev32([0, 20]), dev32([0, 4]), table, owned, free, top, 16, 4, 6, flags=flags)
    assert int(flags.tensor.item()) == lib.FLAG_BAD_LENGTH | lib.FLAG_BAD_PAGE  # the stack has room for one of the two
    flags = ops.Flags(DEV)
    table, owned, free, top = dev32([[0, page, -1], [1, 2, -1]]), dev32([2, 2]), dev32([3, 4, 5, -9, -9]), dev32([3])
    ops.page_plan(dev32([0, 20]), dev32([0, 4]), table, owned, free, top, 16, 4, 6, flags=flags)
    assert int(flags.tensor.item()) == lib.FLAG_BAD_PAGE
    assert table.tolist() == [[-1, -1, -1], [1, 2, -1]] and owned.tolist() == [0, 2] and top.tolist() == [5]
    assert free.tolist() == [3, 4, 5, 0, page]


def test_plan_serves_no_request_behind_one_that_does_not_fit(ops):
    """Five and one pages lacking, three free: neither is served, whichever has its pages there;
    in the other order the small one is.  A request behind them that lacks none has its rows."""
    lib = submodule("_lib")

    def step(counts):
        flags, table, owned = ops.Flags(DEV), torch.full((3, 6), -1, dtype=torch.int32, device=DEV), dev32([0, 0, 1])
        table[2, 0] = 3
        top = dev32([3])
        plan = ops.page_plan(dev32([0, 0, 2]), dev32([*counts, 4]), table, owned, dev32([0, 1, 2, 9]), top, 16, sum(counts) + 4,
                             10, flags=flags)
        assert int(flags.tensor.item()) == lib.FLAG_NO_PAGES and plan.starts.tolist() == [0, counts[0], sum(counts), sum(counts) + 4]
        return plan.slots.tolist(), owned.tolist(), top.tolist()

    last = [3 * 16 + 2 + t for t in range(4)]
    assert step((80, 16)) == ([-1] * 96 + last, [0, 0, 1], [3])
    assert step((16, 80)) == ([2 * 16 + t for t in range(16)] + [-1] * 80 + last, [1, 0, 1], [2])


# ------------------------------------------------------------------ the types' ends


@pytest.mark.parametrize("requests, count, head_dim", [(3, 1, 128), (3, 200, 64), (40, 64, 128), (40, 64, 64), (160, 3, 128)])
@pytest.mark.parametrize("value", [65504.0, -65504.0])
def test_fp16_outputs_of_the_largest_values_are_finite(ops, requests, count, head_dim, value):
    """An output lies between the values that it weights.  Every weight but the first key's is
    one quarter x (1 + 1.2 x 2^-11), which fp16 rounds up by 0.8 x 2^-11: that must not carry
    the output past the type's largest number."""
    batch = Batch([(900, count)] * requests, 32, 8, head_dim, 16, torch.float16, seed=61)
    batch.q = torch.zeros_like(batch.q)
    batch.q[..., 0] = 1.0
    batch.k.zero_()
    batch.k[batch.table[:, 0].long(), 0, :, 0] = 1.0
    batch.v.fill_(value)
    got = batch.run(ops, scale=math.log(4.0 / (1 + 1.2 * 2.0 ** -11))).float()
    assert bool(((got - value).abs() <= 65504.0 * 2.0 ** -10).all())  # (an infinity is not)


@pytest.mark.parametrize("row_type", TYPES)
@pytest.mark.parametrize("count, head_dim", [(1, 64), (40, 128)])
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-40, 1e-38, -1e-38])
def test_scales_near_zero(ops, row_type, count, head_dim, scale):
    """Flat weights whatever the scores, or the scores times a scale below the normal numbers."""
    batch = Batch([(90, count), (0, 3)], 4, 2, head_dim, 16, row_type, seed=62)
    if row_type == torch.bfloat16:  # scores of about 1e36
        batch.q, batch.k = batch.q * 1e18, batch.k.mul_(1e17)
    want, *how = exact(batch, scale=scale)
    err = (batch.run(ops, scale=scale).double() - want).abs()
    # the scale itself is held to 2^-150, and 0 as 2^-149; the scores are below 1e38
    lost = 2.0 ** -149 * 1e38 if row_type == torch.bfloat16 else 0.0
    assert bool((err <= small_weights_bound(batch, want, *how) + 2.2 * lost * how[0]).all())


def test_windows_beyond_every_position_are_none(ops):
    batch = Batch([(90, 20), (3, 1)], 4, 2, 64, 16, torch.float16, seed=63)
    want = batch.run(ops)
    for window in (110, 2 ** 31 - 1, 2 ** 31, 2 ** 40, 2 ** 80):
        assert torch.equal(batch.run(ops, window=window), want)


# ------------------------------------------------------------------ memory in common


def test_attention_refuses_an_output_over_what_it_reads(ops):
    batch = Batch([(30, 5), (7, 2)], 4, 2, 64, 16, torch.float16, seed=71)
    for cache in (batch.k, batch.v):
        out = cache.flatten()[64:64 + batch.q.numel()].view(batch.q.shape)
        with pytest.raises(ValueError, match="must not overlap the caches"):
            batch.run(ops, out=out)
    # behind one another in a buffer is fine
    buffer = torch.zeros(batch.k.numel() + batch.q.numel(), dtype=torch.float16, device=DEV)
    buffer[:batch.k.numel()] = batch.k.flatten()
    want = batch.run(ops)
    batch.k = buffer[:batch.k.numel()].view(batch.k.shape)
    assert torch.equal(batch.run(ops, out=buffer[batch.k.numel():].view(batch.q.shape)), want)


def test_store_refuses_caches_that_share_elements(ops):
    cache, rows, slots = torch.zeros((3, 16, 2, 64), dtype=torch.float16, device=DEV), torch.ones((5, 2, 64), device=DEV), dev32(range(5))
    one = torch.zeros((1, 16, 2, 64), dtype=torch.float16, device=DEV)
    for k, v in ((cache, cache), (one.expand(3, -1, -1, -1), cache), (cache, cache[:, :, :1].expand(-1, -1, 2, -1))):
        with pytest.raises(ValueError, match="share elements"):
            ops.paged_store(rows, rows, slots, k, v)
    assert not cache.any() and not one.any()


def test_a_page_is_copied_within_the_caches(ops):
    """Rows that lie in the caches themselves, into slots of other pages."""
    g = torch.Generator(device=DEV).manual_seed(72)
    both = torch.randn((6, 16, 2, 3, 64), generator=g, device=DEV).half()
    k, v = both[:, :, 0], both[:, :, 1]
    want = both.clone()
    want[5], want[2] = both[1], both[4]
    for source, target in ((1, 5), (4, 2)):
        ops.paged_store(k[source], v[source], torch.arange(target * 16, target * 16 + 16, dtype=torch.int32, device=DEV), k, v)
    assert torch.equal(both, want)


# ------------------------------------------------------------------ launches


def test_launches_are_counted_as_made(ops):
    """Against the nodes of a captured graph; none for calls without rows."""
    lib, runtime = submodule("_lib"), ctypes.CDLL("libcudart.so.12")
    flags, pages, no_rows = ops.Flags(DEV), dev32([[0, 1, 2, 3]]), dev32([0, 0])

    def counted(call):
        call()
        torch.cuda.synchronize()
        graph, nodes = torch.cuda.CUDAGraph(keep_graph=True), ctypes.c_size_t()
        before = lib.launches
        with torch.cuda.graph(graph):
            call()
        assert runtime.cudaGraphGetNodes(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(nodes)) == 0
        made = nodes.value
        assert made == lib.launches - before
        return made

    for row_type, lengths, kv_heads, want in ((torch.float32, [(30, 80)] * 70, 4, 2), (torch.float16, [(30, 3)] * 70, 4, 2),
                                              (torch.float16, [(30, 80)] * 64, 4, 2), (torch.float16, [(30, 80)] * 65, 4, 3)):
        batch = Batch(lengths, 8, kv_heads, 64, 16, row_type, seed=81)
        assert counted(lambda: batch.run(ops, longest=lengths[0][1], flags=flags)) == want
    none = batch.q[:0]
    assert counted(lambda: ops.paged_attention(none, batch.k, batch.v, batch.table[:1], batch.context[:1], no_rows, flags=flags)) == 0
    k = torch.zeros((3, 4, 64), device=DEV)
    slots = dev32([0, 1, 2])
    assert counted(lambda: ops.paged_store(k, k, slots, batch.k, batch.v, flags=flags)) == 1
    assert counted(lambda: ops.paged_store(k[:0], k[:0], slots[:0], batch.k, batch.v, flags=flags)) == 0
    one, zero, free, top = dev32([1]), dev32([0]), dev32([0, 1]), dev32([2])
    for rows, want in ((0, 1), (4096, 1), (4097, 2)):
        assert counted(lambda: ops.page_plan(one, zero, pages, one, free, top, 16, rows, 4, flags=flags)) == want


# ------------------------------------------------------------------ long rows, captured steps


@pytest.mark.parametrize("row_type", TYPES)
@pytest.mark.parametrize("count, head_dim", [(1, 128), (20, 64), (40, 128), (300, 128)])
@pytest.mark.parametrize("rate", [0.001, 0.005, -0.005, 0.03])
def test_scores_that_grow_along_the_keys(ops, row_type, count, head_dim, rate):
    """Each tile raises the running maximum, by less and by more than what is left unscaled."""
    if row_type == torch.float32 and rate == 0.03:
        rate = 0.01  # scores of 20, whose fp32 rounding the norm's limit allows for
    lengths = [(1700, count), (900, 2)]
    batch = Batch(lengths, 4, 2, head_dim, 16, row_type, seed=91)
    q = batch.q.clone()
    q[..., 0] = 4.0
    batch.q = q
    for b, (context, n) in enumerate(lengths):
        at = torch.arange(context + n, device=DEV)
        batch.k[batch.table[b, at // 16].long(), at % 16, :, 0] = (at * rate * head_dim ** 0.5 / 4)[:, None].to(batch.k.dtype)
    check(ops, batch)
    check(ops, batch, causal=False, window=500)


def test_a_captured_step_replays_with_new_lengths(ops):
    """Plan, store and attention in one graph over buffers of fixed size, replayed while requests
    grow, pause and finish, against the same step made eagerly on copies."""
    heads, kv_heads, d, page, pool, rows, requests = 8, 2, 64, 16, 64, 40, 4
    g = torch.Generator(device=DEV).manual_seed(92)
    flags = ops.Flags(DEV)

    def state():
        return dict(table=torch.full((requests, 16), -1, dtype=torch.int32, device=DEV), owned=dev32([0] * requests),
                    free=torch.arange(pool, dtype=torch.int32, device=DEV), top=dev32([pool]),
                    k=torch.zeros((pool, page, kv_heads, d), dtype=torch.float16, device=DEV),
                    v=torch.zeros((pool, page, kv_heads, d), dtype=torch.float16, device=DEV))

    context, count = dev32([0] * requests), dev32([0] * requests)
    q = torch.zeros((rows, heads, d), dtype=torch.float16, device=DEV)
    kv = torch.zeros((rows, 2 * kv_heads, d), dtype=torch.float16, device=DEV)

    def step(s):
        plan = ops.page_plan(context, count, s["table"], s["owned"], s["free"], s["top"], page, rows, pool, flags=flags)
        ops.paged_store(kv[:, :kv_heads], kv[:, kv_heads:], plan.slots, s["k"], s["v"], flags=flags)
        out = ops.paged_attention(q, s["k"], s["v"], s["table"], context, plan.starts, flags=flags)
        return plan, out

    mine, other = state(), state()
    step(other)  # (no rows yet)
    stream = torch.cuda.Stream(DEV)
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        plan, out = step(mine)
    lengths = [0] * requests
    for counts, finished in (([20, 1, 0, 19], ()), ([1, 1, 30, 8], ()), ([16, 0, 1, 1], (1,)), ([5, 33, 1, 1], ()),
                             ([0, 1, 38, 1], (0, 3)), ([1, 1, 1, 1], ()), ([10, 10, 10, 10], ())):
        for b in finished:
            lengths[b] = 0
        context.copy_(dev32(lengths))
        count.copy_(dev32(counts))
        q.copy_(torch.randn(q.shape, generator=g, device=DEV))
        kv.copy_(torch.randn(kv.shape, generator=g, device=DEV))
        torch.cuda.synchronize()
        graph.replay()
        want_plan, want = step(other)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(plan, want_plan)) and torch.equal(out, want)
        assert all(torch.equal(mine[name], other[name]) for name in mine)
        assert not out[sum(counts):].any()
        lengths = [a + b for a, b in zip(lengths, counts)]
        assert int(mine["top"]) == pool - sum(-(-n // page) for n in lengths)
    flags.check()
