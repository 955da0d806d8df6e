"""Cases of the paged key/value cache: its page plan, its store and the attention that reads it.

Three operators of one serving step over a cache whose rows live in fixed-size pages:

* ``plan``: from the requests' lengths, the pages they need (taken from a stack of
  free pages), the row offset of every request and the position and cache slot of
  every new token;
* ``store``: new key and value rows into their cache slots, rounded to the cache's type;
* ``attend``: softmax attention of every request's new tokens over its cached keys,
  its own new ones among them (they are stored first), with grouped heads, causal or
  over the whole block, optionally within a sliding window.

``run`` computes them in elementary torch operations, or through the package when
``own`` is true.  ``exact`` is the definition in 64 bits, request by request.
"""

import importlib
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
WIDTH = {"fp32": 4, "fp16": 2, "bf16": 2}


def listed():
    return [
        # one draft step of a serving batch: every request plans a block of 16 slots
        dict(name="plan_draft_step", op="plan", requests=32, context=4096, count=16, ragged=False, page=16, spare=0),
        # prompts of very different lengths join a running batch, in a row buffer with room to spare
        dict(name="plan_prompts", op="plan", requests=256, context=8192, count=1024, ragged=True, page=16, spare=777),
        # the draft block's fp32 key and value rows go to the drafter's fp16 cache
        dict(name="store_draft_step", op="store", requests=32, context=4096, count=16, ragged=False, page=16, spare=0,
             kv_heads=8, head_dim=128, rows="fp32", cache="fp16"),
        # ragged prompts of a model with few narrow heads; some rows of the buffer are unused
        dict(name="store_ragged", op="store", requests=37, context=515, count=333, ragged=True, page=8, spare=45,
             kv_heads=5, head_dim=64, rows="fp32", cache="bf16"),
        # a prompt batch at full size
        dict(name="store_prompts", op="store", requests=16, context=0, count=4096, ragged=True, page=64, spare=0,
             kv_heads=8, head_dim=128, rows="bf16", cache="bf16"),
        # the drafter's own block: one request, 16 slots that see each other, 4096 cached positions
        dict(name="draft_block", op="attend", requests=1, context=4096, count=16, ragged=False, page=16, heads=32,
             kv_heads=8, head_dim=128, rows="fp32", cache="fp16", causal=False, window=0),
        # the same block for a serving batch of ragged contexts, in a windowed layer
        dict(name="draft_batch", op="attend", requests=24, context=8192, count=16, ragged=False, page=16, heads=32,
             kv_heads=8, head_dim=128, rows="fp32", cache="fp16", causal=False, window=4096),
        # a target model verifies 16 drafts and the token before them, for every request
        dict(name="verify_batch", op="attend", requests=32, context=4096, count=17, ragged=False, page=32, heads=32,
             kv_heads=8, head_dim=128, rows="fp16", cache="fp16", causal=True, window=0),
        # one token for every request of a large batch
        dict(name="decode_batch", op="attend", requests=64, context=8192, count=1, ragged=False, page=16, heads=32,
             kv_heads=8, head_dim=128, rows="bf16", cache="bf16", causal=True, window=0),
        # one token of one request behind a very long context
        dict(name="decode_long", op="attend", requests=1, context=131071, count=1, ragged=False, page=64, heads=32,
             kv_heads=8, head_dim=128, rows="bf16", cache="bf16", causal=True, window=0),
        # chunks of two long prompts
        dict(name="prompt_chunks", op="attend", requests=2, context=4096, count=2048, ragged=False, page=64, heads=32,
             kv_heads=8, head_dim=128, rows="bf16", cache="bf16", causal=True, window=0),
        # ragged chunks through a sliding-window layer with narrow heads in groups of three
        dict(name="prompt_ragged", op="attend", requests=6, context=2500, count=1501, ragged=True, page=16, heads=12,
             kv_heads=4, head_dim=64, rows="fp16", cache="fp16", causal=True, window=1000),
    ]


def _spread(rng, low, high):
    """A whole number between two, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["plan", "store", "attend", "attend", "attend"])
    page = rng.choice([8, 16, 32, 64, 128])
    if op == "plan":
        return dict(op=op, requests=_spread(rng, 1, 512), context=_spread(rng, 1, 16384), count=_spread(rng, 1, 1024),
                    ragged=rng.random() < 0.7, page=page, spare=rng.choice([0, rng.randrange(1000)]))
    if op == "store":
        count = _spread(rng, 1, 4096)
        return dict(op=op, requests=max(1, min(_spread(rng, 1, 64), 32768 // count)), context=_spread(rng, 1, 2048),
                    count=count, ragged=rng.random() < 0.7, page=page, spare=rng.choice([0, rng.randrange(100)]),
                    kv_heads=rng.choice([1, 2, 3, 4, 5, 8]), head_dim=rng.choice([64, 128]),
                    rows=rng.choice(["fp32", "fp16", "bf16"]), cache=rng.choice(["fp16", "bf16"]))
    kind = rng.choice(["block", "verify", "decode", "chunk"])
    head_dim, kv_heads = rng.choice([64, 128]), rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8])
    rows = "fp32" if kind == "block" else rng.choice(["fp16", "bf16"])
    context = _spread(rng, 100, 8192)
    if kind == "chunk":
        count = _spread(rng, 33, 2048)
        requests = max(1, min(_spread(rng, 1, 8), 4096 // count))
        context = min(context, 4096)
    else:
        count = 1 if kind == "decode" else rng.randrange(2, 18)
        requests = _spread(rng, 1, 48)
    return dict(op=op, requests=requests, context=context, count=count, ragged=rng.random() < 0.5, page=page,
                heads=heads, kv_heads=kv_heads, head_dim=head_dim, rows=rows,
                cache="fp16" if rows == "fp32" else rows, causal=kind != "block",
                window=rng.choice([0, 0, _spread(rng, 1, 4096)]))


def lengths(case):
    """(cached positions, new tokens) of every request: fixed by the case.  Contexts are
    ragged wherever there is more than one request, new tokens where the case says so."""
    rng = random.Random("%(requests)d %(context)d %(count)d %(page)d" % case)
    n, most, count = case["requests"], case["context"], case["count"]
    contexts = [most] if n == 1 else [rng.randint(most // 8, most) for _ in range(n)]
    counts = [rng.randint(1, count) if case["ragged"] else count for _ in range(n)]
    return contexts, counts


def _pages(tokens, page):
    return -(-tokens // page)


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=device).manual_seed(seed)
    page, n = case["page"], case["requests"]
    contexts, counts = lengths(case)
    total = sum(counts)
    context = torch.tensor(contexts, dtype=torch.int32, device=device)
    count = torch.tensor(counts, dtype=torch.int32, device=device)
    owned = (context + page - 1) // page
    needed = (context + count + page - 1) // page
    width = max(_pages(a + b, page) for a, b in zip(contexts, counts)) + 2
    pool = sum(_pages(a + b, page) for a, b in zip(contexts, counts)) + 5
    ids = torch.randperm(pool, generator=g, device=device).to(torch.int32)
    column = torch.arange(width, device=device)
    first = torch.cumsum(needed, 0) - needed
    everything = torch.where(column < needed[:, None],
                             ids[(first[:, None] + column).clamp(max=pool - 1).long()], -1).to(torch.int32)
    state = dict(case=case, context=context, count=count, pool=pool)
    if case["op"] == "plan":
        # the pages of the cached positions are in the table, the others on the free stack
        held = column < owned[:, None]
        state["table"] = torch.where(held, everything, -1).to(torch.int32).contiguous()
        state["owned"] = owned.to(torch.int32)
        spread = torch.ones(pool, dtype=torch.bool, device=device)
        spread[everything[held].long()] = False
        state["free"] = torch.cat((ids[spread[ids.long()]], ids[~spread[ids.long()]]))
        state["top"] = spread.sum().to(torch.int32).reshape(1)
        state["rows"] = total + case["spare"]
        return state
    starts = torch.zeros(n + 1, dtype=torch.int32, device=device)
    starts[1:] = torch.cumsum(count, 0)
    kv_heads, head_dim, cache = case["kv_heads"], case["head_dim"], DTYPES[case["cache"]]
    shape = (pool, page, kv_heads, head_dim)
    state["k_cache"] = torch.randn(shape, generator=g, device=device, dtype=cache)
    state["v_cache"] = torch.randn(shape, generator=g, device=device, dtype=cache)
    width = kv_heads * head_dim
    if case["op"] == "store":
        # key and value rows side by side, as one projection leaves them
        rows = total + case["spare"]
        fused = torch.randn((rows, 2 * width), generator=g, device=device, dtype=DTYPES[case["rows"]])
        state["k"] = fused[:, :width].unflatten(1, (kv_heads, head_dim))
        state["v"] = fused[:, width:].unflatten(1, (kv_heads, head_dim))
        row = torch.arange(rows, device=device)
        request = torch.searchsorted(starts[1:].long(), row, right=True).clamp(max=n - 1)
        position = context[request] + row - starts[request]
        slot = everything[request, (position // page).clamp(max=everything.shape[1] - 1)] * page + position % page
        state["slots"] = torch.where(row < total, slot, -1).to(torch.int32)
        return state
    heads = case["heads"]
    state["q"] = torch.randn((total, heads, head_dim), generator=g, device=device).to(DTYPES[case["rows"]])
    state["table"], state["starts"] = everything, starts
    return state


# ------------------------------------------------------------------ the framework's operators


def _package():
    return importlib.import_module("binary-eagle-decoding_b200")


def _own(state):
    case, ops = state["case"], _package().ops
    if "flags" not in state:
        state["flags"] = ops.Flags(state["context"].device)  # a serving loop keeps one and reads it when it likes
    flags = state["flags"]
    if case["op"] == "plan":
        owned, top = torch.empty_like(state["owned"]), torch.empty_like(state["top"])
        plan = ops.page_plan(state["context"], state["count"], state["table"], state["owned"], state["free"],
                             state["top"], case["page"], state["rows"], state["pool"], owned_out=owned, top_out=top,
                             flags=flags)
        return dict(starts=plan.starts, positions=plan.positions, slots=plan.slots, table=state["table"], owned=owned,
                    top=top)
    if case["op"] == "store":
        ops.paged_store(state["k"], state["v"], state["slots"], state["k_cache"], state["v_cache"], flags=flags)
        return dict(k_cache=state["k_cache"], v_cache=state["v_cache"])
    return ops.paged_attention(state["q"], state["k_cache"], state["v_cache"], state["table"], state["context"],
                               state["starts"], causal=case["causal"], window=case["window"] or None,
                               longest=case["count"], flags=flags)


# ------------------------------------------------------------------ the plain forms


def _plain_plan(s):
    page, rows, n = s["case"]["page"], s["rows"], s["case"]["requests"]
    context, count, owned, table = s["context"].long(), s["count"].long(), s["owned"].long(), s["table"]
    need = (context + count + page - 1) // page
    take = need - owned
    before = torch.cumsum(take, 0) - take
    column = torch.arange(table.shape[1], device=table.device)
    new = (column >= owned[:, None]) & (column < need[:, None])
    at = s["top"] - 1 - (before[:, None] + column - owned[:, None])
    table = torch.where(new, s["free"][at.clamp(0, s["free"].numel() - 1)], table)
    ends = torch.cumsum(count, 0)
    starts = torch.cat((ends.new_zeros(1), ends))
    row = torch.arange(rows, device=table.device)
    request = torch.searchsorted(ends, row, right=True).clamp(max=n - 1)
    position = context[request] + row - starts[request]
    live = row < ends[-1]
    entry = table[request, torch.where(live, position // page, 0)]
    slot = entry.long() * page + position % page
    return dict(starts=starts.to(torch.int32), positions=torch.where(live, position, -1).to(torch.int32),
                slots=torch.where(live, slot, -1).to(torch.int32), table=table, owned=need.to(torch.int32),
                top=(s["top"] - take.sum()).to(torch.int32))


def _plain_store(s):
    live = s["slots"] >= 0
    at = s["slots"][live].long()
    k_rows, v_rows = s["k_cache"].flatten(0, 1), s["v_cache"].flatten(0, 1)
    k_rows[at] = s["k"][live].float().to(k_rows.dtype)
    v_rows[at] = s["v"][live].float().to(v_rows.dtype)
    return dict(k_cache=s["k_cache"], v_cache=s["v_cache"])


def _plain_attend(s):
    case, q = s["case"], s["q"]
    page, n, kv_heads, head_dim = case["page"], case["requests"], case["kv_heads"], case["head_dim"]
    group, most, device = case["heads"] // kv_heads, case["count"], q.device
    context, starts = s["context"].long(), s["starts"].long()
    count = starts[1:] - starts[:-1]
    # every request's rows and keys at one padded length
    slot = torch.arange(most, device=device)
    row = (starts[:-1, None] + slot).clamp(max=q.shape[0] - 1)
    rows = q[row].float().view(n, most, kv_heads, group, head_dim)
    table = s["table"].clamp(min=0).long()
    keys = s["k_cache"][table].flatten(1, 2).float()
    values = s["v_cache"][table].flatten(1, 2).float()
    scores = torch.einsum("btkgd,bskd->bkgts", rows, keys) * (head_dim ** -0.5)
    position = (context[:, None] + slot)[:, :, None]
    key = torch.arange(keys.shape[1], device=device)
    seen = key < (context + count)[:, None, None]
    if case["causal"]:
        seen = seen & (key <= position)
    if case["window"]:
        seen = seen & ((position - key).abs() < case["window"])
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    weight = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e30))
    out = torch.einsum("bkgts,bskd->btkgd", weight, values)
    out = out / weight.sum(-1).clamp(min=1e-30).permute(0, 3, 1, 2)[..., None]
    index = torch.arange(q.shape[0], device=device)
    request = torch.searchsorted(starts[1:], index, right=True)
    return out[request, index - starts[request]].reshape(q.shape).to(q.dtype)


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return _plain_plan(state) if op == "plan" else _plain_store(state) if op == "store" else _plain_attend(state)


# ------------------------------------------------------------------ work and the definition in 64 bits


def _visible(case):
    """(keys that some new token of a request sees, pairs of new token and key that meet), over all requests."""
    keys = pairs = 0
    for context, count in zip(*lengths(case)):
        low = 0
        for t in range(count):
            position, window = context + t, case["window"] or context + count
            first = max(0, position - window + 1)
            last = position if case["causal"] else min(context + count - 1, position + window - 1)
            low = first if t == 0 else low
            pairs += last - first + 1
        keys += last - low + 1
    return keys, pairs


def work(case):
    contexts, counts = lengths(case)
    n, total, page = case["requests"], sum(counts), case["page"]
    if case["op"] == "plan":
        new = sum(_pages(a + b, page) - _pages(a, page) for a, b in zip(contexts, counts))
        old = sum(1 for a in contexts if a % page)  # half-filled pages that new tokens go on with
        # lengths and page counts in, row offsets and page counts out, taken pages in and out, two words a row
        return {"bytes": 4 * (3 * n + 2 * n + 2 * new + old + 2 * (total + case["spare"])), "flops": 0}
    if case["op"] == "store":
        values = 2 * total * case["kv_heads"] * case["head_dim"]
        return {"bytes": values * (WIDTH[case["rows"]] + WIDTH[case["cache"]]) + 4 * (total + case["spare"]), "flops": 0}
    keys, pairs = _visible(case)
    rows = 2 * total * case["heads"] * case["head_dim"] * WIDTH[case["rows"]]
    cache = 2 * keys * case["kv_heads"] * case["head_dim"] * WIDTH[case["cache"]]
    table = 4 * sum(_pages(a + b, page) for a, b in zip(contexts, counts))
    return {"bytes": rows + cache + table + 8 * n, "flops": 4 * pairs * case["heads"] * case["head_dim"]}


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    contexts, counts = lengths(case)
    if case["op"] == "store":
        answer = {}
        for name, rows in (("k_cache", s["k"]), ("v_cache", s["v"])):
            cache = s[name].double()
            flat = cache.view(-1, case["kv_heads"], case["head_dim"])
            for r0 in range(0, sum(counts), 4096):
                at = s["slots"][r0:r0 + 4096]
                flat.index_copy_(0, at[at >= 0].long(), rows[r0:r0 + 4096][at >= 0].double())
            answer[name] = cache
        return answer
    group, page, head_dim = case["heads"] // case["kv_heads"], case["page"], case["head_dim"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    row = 0
    for b, (context, count) in enumerate(zip(contexts, counts)):
        length = context + count
        pages = s["table"][b, :_pages(length, page)].long()
        k = s["k_cache"].index_select(0, pages).reshape(-1, case["kv_heads"], head_dim)[:length]
        v = s["v_cache"].index_select(0, pages).reshape(-1, case["kv_heads"], head_dim)[:length]
        gap = (context + torch.arange(count, device=out.device))[:, None] - torch.arange(length, device=out.device)[None]
        hidden = torch.zeros_like(gap, dtype=torch.bool)
        if case["causal"]:
            hidden |= gap < 0
        if case["window"]:
            hidden |= gap.abs() >= case["window"]
        for h in range(case["heads"]):
            x = s["q"][row:row + count, h].double()
            logit = x @ k[:, h // group].double().T / math.sqrt(head_dim)
            logit[hidden] = -math.inf
            out[row:row + count, h] = torch.softmax(logit, -1) @ v[:, h // group].double()
        row += count
    return out
