"""Measured cases of the paged 8-bit cache: its plan (block tables and slot maps from request lengths), the append that
quantises new keys and values into it, and attention over it.

The cache holds e4m3 codes [pages, page size, kv heads, d] for keys and for values, and one f32 scale for each page and
kv head. `run` computes the operators in elementary torch operations, or, with `own`, through `krn_b200.ops`."""

import math

import numpy as np
import torch

own = False

E4M3_MAX = 448.0
LEAST_EXPONENT = -100  # of a page's power-of-two scale


def listed():
    return [
        # the step of a small server: every request brings one token
        dict(name="plan, 16 requests", op="plan", batch=16, page=64, context=8192, prompts=0, chunk=1, done=0),
        # a large server's step: most requests decode, two dozen prompts arrive in chunks, some requests are finished
        dict(name="plan, 1000 requests mixed", op="plan", batch=1000, page=16, context=32768, prompts=24, chunk=2048, done=40),
        # one token each of 64 requests, most of them inside a page that holds tokens already
        dict(name="append, 64 tokens", op="append", dtype="bf16", batch=64, new=1, rows=64, page=64, heads=8, d=128, context=8192),
        # odd chunks of prompts into half-filled small pages, f16, small heads
        dict(name="append, odd chunks f16", op="append", dtype="f16", batch=7, new=301, rows=2107, page=16, heads=3, d=64, context=1000),
        # a full prompt step: 8 chunks of up to 2048 tokens
        dict(name="append, 16384 rows", op="append", dtype="bf16", batch=8, new=2048, rows=16384, page=64, heads=8, d=128, context=4096),
        # the first tokens of one short chat: latency
        dict(name="attention, one short", op="attention", dtype="bf16", batch=1, new=1, prompts=0, chunk=0, page=64, heads=8, group=4,
             d=128, low=100, high=500),
        # the decode mix of the benchmark: 64 sequences, 1024 to 8192 tokens each
        dict(name="attention, 64 decode", op="attention", dtype="bf16", batch=64, new=1, prompts=0, chunk=0, page=64, heads=8, group=4,
             d=128, low=1024, high=8192),
        # one very long document
        dict(name="attention, one long", op="attention", dtype="bf16", batch=1, new=1, prompts=0, chunk=0, page=128, heads=8, group=4,
             d=128, low=120001, high=131072),
        # drafted tokens are verified, up to four a request; f16, small heads and small pages
        dict(name="attention, verify f16", op="attention", dtype="f16", batch=24, new=4, prompts=0, chunk=0, page=16, heads=2, group=8,
             d=64, low=5, high=4096),
        # decode requests and chunks of prompts in one batch
        dict(name="attention, mixed", op="attention", dtype="bf16", batch=40, new=1, prompts=4, chunk=512, page=32, heads=4, group=4,
             d=128, low=500, high=4096),
        # chunks of long prompts over what the cache holds of them
        dict(name="attention, chunks", op="attention", dtype="bf16", batch=3, new=0, prompts=3, chunk=1500, page=64, heads=8, group=4,
             d=128, low=6000, high=8192),
        # a whole prompt
        dict(name="attention, prompt of 8192", op="attention", dtype="bf16", batch=1, new=0, prompts=1, chunk=8192, page=64, heads=8,
             group=4, d=128, low=8192, high=8192),
    ]


def _log(rng, low, high):
    """An integer spread evenly over the logarithm of its range."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1))) - 0.5))))


def draw(rng):
    op = rng.choice(["plan", "append", "attention", "attention"])
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        batch = _log(rng, 1, 1000)
        prompts = rng.randint(0, min(batch, 24))
        return dict(op=op, batch=batch, page=page, context=_log(rng, 100, 32768), prompts=prompts,
                    chunk=_log(rng, 1, 2048), done=rng.randint(0, (batch - prompts) // 8))
    dtype, d = rng.choice(["bf16", "bf16", "f16"]), rng.choice([64, 128, 128])
    if op == "append":
        heads = rng.randint(1, 8)
        if rng.random() < 0.5:  # one or a few tokens a request
            batch, new = _log(rng, 1, 256), rng.randint(1, 4)
        else:
            batch, new = rng.randint(1, 8), _log(rng, 5, 2048)
        return dict(op=op, dtype=dtype, batch=batch, new=new, rows=batch * new + rng.choice([0, 0, rng.randint(1, 64)]), page=page,
                    heads=heads, d=d, context=_log(rng, 1, 4096))
    kind = rng.choice(["decode", "decode", "verify", "mixed", "prompt"])
    heads, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 4, 5, 6, 8])
    case = dict(op=op, dtype=dtype, batch=1, new=1, prompts=0, chunk=0, page=page, heads=heads, group=group, d=d, low=1, high=1)
    if kind in ("decode", "verify"):
        case["batch"] = _log(rng, 1, 64)
        case["high"] = _log(rng, 16, min(131072, 250000 // case["batch"]))
        case["new"] = 1 if kind == "decode" else rng.randint(2, 8)
    elif kind == "mixed":
        case["batch"] = _log(rng, 2, 32)
        case["prompts"], case["chunk"] = rng.randint(1, 2), _log(rng, 10, 512)
        case["high"] = _log(rng, case["chunk"], 4096)
    else:
        case["batch"] = case["prompts"] = rng.randint(1, 3)
        case["chunk"], case["new"] = _log(rng, 30, 1000), 0
        case["high"] = case["chunk"] + _log(rng, 1, 4000)
    case["low"] = rng.randint(1, case["high"])
    return case


# ---- lengths and inputs ----------------------------------------------------------------------------------------------


def _chance(rng, low, high, size):
    return rng.integers(low, high + 1, size)


def _table(rng, pages_of, width, spare):
    """A page table over a shuffled pool, entries past a request's pages left at -1; the pages nobody holds."""
    total = int(pages_of.sum())
    order = rng.permutation(total + spare).astype(np.int32)
    table = np.full((len(pages_of), width), -1, np.int32)
    table[np.arange(width)[None, :] < pages_of[:, None]] = order[:total]
    return table, order[total:]


def _runs_bound(rows, batch, page):
    return min(rows, rows // page + 2 * batch)


def _plan_inputs(case, rng):
    batch, page, width = case["batch"], case["page"], -(-(case["context"] + case["chunk"]) // case["page"])
    context = _chance(rng, 1, case["context"], batch).astype(np.int32)
    new = np.ones(batch, np.int32)
    who = rng.permutation(batch)
    prompts, done = who[: case["prompts"]], who[case["prompts"]: case["prompts"] + case["done"]]
    new[prompts] = _chance(rng, 1, case["chunk"], len(prompts))
    context[prompts[::2]] = 0  # every other one begins
    new[done] = -1
    have = -(-context // page)
    need = int((-(-(context + np.maximum(new, 0)) // page) - have).sum())
    table, free = _table(rng, have, width, need + int(rng.integers(1, 64)))
    capacity = batch * -(-(case["context"] + case["chunk"]) // page) + 64  # one size of pool for all seeds
    taken = int(rng.integers(0, 4 * capacity))
    ring = np.full(capacity, -1, np.int32)
    ring[(taken + np.arange(len(free))) % capacity] = free
    state = dict(context_len=context, new_len=new, page_table=table, free_pages=ring,
                 pool_state=np.array([taken, taken + len(free), 0], np.int64))
    state = {k: torch.from_numpy(v).cuda() for k, v in state.items()}
    rows = batch + case["prompts"] * case["chunk"]
    return dict(state, rows=rows, page=page, num_pages=capacity)


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


def _pool(gen, num_pages, page, heads, d):
    """Codes and scales of normally distributed values, each page and head with a magnitude of its own."""
    x = torch.randn(num_pages, page, heads, d, generator=gen, device="cuda", dtype=torch.float16)
    peak = x.abs().amax(dim=(1, 3), keepdim=True).float()
    codes = (x * (E4M3_MAX / peak).half()).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
    size = torch.exp2(2 * torch.rand(num_pages, heads, generator=gen, device="cuda") - 1)
    return codes, (peak.view(num_pages, heads) / E4M3_MAX * size).contiguous()


def prepare(case, seed):
    rng = np.random.default_rng([seed, 17])
    if case["op"] == "plan":
        s = _plan_inputs(case, rng)
        rows, batch = s["rows"], case["batch"]
        like = dict(dtype=torch.int32, device="cuda")
        s["out"] = dict(context_len=torch.empty(batch, **like), row_start=torch.empty(batch + 1, **like),
                        slot_map=torch.empty(rows, dtype=torch.int64, device="cuda"),
                        runs=torch.empty(_runs_bound(rows, batch, case["page"]), **like),
                        pool_state=torch.empty(3, dtype=torch.int64, device="cuda"))
        return dict(s, op="plan")
    gen = torch.Generator(device="cuda").manual_seed(seed)
    batch, page, heads, d = case["batch"], case["page"], case["heads"], case["d"]
    if case["op"] == "append":
        context = _chance(rng, 0, case["context"], batch)
        new = _chance(rng, 1, case["new"], batch)
        pages = -(-(context + new) // page)
        table, free = _table(rng, pages, int(pages.max()), 3)
        start = np.concatenate([[0], np.cumsum(new)])
        slot = np.full(case["rows"], -1, np.int64)
        first = np.zeros(case["rows"], bool)
        for b in range(batch):
            pos = context[b] + np.arange(new[b])
            slot[start[b]: start[b + 1]] = table[b, pos // page].astype(np.int64) * page + pos % page
            first[start[b]: start[b + 1]] = (pos % page == 0) | (pos == context[b])
        runs = np.full(_runs_bound(case["rows"], batch, page), -1, np.int32)
        runs[: first.sum()] = np.flatnonzero(first)
        num_pages = int(pages.sum()) + len(free)
        extra = batch * (case["context"] + case["new"]) // page + 2 * batch + 3 - num_pages  # one size of pool for all seeds
        num_pages += max(0, extra)
        s = dict(op="append", page=page, slot_map=torch.from_numpy(slot).cuda(), runs=torch.from_numpy(runs).cuda())
        for name in ("k", "v"):
            codes, _ = _pool(gen, num_pages, page, heads, d)
            s[name + "_pages"] = codes
            s[name + "_scale"] = torch.exp2(torch.randint(-9, -5, (num_pages, heads), generator=gen, device="cuda").float())
            # one row in eight is larger than what came before it: its page's scale has to grow
            size = torch.where(torch.rand(case["rows"], heads, 1, generator=gen, device="cuda") < 0.125, 16.0, 1.0)
            x = torch.randn(case["rows"], heads, d, generator=gen, device="cuda") * size
            s[name] = x.to(_dtype(case))
        return s
    new = np.full(batch, 1) if case["new"] <= 1 else _chance(rng, 1, case["new"], batch)
    who = rng.permutation(batch)[: case["prompts"]]
    new[who] = _chance(rng, max(1, case["chunk"] // 2), case["chunk"], len(who)) if case["low"] < case["high"] else case["chunk"]
    context = np.maximum(_chance(rng, case["low"], case["high"], batch), new)
    longest = max(case["high"], case["chunk"], case["new"])
    pages = -(-context // page)
    width = -(-longest // page)
    table, free = _table(rng, pages, width, 2)
    rows = _rows(case)
    q_heads = heads * case["group"]
    s = dict(op="attention", page=page, page_table=torch.from_numpy(table).cuda(),
             context_len=torch.from_numpy(context.astype(np.int32)).cuda(),
             row_start=torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).cuda(),
             max_new=max(1, case["new"], case["chunk"]), max_context=longest, scale=1.0 / math.sqrt(d))
    s["k_pages"], s["k_scale"] = _pool(gen, int(pages.sum()) + len(free), page, heads, d)
    s["v_pages"], s["v_scale"] = _pool(gen, int(pages.sum()) + len(free), page, heads, d)
    s["q"] = torch.randn(rows, q_heads, d, generator=gen, device="cuda").to(_dtype(case))
    s["out"] = torch.zeros_like(s["q"])
    s["held"] = {}  # the workspace that a program keeps from its first call on
    return s


def _rows(case):
    """Rows of q: room for every request's most, as a program that pads its steps has it."""
    return (case["batch"] - case["prompts"]) * max(1, case["new"]) + case["prompts"] * case["chunk"]


# ---- the plain forms ---------------------------------------------------------------------------------------------------


def _plan(s):
    page, rows, table, ring = s["page"], s["rows"], s["page_table"].long(), s["free_pages"]
    context, new, width, capacity = s["context_len"].long(), s["new_len"].long(), s["page_table"].shape[1], s["free_pages"].shape[0]
    taken, given = s["pool_state"][0], s["pool_state"][1]
    n = new.clamp(min=0)
    have, after = (context + page - 1) // page, (context + n + page - 1) // page
    need = after - have
    refused = (need.sum() > given - taken) | (after > width).any()
    n, need = torch.where(refused, 0, n), torch.where(refused, 0, need)
    first, total = torch.cumsum(need, 0) - need, need.sum()
    start = torch.cumsum(n, 0)
    row_start = torch.cat([start.new_zeros(1), start])
    j = torch.arange(width, device="cuda")[None, :]
    fresh = (j >= have[:, None]) & (j < (have + need)[:, None])
    table = torch.where(fresh, ring[(taken + first[:, None] + j - have[:, None]) % capacity].long(), table)
    r = torch.arange(rows, device="cuda")
    b = torch.searchsorted(start, r, right=True).clamp(max=context.shape[0] - 1)
    live = r < start[-1]
    pos = torch.where(live, context[b] + r - row_start[b], 0)
    slot = torch.where(live, table[b, pos // page] * page + pos % page, -1)
    lead = live & ((pos % page == 0) | (r == row_start[b]))
    bound = s["out"]["runs"].shape[0]
    runs = torch.full((bound + 1,), -1, device="cuda")
    runs.scatter_(0, torch.where(lead, torch.cumsum(lead, 0) - 1, bound), torch.where(lead, r, -1))
    done = (new < 0)[:, None] & (j < have[:, None])
    order = torch.cumsum(done.reshape(-1), 0).reshape(done.shape) - 1
    back = torch.cat([ring.long(), ring.new_zeros(1).long()])
    back.scatter_(0, torch.where(done, (given + order) % capacity, capacity).reshape(-1), table.reshape(-1))
    state = torch.stack([taken + total, given + done.sum(), refused.long()])
    return dict(context_len=torch.where(new < 0, 0, context + n).int(), row_start=row_start.int(), slot_map=slot,
                runs=runs[:bound].int(), page_table=table.int(), free_pages=back[:capacity].int(), pool_state=state)


def _power(exponent):
    return ((exponent + 127) << 23).to(torch.int32).view(torch.float32)


def _append_one(x, pages, scale, slot, runs, page):
    """One of K and V: the pool's codes and scales with the rows put in, in place."""
    rows, heads, d = x.shape
    x = x.float()
    live = slot >= 0
    number = torch.zeros(rows + 1, dtype=torch.long, device="cuda")
    number[torch.where(runs >= 0, runs, rows).long()] = 1
    number = (torch.cumsum(number[:rows], 0) - 1).clamp(min=0)
    size = torch.where(torch.isfinite(x) & live[:, None, None], x.abs(), 0.0).amax(dim=2)
    peak = torch.zeros(runs.shape[0], heads, device="cuda").scatter_reduce_(0, number[:, None].expand(rows, heads), size, "amax")
    part, exponent = torch.frexp(peak)
    exponent = torch.where(peak > 0, exponent - 9 + (part > 0.875).int(), LEAST_EXPONENT).clamp(min=LEAST_EXPONENT)
    used = runs >= 0
    lead = slot[runs.clamp(min=0).long()]
    where, offset = (lead // page)[used], (lead % page)[used]
    old = torch.where((offset == 0)[:, None], 0.0, scale[where])
    now = torch.maximum(old, _power(exponent[used]))
    codes = pages[where].view(torch.float8_e4m3fn).float()
    moved = (codes * (old / now)[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    before = torch.arange(page, device="cuda")[None, :, None, None] < offset[:, None, None, None]
    pages[where] = torch.where(before, moved, pages[where])
    scale[where] = now
    share = now[number[live]]
    values = (x[live] / share[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
    pages[slot[live] // page, slot[live] % page] = values


def _append(s):
    _append_one(s["k"], s["k_pages"], s["k_scale"], s["slot_map"], s["runs"], s["page"])
    _append_one(s["v"], s["v_pages"], s["v_scale"], s["slot_map"], s["runs"], s["page"])
    return _cache_out(s)


def _cache_out(s):
    return dict(k_pages=s["k_pages"].view(torch.float8_e4m3fn), v_pages=s["v_pages"].view(torch.float8_e4m3fn),
                k_scale=s["k_scale"], v_scale=s["v_scale"])


def _values(pages, scale, table, longest):
    """[batch, heads, tokens, d] of the requests' keys or values, in f32."""
    held = table.clamp(min=0).long()
    x = pages[held].view(torch.float8_e4m3fn).float() * scale[held][:, :, None, :, None]
    return x.reshape(x.shape[0], -1, *x.shape[3:])[:, :longest].permute(0, 2, 1, 3)


def _attention(s):
    """Requests padded to the longest of each kind: their rows [batch, heads, group * rows, d] against all keys."""
    q, context, start = s["q"], s["context_len"].long(), s["row_start"].long()
    rows, q_heads, d = q.shape
    heads = s["k_pages"].shape[2]
    group, most, longest = q_heads // heads, s["max_new"], s["max_context"]
    k = _values(s["k_pages"], s["k_scale"], s["page_table"], longest)
    v = _values(s["v_pages"], s["v_scale"], s["page_table"], longest)
    i = torch.arange(most, device="cuda")[None, :]
    count = (start[1:] - start[:-1])[:, None]
    at = (start[:-1, None] + i).clamp(max=rows - 1)
    batch = at.shape[0]
    x = q[at].float().reshape(batch, most, heads, group, d).permute(0, 2, 3, 1, 4).reshape(batch, heads, group * most, d)
    score = torch.matmul(x, k.transpose(2, 3)).mul_(s["scale"]).reshape(batch, heads, group, most, longest)
    pos = context[:, None] - count + i
    key = torch.arange(longest, device="cuda")
    hidden = (key[None, None, :] > pos[:, :, None]) | (key[None, None, :] >= context[:, None, None])
    score.masked_fill_(hidden[:, None, None], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    weight = score.sub_(torch.where(torch.isfinite(top), top, 0.0)).exp_()
    total = weight.sum(dim=-1, keepdim=True)
    v = torch.where((key[None, :] < context[:, None])[:, None, :, None], v, 0.0)
    y = torch.matmul(weight.reshape(batch, heads, group * most, longest), v).reshape(batch, heads, group, most, d)
    y = torch.where(total > 0, y / total, 0.0).permute(0, 3, 1, 2, 4).reshape(batch, most, q_heads, d)
    live = i < count
    s["out"][at[live]] = y[live].to(q.dtype)
    return s["out"]


# ---- the framework's calls -----------------------------------------------------------------------------------------------


def _own(s):
    from krn_b200 import ops

    if s["op"] == "plan":
        plan = ops.CachePlan(**s["out"])
        ops.plan_cache(s["context_len"], s["new_len"], s["page_table"], s["free_pages"], s["pool_state"], plan, page_size=s["page"],
                       num_pages=s["num_pages"])
        return dict(s["out"], page_table=s["page_table"], free_pages=s["free_pages"])
    cache = ops.PagedCache(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"])
    if s["op"] == "append":
        ops.append_cache(s["k"], s["v"], s["slot_map"], s["runs"], cache)
        return _cache_out(s)
    held = s["held"]
    if "workspace" not in held:
        need = ops.cache_attention_workspace(s["context_len"].shape[0], s["q"].shape[0], s["q"].shape[1], s["k_pages"].shape[2],
                                             s["q"].shape[2], max_new=s["max_new"], max_context=s["max_context"])
        held["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda")
    return ops.cache_attention(s["q"], cache, s["page_table"], s["context_len"], s["row_start"], s["out"], max_new=s["max_new"],
                               max_context=s["max_context"], workspace=held["workspace"], scale=s["scale"])


def run(state):
    if own:
        return _own(state)
    return {"plan": _plan, "append": _append, "attention": _attention}[state["op"]](state)


def work(case):
    page = case["page"]
    if case["op"] == "plan":
        rows = case["batch"] - case["prompts"] - case["done"] + case["prompts"] * (case["chunk"] + 1) // 2
        padded = case["batch"] + case["prompts"] * case["chunk"]
        pages = rows / page + case["done"] * case["context"] / 2 / page  # taken and given back
        return {"bytes": 20 * case["batch"] + 8 * padded + 8 * pages + 4 * _runs_bound(padded, case["batch"], page) + 60, "flops": 0}
    heads, d = case["heads"], case["d"]
    if case["op"] == "append":
        rows = case["batch"] * (case["new"] + 1) / 2
        return {"bytes": 2 * (rows * heads * d * 3 + 8 * heads * (rows / page + case["batch"])) + 8 * rows,
                "flops": 2 * rows * heads * d * 3}
    new = [max(1, (1 + case["new"]) / 2)] * (case["batch"] - case["prompts"])
    new += [case["chunk"] * (0.75 if case["low"] < case["high"] else 1)] * case["prompts"]
    context = [max((case["low"] + case["high"]) / 2, n) for n in new]
    q_heads = heads * case["group"]
    seen = sum(n * (c - n) + n * (n + 1) / 2 for n, c in zip(new, context))
    return {"bytes": sum(context) * heads * 2 * (d + 4 / page) + sum(new) * q_heads * d * 4 + sum(context) / page * 4,
            "flops": 4 * q_heads * d * seen}


# ---- from the definition, in 64 bits ----------------------------------------------------------------------------------


def _decoded():
    """The value of every e4m3 code: sign, four bits of exponent (bias 7), three of mantissa; 0x7f and 0xff are NaN."""
    def value(code):
        e, m = code >> 3 & 15, code & 7
        if e == 15 and m == 7:
            return math.nan
        return (-1.0 if code >> 7 else 1.0) * (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))

    return torch.tensor([value(c) for c in range(256)], dtype=torch.float64, device="cuda")


def _nearest(x):
    """x rounded to the nearest e4m3 value, halves to even, saturated."""
    _, e = torch.frexp(x)
    step = torch.exp2((torch.clamp(e - 1, min=-6) - 3).double())
    return torch.clamp(torch.round(x / step) * step, -E4M3_MAX, E4M3_MAX)


def _exact_append(s):
    page, slot, table = s["page"], s["slot_map"].cpu().numpy(), _decoded()
    out = {}
    for name in ("k", "v"):
        codes, scale, x = table[s[name + "_pages"].long()], s[name + "_scale"].double(), s[name].double()
        row = 0
        while row < len(slot) and slot[row] >= 0:
            where, offset = divmod(int(slot[row]), page)
            count = 1
            while row + count < len(slot) and slot[row + count] == slot[row] + count and offset + count < page:
                count += 1
            new = x[row: row + count]
            peak = new.abs().amax(dim=(0, 2))
            need = torch.exp2((torch.round(torch.log2(peak / E4M3_MAX)) - 1).clamp(min=LEAST_EXPONENT))
            need = torch.where(peak > need * E4M3_MAX, 2 * need, need)  # the least power of two, whatever the logarithm's last bit
            need = torch.where(peak > need * E4M3_MAX, 2 * need, need)
            old = scale[where] if offset else torch.zeros_like(need)
            now = torch.maximum(old, need)
            if offset:
                codes[where, :offset] = _nearest(codes[where, :offset] * (old / now)[None, :, None])
            codes[where, offset: offset + count] = _nearest(new / now[None, :, None])
            scale[where] = now
            row += count
        out[name + "_pages"], out[name + "_scale"] = codes, scale
    return out


def _exact_attention(s):
    start, context, table = s["row_start"].tolist(), s["context_len"].tolist(), _decoded()
    page, (rows, q_heads, d), heads = s["page"], s["q"].shape, s["k_pages"].shape[2]
    out = torch.zeros(rows, q_heads, d, dtype=torch.float64, device="cuda")
    for b, length in enumerate(context):
        ids = s["page_table"][b, : -(-length // page)].long()
        n = start[b + 1] - start[b]
        ahead = torch.ones(n, length, dtype=torch.bool, device="cuda").tril(length - n).logical_not()
        for h in range(q_heads):
            g = h * heads // q_heads
            k = (table[s["k_pages"][ids, :, g].long()] * s["k_scale"][ids, g].double()[:, None, None]).reshape(-1, d)[:length]
            v = (table[s["v_pages"][ids, :, g].long()] * s["v_scale"][ids, g].double()[:, None, None]).reshape(-1, d)[:length]
            score = (s["q"][start[b]: start[b + 1], h].double() @ k.T * s["scale"]).masked_fill(ahead, -math.inf)
            out[start[b]: start[b + 1], h] = torch.softmax(score, dim=1) @ v
    return out


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    return _exact_append(s) if case["op"] == "append" else _exact_attention(s)
