"""Calls of the paged 8-bit cache that its documentation allows: memory side by side, attention in place, contexts that are cut."""

from __future__ import annotations

import numpy as np
import pytest

from krn_b200 import ops
from tests import cache_reference as ref
from tests.test_cache_gpu import Server, attention_case, exact_check, plan_case, run_attention

pytestmark = pytest.mark.gpu


def test_plan_in_memory_side_by_side(cuda) -> None:
    """Outputs that end where inputs begin, in one allocation, and between the rows of the table: nothing is shared, so nothing
    is refused, and the plan is the same."""
    torch = cuda
    page, batch, rows = 16, 6, 41
    case = plan_case(np.random.default_rng(60), batch, page, 2, 12, 1, 60)
    width = case["table"].shape[1]
    pitch = 4 * width + 64  # room for a vector between two rows
    bound = ops.cache_plan(batch, rows, page).runs.shape[0]
    memory = torch.full((batch * pitch + 4 * (batch + rows + bound) + 2 * len(case["ring"]) + 64,), -3, dtype=torch.int32, device="cuda")
    at = 0

    def cut(n, dtype=torch.int32):
        nonlocal at
        words = n * (2 if dtype is torch.int64 else 1)
        piece = memory[at: at + words].view(dtype)
        at += words
        return piece

    slot, state, state_out = cut(rows, torch.int64), cut(3, torch.int64), cut(3, torch.int64)
    context, context_out, new, ring = cut(batch), cut(batch), cut(batch), cut(len(case["ring"]))
    base = at
    table = memory[base: base + batch * pitch].view(batch, pitch)[:, :width]
    start, runs = memory[base + width: base + width + batch + 1], memory[base + 3 * pitch - bound: base + 3 * pitch]
    assert batch + 1 + bound <= pitch - width
    for held, name in ((context, "context"), (new, "new"), (ring, "ring"), (state, "state"), (table, "table")):
        held.copy_(torch.from_numpy(case[name]))
    plan = ops.CachePlan(context_out, start, slot, runs, state_out)
    ops.plan_cache(context, new, table, ring, state, plan, page_size=page, num_pages=case["num_pages"])
    want = ref.plan(case["context"], case["new"], case["table"], case["ring"], case["state"], page=page, rows=rows, runs_len=bound,
                    num_pages=case["num_pages"])
    for got, expected in zip((context_out, start, slot, runs, table, ring, state_out), want):
        np.testing.assert_array_equal(got.cpu().numpy(), expected)
    np.testing.assert_array_equal(context.cpu().numpy(), case["context"])
    np.testing.assert_array_equal(new.cpu().numpy(), case["new"])


@pytest.mark.parametrize("dtype,context,new,page,heads,group,d", [
    ("bfloat16", [300, 65], [1, 1], 64, 2, 4, 128), ("float16", [5000, 700], [3, 2], 16, 1, 4, 64),  # streamed, whole and in pieces
    ("bfloat16", [500, 130], [200, 70], 32, 2, 4, 128), ("float16", [6000], [90], 64, 1, 4, 128),   # tiled, whole and in shares
    ("bfloat16", [2900, 80, 700], [150, 1, 2], 64, 2, 4, 64)])                                      # side by side
def test_attention_in_place(cuda, dtype, context, new, page, heads, group, d) -> None:
    """`out` may be q itself: a row of q is read by those only that write it."""
    torch = cuda
    case = attention_case(torch, np.random.default_rng(61), dtype, context, new, page, heads, group, d)
    want = run_attention(torch, case)
    q, rows = case["q"].clone(), sum(new)
    cache = ops.PagedCache(*(torch.from_numpy(x).cuda() for x in (*case["codes"], *case["scales"])))
    table, lengths, start = (torch.from_numpy(case[x]).cuda() for x in ("table", "context", "start"))
    given = dict(max_new=max(new), max_context=table.shape[1] * page)
    workspace = torch.empty(ops.cache_attention_workspace(len(new), len(q), heads * group, heads, d, **given), dtype=torch.uint8,
                            device="cuda")
    ops.cache_attention(q, cache, table, lengths, start, q, workspace=workspace, **given)
    assert torch.equal(q[:rows], want[:rows]) and torch.equal(q[rows:], case["q"][rows:])


def test_drafted_tokens_that_are_not_kept(cuda) -> None:
    """Each step brings up to four tokens a request, of which some are kept: the context is cut, and a page that it no longer
    reaches goes back to the ring. No page is lost, and the outputs are those over the tokens that were kept."""
    torch, rng = cuda, np.random.default_rng(62)
    batch, page, pages = 5, 16, 40
    server = Server(torch, batch, 60, page=page, pages=pages, width=6, max_new=20)
    new = [20, 15, 1, 16, 3]
    for step in range(14):
        server.inputs(rng, new)
        server.out.fill_(7.0)
        plan = server.step()
        assert plan.pool_state[2].item() == 0
        assert plan.context_len.tolist() == [len(h) for h in server.held]
        server.check(new)
        exact_check(server, plan, new)
        cut = [int(rng.integers(0, n)) if step else 0 for n in new]
        for b, n in enumerate(cut):
            del server.held[b][len(server.held[b]) - n:]
        before, after = plan.context_len.clone(), plan.context_len - torch.tensor(cut, dtype=torch.int32, device="cuda")
        left, right = (after + page - 1) // page, (before + page - 1) // page
        entry = torch.arange(server.table.shape[1], device="cuda")
        back = server.table[(entry >= left[:, None]) & (entry < right[:, None])]
        given = plan.pool_state[1].item()
        server.ring[(given + torch.arange(len(back), device="cuda")) % pages] = back
        plan.pool_state[1] += len(back)
        plan.context_len.copy_(after)
        state = plan.pool_state.tolist()
        free = server.ring[(state[0] + torch.arange(state[1] - state[0], device="cuda")) % pages].tolist()
        held = server.table[entry < left[:, None]].tolist()
        assert sorted(free + held) == list(range(pages))
        new = [int(n) for n in rng.integers(1, 5, batch)]
