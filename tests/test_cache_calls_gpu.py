"""Calls of the paged 8-bit cache that its documentation allows: memory side by side."""

from __future__ import annotations

import numpy as np
import pytest

from krn_b200 import ops
from tests import cache_reference as ref
from tests.test_cache_gpu import plan_case

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
