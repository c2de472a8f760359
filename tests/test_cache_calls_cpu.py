"""The paged 8-bit cache's calls without a GPU: sizes that a program asks for before it launches anything, and refusals."""

from __future__ import annotations

import pytest

from krn_b200 import ops
from krn_b200.runtime import calls, native
from tests.test_cache_cpu import attention_status, plan_status


@pytest.mark.parametrize("group", [129, 256, 1000])
@pytest.mark.parametrize("max_new", [1, 40])
@pytest.mark.parametrize("max_context", [512, 1024, 100000])
@pytest.mark.parametrize("d", [64, 128])
def test_workspace_of_groups_that_the_call_refuses(group, max_new, max_context, d) -> None:
    """The size of what cannot be launched is the least one, as for other refused extents, and the call says why."""
    assert ops.cache_attention_workspace(3, 40, 2 * group, 2, d, max_new=max_new, max_context=max_context) == 16
    assert attention_status(q_heads=2 * group, size=16, max_new=max_new) == native.ERR_UNSUPPORTED
    assert f"{group} q heads per kv head" in native.last_error()


@pytest.mark.parametrize("group", [1, 64, 127, 128])
def test_workspace_of_the_largest_groups(group) -> None:
    assert ops.cache_attention_workspace(3, 40, group, 1, 128, max_new=40, max_context=100000) > 1 << 20


@pytest.fixture
def host_tensors(monkeypatch):
    """Lets the checks behind the calls see host tensors. For refusals only: a call that passes them would launch on them."""
    monkeypatch.setattr(calls._Checks, "addresses", lambda self, names, tensors: [t.data_ptr() for t in tensors])
    import torch

    return torch


@pytest.mark.parametrize("slots", [0, 3, 5, 80])
def test_append_refuses_slots_and_rows_of_other_numbers(host_tensors, slots) -> None:
    """Rows without a slot would not be written, slots without a row would keep what their page held."""
    torch = host_tensors
    cache = ops.PagedCache(*(torch.zeros(2, 16, 2, 64, dtype=torch.uint8) for _ in range(2)), *(torch.zeros(2, 2) for _ in range(2)))
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match=f"`slot_map` has {slots} elements, 4 expected"):
        ops.append_cache(x, x, torch.zeros(slots, dtype=torch.int64), torch.zeros(4, dtype=torch.int32), cache)


def test_attention_refuses_a_workspace_that_is_not_one_piece_of_memory(host_tensors) -> None:
    """An expanded tensor counts more bytes than there are behind it, a strided one shares its bytes with another."""
    torch = host_tensors
    cache = ops.PagedCache(*(torch.zeros(2, 16, 2, 64, dtype=torch.uint8) for _ in range(2)), *(torch.zeros(2, 2) for _ in range(2)))
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    table, lengths = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for workspace in (torch.zeros(1, dtype=torch.uint8).expand(1 << 26), torch.zeros(64, 2, dtype=torch.uint8)[:, 0]):
        with pytest.raises(ValueError, match="`workspace` must be contiguous"):
            ops.cache_attention(q, cache, table, lengths, torch.zeros(2, dtype=torch.int32), torch.zeros_like(q), max_new=4,
                                max_context=32, workspace=workspace)


# addresses that share nothing: 4 requests, 8 table entries at a pitch of 20, ring of 32, 16 rows, 9 runs
APART = dict(context=0x1000, new=0x1010, table=0x2000, pitch=20, ring=0x3000, state=0x4000, context_out=0x5000, start=0x5010, slot=0x6000,
             runs=0x6080, out=0x7000)


@pytest.mark.parametrize("change", [
    dict(context_out=0x100c), dict(context_out=0x0ff4), dict(start=0x101c), dict(out=0x4010), dict(out=0x3ff0),  # inputs
    dict(slot=0x1008), dict(runs=0x0fe0), dict(ring=0x0f84), dict(ring=0x3f90),
    dict(start=0x500c), dict(slot=0x6004), dict(runs=0x607c), dict(out=0x5008), dict(ring=0x6f90),                  # other outputs
    dict(context_out=0x201c), dict(start=0x1ff0), dict(runs=0x204c), dict(out=0x2108), dict(context=0x20fc),      # rows of the table
])
def test_plan_refuses_memory_that_outputs_share(change) -> None:
    assert plan_status(**(APART | change)) == native.ERR_INVALID_ARGUMENT
    assert "share memory" in native.last_error()
