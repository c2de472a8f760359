"""The paged 8-bit cache's calls without a GPU: sizes that a program asks for before it launches anything, and refusals."""

from __future__ import annotations

import pytest

from krn_b200 import ops
from krn_b200.runtime import calls, native
from tests.test_cache_cpu import attention_status


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
