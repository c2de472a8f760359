"""The paged 8-bit cache's calls without a GPU: sizes that a program asks for before it launches anything, and refusals."""

from __future__ import annotations

import pytest

from krn_b200 import ops
from krn_b200.runtime import native
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
