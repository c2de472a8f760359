"""Attention over the paged 8-bit cache against its definition, held to what its roundings add up to (tests/cache_precision.py):
queries kept whole, weights far below the largest, keys split and joined."""

from __future__ import annotations

import math

import numpy as np
import pytest

from krn_b200 import ops
from tests import cache_precision as precision
from tests.test_cache_precision_cpu import case

pytestmark = pytest.mark.gpu


def check(torch, rng, dtype, shape, scale=1.0, **what):
    context, new, page, heads, group, d = shape
    q, cache = case(rng, dtype, *shape, **what)
    *pools, table, lengths, start = (torch.from_numpy(x).cuda() for x in cache)
    dq = torch.from_numpy(q).to(getattr(torch, dtype)).cuda()
    out = torch.full_like(dq, 7.0)
    longest, most, scale = table.shape[1] * page, max(new), scale / math.sqrt(d)
    workspace = torch.empty(ops.cache_attention_workspace(len(new), len(q), heads * group, heads, d, max_new=most, max_context=longest),
                            dtype=torch.uint8, device="cuda")
    ops.cache_attention(dq, ops.PagedCache(*pools), table, lengths, start, out, max_new=most, max_context=longest, workspace=workspace,
                        scale=scale)
    worst, together = precision.deviations(out.double().cpu().numpy(), *precision.expected(dtype, q, *cache, page=page, scale=scale))
    assert precision.holds(worst, together), (worst, together)


BOTH = pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
STREAMED = [([300], [1], 16, 2, 4, 128), ([3000, 90, 700], [1, 1, 1], 64, 2, 8, 64), ([900, 333], [8, 3], 32, 1, 4, 128),
            ([500, 70], [9, 4], 128, 2, 7, 64), ([20001], [1], 256, 1, 4, 128)]
TILED = [([300], [20], 16, 1, 4, 128), ([1000, 90], [9, 40], 64, 2, 2, 64), ([500, 400, 64], [70, 300, 64], 128, 1, 3, 128),
         ([6000], [40], 32, 1, 4, 128), ([2500, 3000], [33, 100], 256, 2, 8, 64), ([4000], [12], 64, 1, 128, 128)]


@BOTH
@pytest.mark.parametrize("shape", STREAMED + TILED)
@pytest.mark.parametrize("scale", [1.0, 3.0])
def test_attention_is_held_to_its_roundings(cuda, dtype, shape, scale) -> None:
    check(cuda, np.random.default_rng(70), dtype, shape, scale)


@BOTH
@pytest.mark.parametrize("shape", STREAMED + TILED)
@pytest.mark.parametrize("sink", [12.0, 18.0, 22.0, 24.0])
def test_attention_beside_a_sink(cuda, dtype, shape, sink) -> None:
    """One key has nearly all the weight and a value of zero: the output is made of the small weights."""
    check(cuda, np.random.default_rng(71), dtype, shape, sink=sink)


@BOTH
@pytest.mark.parametrize("shape", STREAMED + TILED)
@pytest.mark.parametrize("outlier", [6.0, 10.0, 12.0])
def test_attention_of_queries_with_a_large_element(cuda, dtype, shape, outlier) -> None:
    """An element of the query far above the others, where the keys are zero: the scores are made of the others."""
    check(cuda, np.random.default_rng(72), dtype, shape, 4.0, outlier=outlier)
