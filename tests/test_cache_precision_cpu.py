"""The precision that attention over the paged 8-bit cache is held to: a model of its roundings passes, planted mistakes do not."""

from __future__ import annotations

import math

import numpy as np
import pytest

from tests import cache_precision as precision
from tests import cache_reference as ref


def case(rng, dtype, context, new, page, heads, group, d):
    """Normally distributed queries, keys and values."""
    import torch

    context, new = np.array(context), np.array(new)
    pages = -(-context // page)
    order = rng.permutation(int(pages.sum())).astype(np.int32)
    table = np.full((len(context), int(pages.max())), -1, np.int32)
    table[np.arange(table.shape[1])[None, :] < pages[:, None]] = order
    q = rng.standard_normal((int(new.sum()), heads * group, d))
    codes, scales = [], []
    x, y = (rng.standard_normal((len(order), page, heads, d)) for _ in range(2))
    for z in (x, y):
        s = np.abs(z).max(axis=(1, 3)) / 448.0
        codes.append(ref.encode(z / s[:, None, :, None]))
        scales.append((s * np.exp2(rng.uniform(-1, 1, s.shape))).astype(np.float32))
    q = torch.from_numpy(q).to(getattr(torch, dtype)).double().numpy()
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    return q, (*codes, *scales, table, context.astype(np.int32), start)


def judged(rng, dtype, shape, scale=1.0, **mistake):
    q, cache = case(rng, dtype, *shape)
    given = dict(page=shape[2], scale=scale / math.sqrt(shape[5]))
    return precision.judge(precision.modelled(dtype, q, *cache, **given, **mistake), *precision.expected(dtype, q, *cache, **given))


SHAPES = [([300], [20], 16, 1, 4, 128), ([1000, 90], [9, 30], 64, 2, 2, 64), ([4000], [12], 64, 1, 4, 128)]
BOTH = pytest.mark.parametrize("dtype", ["bfloat16", "float16"])


@BOTH
def test_query_parts(dtype) -> None:
    """Exact down to 2^-9 of the row's largest magnitude, off by 2^-17 of it at most below."""
    import torch

    rng = np.random.default_rng(2)
    parts, exact = (2, 9) if dtype == "bfloat16" else (3, 6)
    x = rng.standard_normal((3000, 64)) * np.exp2(-rng.uniform(0, 22, (3000, 64)))
    x = torch.from_numpy(x).to(getattr(torch, dtype)).double().numpy()
    largest = np.abs(x).max(axis=1, keepdims=True)
    off = np.abs(precision.query_parts(x, parts) - x)
    assert not off[np.abs(x) >= largest * 2.0 ** -exact].any()
    assert (off <= largest * 2.0 ** -17).all()


@BOTH
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("scale", [1.0, 3.0])
def test_roundings_pass(dtype, shape, scale) -> None:
    assert precision.holds(*judged(np.random.default_rng(3), dtype, shape, scale))


@BOTH
@pytest.mark.parametrize("shape", SHAPES)
def test_a_lost_part_of_the_query_does_not_pass(dtype, shape) -> None:
    parts = 1 if dtype == "bfloat16" else 2
    assert not precision.holds(*judged(np.random.default_rng(7), dtype, shape, 3.0, parts=parts))


@BOTH
@pytest.mark.parametrize("by", [1.02, 0.98])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_fiftieth_does_not_pass(dtype, shape, by) -> None:
    assert not precision.holds(*judged(np.random.default_rng(8), dtype, shape, by=by))
