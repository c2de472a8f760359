"""The precision that attention over the paged 8-bit cache is held to: a model of its roundings passes, planted mistakes do not."""

from __future__ import annotations

import math

import numpy as np
import pytest

from krn_b200 import formats
from tests import cache_precision as precision
from tests import cache_reference as ref


def case(rng, dtype, context, new, page, heads, group, d, sink=0.0, outlier=0.0):
    """Normally distributed queries, keys and values. sink: octaves that the first key's score lies above the others', its value
    being zero. outlier: octaves that a query's first element lies above the others, which the keys do not have."""
    import torch

    context, new = np.array(context), np.array(new)
    pages = -(-context // page)
    order = rng.permutation(int(pages.sum())).astype(np.int32)
    table = np.full((len(context), int(pages.max())), -1, np.int32)
    table[np.arange(table.shape[1])[None, :] < pages[:, None]] = order
    q = rng.standard_normal((int(new.sum()), heads * group, d))
    codes, scales = [], []
    x, y = (rng.standard_normal((len(order), page, heads, d)) for _ in range(2))
    if sink or outlier:
        x[..., 0] = 0.0
    if outlier:
        q[..., 0] = 2.0 ** outlier
    if sink:
        q[..., 0] = 4.0
        for b in range(len(context)):
            x[table[b, 0], 0] = 0.0
            x[table[b, 0], 0, :, 0] = sink * math.log(2.0) * math.sqrt(d) / 4.0
            y[table[b, 0], 0] = 0.0
    for z in (x, y):
        s = np.abs(z).max(axis=(1, 3)) / 448.0
        codes.append(ref.encode(z / s[:, None, :, None]))
        scales.append((s * np.exp2(rng.uniform(-1, 1, s.shape) if not sink else 0.0)).astype(np.float32))
    q = torch.from_numpy(q).to(getattr(torch, dtype)).double().numpy()
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    return q, (*codes, *scales, table, context.astype(np.int32), start)


def deviations(rng, dtype, shape, scale=1.0, sink=0.0, outlier=0.0, **mistake):
    q, cache = case(rng, dtype, *shape, sink=sink, outlier=outlier)
    given = dict(page=shape[2], scale=scale / math.sqrt(shape[5]))
    return precision.deviations(precision.modelled(dtype, q, *cache, **given, **mistake), *precision.expected(dtype, q, *cache, **given))


SHAPES = [([300], [20], 16, 1, 4, 128), ([1000, 90], [9, 30], 64, 2, 2, 64), ([4000], [12], 64, 1, 4, 128)]
BOTH = pytest.mark.parametrize("dtype", ["bfloat16", "float16"])


def test_model_rounds_to_e5m2() -> None:
    import torch

    x = np.concatenate([np.random.default_rng(0).standard_normal(4000) * np.exp2(np.random.default_rng(1).integers(-18, 15, 4000)), [0.0]])
    x = x.astype(np.float32).astype(np.float64)
    np.testing.assert_array_equal(precision.e5m2(x), torch.from_numpy(x).float().to(torch.float8_e5m2).double().numpy())
    table = [c for c in formats.E5M2.table if math.isfinite(c)]
    np.testing.assert_array_equal(precision.e5m2(np.array(table)), table)


@BOTH
def test_query_parts(dtype) -> None:
    """Exact down to 2^-13 (bf16) and 2^-10 (f16) of the row's largest magnitude, off by 2^-21 of it at most below."""
    import torch

    rng = np.random.default_rng(2)
    parts, exact = (2, 13) if dtype == "bfloat16" else (3, 10)
    x = rng.standard_normal((3000, 64)) * np.exp2(-rng.uniform(0, 22, (3000, 64)))
    x = torch.from_numpy(x).to(getattr(torch, dtype)).double().numpy()
    largest = np.abs(x).max(axis=1, keepdims=True)
    off = np.abs(precision.query_parts(x, parts) - x)
    assert not off[np.abs(x) >= largest * 2.0 ** -exact].any()
    assert (off <= largest * 2.0 ** -21).all()


@BOTH
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("scale", [1.0, 3.0])
def test_roundings_pass(dtype, shape, scale) -> None:
    assert precision.holds(*deviations(np.random.default_rng(3), dtype, shape, scale))


@BOTH
@pytest.mark.parametrize("sink", [12.0, 18.0, 22.0, 24.0])
def test_roundings_pass_beside_a_sink(dtype, sink) -> None:
    assert precision.holds(*deviations(np.random.default_rng(4), dtype, SHAPES[0], sink=sink))
    assert precision.holds(*deviations(np.random.default_rng(5), dtype, SHAPES[2], sink=sink))


@BOTH
@pytest.mark.parametrize("outlier", [4.0, 8.0, 10.0, 12.0])
def test_roundings_pass_with_a_large_element(dtype, outlier) -> None:
    assert precision.holds(*deviations(np.random.default_rng(6), dtype, SHAPES[0], outlier=outlier))


@BOTH
@pytest.mark.parametrize("shape", SHAPES)
def test_a_lost_part_of_the_query_does_not_pass(dtype, shape) -> None:
    parts = 1 if dtype == "bfloat16" else 2
    assert not precision.holds(*deviations(np.random.default_rng(7), dtype, shape, 3.0, parts=parts))


@BOTH
@pytest.mark.parametrize("by", [1.02, 0.98])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_fiftieth_does_not_pass(dtype, shape, by) -> None:
    assert not precision.holds(*deviations(np.random.default_rng(8), dtype, shape, by=by))


@BOTH
@pytest.mark.parametrize("sink", [22.0, 24.0])
def test_weights_that_are_not_lifted_do_not_pass_beside_a_sink(dtype, sink) -> None:
    """Of 22 octaves on: at 18 they lose less than bf16's own rounding."""
    assert not precision.holds(*deviations(np.random.default_rng(9), dtype, SHAPES[0], sink=sink, lift=0))
    assert not precision.holds(*deviations(np.random.default_rng(10), dtype, SHAPES[2], sink=sink, lift=0))


@BOTH
@pytest.mark.parametrize("outlier", [10.0, 12.0])
def test_parts_of_e4m3_alone_do_not_pass_with_a_large_element(dtype, outlier) -> None:
    e4m3 = lambda x: ref.DECODE[ref.encode(x)]  # noqa: E731
    assert not precision.holds(*deviations(np.random.default_rng(11), dtype, SHAPES[0], outlier=outlier, last=e4m3, scale=4.0))
