"""The paged 8-bit cache without a GPU: the 64-bit reference against the number formats, and every refusal that is made
before anything is launched."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

from krn_b200 import formats, ops
from krn_b200.runtime import calls, native
from tests import cache_reference as ref


def test_reference_decodes_and_encodes_every_code() -> None:
    table = np.array(formats.E4M3FN.table)
    np.testing.assert_array_equal(ref.DECODE, table)
    codes = np.array([c for c in range(256) if not math.isnan(table[c])], np.uint8)
    np.testing.assert_array_equal(ref.encode(table[codes]), codes)


def test_reference_rounds_to_nearest_even_and_saturates() -> None:
    values = np.sort(np.unique(np.abs(ref.DECODE[~np.isnan(ref.DECODE)])))
    middle = (values[:-1] + values[1:]) / 2
    codes = ref.encode(middle)
    assert (codes % 2 == 0).all()  # the even one of the two neighbours
    assert (np.abs(ref.DECODE[codes] - middle) == (values[1:] - values[:-1]) / 2).all()
    assert ref.encode(np.array([449.0, 1e9, np.inf, -np.inf])).tolist() == [0x7E, 0x7E, 0x7E, 0xFE]
    assert ref.encode(np.array([np.nan]))[0] == 0x7F


@pytest.mark.parametrize("peak,scale", [(0.0, 2.0 ** -100), (448.0, 1.0), (449.0, 2.0), (3.5, 2.0 ** -7), (1e-45, 2.0 ** -100)])
def test_reference_scale(peak, scale) -> None:
    assert ref.least_scale(peak) == scale


def test_run_list_length() -> None:
    """Never shorter than the pages that any split of the rows over the requests can touch."""
    rng = np.random.default_rng(3)
    for _ in range(300):
        page = int(rng.choice([16, 32, 64, 128, 256]))
        batch = int(rng.integers(1, 40))
        new = rng.integers(0, 200, batch) * rng.integers(0, 2, batch)
        context = rng.integers(0, 500, batch)
        touched = sum(int((c + n - 1) // page - c // page + 1) for c, n in zip(context, new) if n)
        assert touched <= calls.cache_runs(int(new.sum()), batch, page)
    assert calls.cache_runs(0, 4, 64) == 0 and calls.cache_runs(1, 1, 256) == 1


def _strides(*values: int):
    return (ctypes.c_int64 * len(values))(*values)


def plan_status(**change) -> int:
    a = dict(context=16, new=32, table=48, ring=64, state=80, context_out=96, start=112, slot=128, runs=144, out=160, batch=4,
             width=8, pitch=8, capacity=32, page=64, pages=32, rows=16, runs_len=9, stream=None)
    a.update(change)
    return native.library().krn_b200_cache_plan(*a.values())


@pytest.mark.parametrize("change,status,text", [
    (dict(page=48), native.ERR_UNSUPPORTED, "page size 48"),
    (dict(page=8), native.ERR_UNSUPPORTED, "page size 8"),
    (dict(batch=8193, rows=0, runs_len=0), native.ERR_UNSUPPORTED, "at most 8192"),
    (dict(batch=0), native.ERR_INVALID_ARGUMENT, "at least one request"),
    (dict(runs_len=7), native.ERR_INVALID_ARGUMENT, "8 needed"),
    (dict(pitch=7), native.ERR_INVALID_ARGUMENT, "pitch 7"),
    (dict(rows=1 << 30, runs_len=1 << 30), native.ERR_UNSUPPORTED, "32-bit"),
    (dict(capacity=0), native.ERR_INVALID_ARGUMENT, "bad extents"),
    (dict(ring=None), native.ERR_INVALID_ARGUMENT, "null"),
    (dict(context_out=16), native.ERR_INVALID_ARGUMENT, "share memory"),
    (dict(out=80), native.ERR_INVALID_ARGUMENT, "share memory"),
])
def test_plan_refusals(change, status, text) -> None:
    assert plan_status(**change) == status
    assert text in native.last_error()


def append_status(**change) -> int:
    a = dict(type=native.BF16, k=16, v=16, slot=16, runs=16, kp=16, vp=16, ks=16, vs=16, rows=8, runs_len=8, heads=2, d=128, page=64,
             pages=4, strides=_strides(256, 128, 256, 128, 16384, 256, 128, 16384, 256, 128), stream=None)
    a.update(change)
    return native.library().krn_b200_cache_append(*a.values())


@pytest.mark.parametrize("change,status,text", [
    (dict(type=native.F32), native.ERR_UNSUPPORTED, "16 bits"),
    (dict(d=96), native.ERR_UNSUPPORTED, "head dimension 96"),
    (dict(page=20), native.ERR_UNSUPPORTED, "page size 20"),
    (dict(k=24), native.ERR_INVALID_ARGUMENT, "16 bytes"),
    (dict(strides=_strides(256, 128, 256, 132, 16384, 256, 128, 16384, 256, 128)), native.ERR_INVALID_ARGUMENT, "16 bytes"),
    (dict(strides=_strides(256, 128, 256, 128, 16384, 264, 128, 16384, 256, 128)), native.ERR_INVALID_ARGUMENT, "strides of a page pool"),
    (dict(strides=_strides(256, 128, 256, 128, 16384, 256, 128, 0, 256, 128)), native.ERR_INVALID_ARGUMENT, "strides of a page pool"),
    (dict(ks=None), native.ERR_INVALID_ARGUMENT, "null"),
    (dict(pages=0), native.ERR_INVALID_ARGUMENT, "bad extents"),
    (dict(heads=65536), native.ERR_UNSUPPORTED, "32-bit"),
])
def test_append_refusals(change, status, text) -> None:
    assert append_status(**change) == status
    assert text in native.last_error()


def attention_status(**change) -> int:
    a = dict(type=native.BF16, q=16, kp=16, vp=16, ks=16, vs=16, table=16, context=16, start=16, o=16, batch=2, rows=2, q_heads=8,
             kv_heads=2, d=128, page=64, pages=4, width=2, pitch=2, max_new=1, max_context=128,
             strides=_strides(1024, 128, 1024, 128, 16384, 256, 128, 16384, 256, 128), scale=1.0, workspace=16,
             size=1 << 40, stream=None)
    a.update(change)
    return native.library().krn_b200_cache_attn(*a.values())


@pytest.mark.parametrize("change,status,text", [
    (dict(type=native.E4M3), native.ERR_UNSUPPORTED, "16 bits"),
    (dict(d=256), native.ERR_UNSUPPORTED, "head dimension 256"),
    (dict(page=512), native.ERR_UNSUPPORTED, "page size 512"),
    (dict(q_heads=7), native.ERR_INVALID_ARGUMENT, "bad extents"),
    (dict(q_heads=258), native.ERR_UNSUPPORTED, "129 q heads per kv head"),
    (dict(max_context=129), native.ERR_INVALID_ARGUMENT, "does not fit 2 pages"),
    (dict(max_new=0), native.ERR_INVALID_ARGUMENT, "bad extents"),
    (dict(batch=8193), native.ERR_UNSUPPORTED, "at most 8192"),
    (dict(batch=8192, width=1 << 24, pitch=1 << 24, max_context=1 << 30), native.ERR_UNSUPPORTED, "32-bit"),
    (dict(o=None), native.ERR_INVALID_ARGUMENT, "null"),
    (dict(q=8), native.ERR_INVALID_ARGUMENT, "16 bytes"),
    (dict(strides=_strides(1028, 128, 1024, 128, 16384, 256, 128, 16384, 256, 128)), native.ERR_INVALID_ARGUMENT, "16 bytes"),
    (dict(strides=_strides(1024, 128, 1024, 128, 16384, 256, 100, 16384, 256, 128)), native.ERR_INVALID_ARGUMENT, "strides of a page pool"),
    (dict(size=8), native.ERR_WORKSPACE, "too small"),
    (dict(workspace=None), native.ERR_WORKSPACE, "too small"),
])
def test_attention_refusals(change, status, text) -> None:
    assert attention_status(**change) == status
    assert text in native.last_error()


def test_empty_steps_are_no_work() -> None:
    assert append_status(rows=0) == native.OK and append_status(runs_len=0) == native.OK
    assert attention_status(rows=0) == native.OK and attention_status(batch=0) == native.OK


def test_host_tensors_are_refused() -> None:
    import torch

    plan = ops.CachePlan(torch.empty(2, dtype=torch.int32), torch.empty(3, dtype=torch.int32), torch.empty(4, dtype=torch.int64),
                         torch.empty(4, dtype=torch.int32), torch.empty(3, dtype=torch.int64))
    lengths, table = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="`context_len` must be a CUDA tensor"):
        ops.plan_cache(lengths, lengths, table, lengths, torch.zeros(3, dtype=torch.int64), plan, page_size=64, num_pages=2)
    codes, scale = torch.zeros(2, 64, 2, 128, dtype=torch.uint8), torch.zeros(2, 2)
    cache = ops.PagedCache(codes, codes, scale, scale)
    x = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        ops.append_cache(x, x, plan.slot_map, plan.runs, cache)
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        ops.cache_attention(x, cache, table, lengths, plan.row_start, x, max_new=1, max_context=64, workspace=x)


def test_layout_checks() -> None:
    """The checks behind the calls, on host tensors."""
    import torch

    at = calls._Checks("t")
    x = torch.zeros(6, 4, 128)
    assert list(at.strides("x", x, True)) == [512, 128]
    assert list(at.strides("x", x.transpose(0, 1), True)) == [128, 512]
    assert list(at.strides("x", x[:, :1], True)) == [512, 128]
    assert list(at.strides("x", torch.zeros(6, 1, 128).as_strided((6, 1, 128), (128, 7, 1)), True)) == [128, 128]
    assert list(at.strides("x", x[:1].expand(6, 4, 128), False)) == [0, 128]
    with pytest.raises(ValueError, match="must not overlap"):
        at.strides("x", x[:1].expand(6, 4, 128), True)
    with pytest.raises(ValueError, match="must not overlap"):
        at.strides("x", torch.zeros(4096).as_strided((6, 4, 128), (256, 128, 1)), True)
    with pytest.raises(ValueError, match="last axis"):
        at.strides("x", torch.zeros(6, 4, 256)[..., ::2], False)
    codes, scale = torch.zeros(3, 16, 2, 64, dtype=torch.uint8), torch.zeros(3, 2)
    assert list(at.pool(codes, codes, scale, scale, True)[1]) == [2048, 128, 64] * 2
    with pytest.raises(TypeError, match="e4m3"):
        at.pool(codes.to(torch.int8), codes, scale, scale, True)
    with pytest.raises(TypeError, match="float32"):
        at.pool(codes, codes, scale.double(), scale, True)
    with pytest.raises(ValueError, match=r"contiguous \[3, 2\]"):
        at.pool(codes, codes, scale.t().contiguous().t(), scale, True)
    with pytest.raises(ValueError, match="page pools"):
        at.pool(codes, codes[:2], scale, scale, True)
    with pytest.raises(TypeError, match="int32"):
        at.table("page_table", torch.zeros(2, 4, dtype=torch.int64), 2)
    with pytest.raises(ValueError, match=r"\[3, entries\]"):
        at.table("page_table", torch.zeros(2, 4, dtype=torch.int32), 3)
    with pytest.raises(ValueError, match="5 expected"):
        at.vector("x", torch.zeros(4, dtype=torch.int32), torch.int32, 5)
    with pytest.raises(ValueError, match="contiguous vector"):
        at.vector("x", torch.zeros(8, dtype=torch.int32)[::2], torch.int32, -1)
    with pytest.raises(TypeError, match="must be int32, got torch.int64"):
        at.vector("x", torch.zeros(8, dtype=torch.int64), torch.int32, -1)
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        at.addresses("a b", (torch.zeros(2, device="meta"), object()))


def test_workspace_of_the_largest_step_serves_all() -> None:
    rng = np.random.default_rng(52)
    for _ in range(2000):
        heads, group, d = (int(rng.choice(x)) for x in ((1, 2, 8, 500), (1, 2, 4, 7, 8, 12, 33, 128), (64, 128)))
        largest = [int(2 ** rng.uniform(0, top)) for top in (9, 15, 14, 18)]  # requests, rows, new tokens, context
        smaller = [int(rng.integers(1, x + 1)) if rng.random() < 0.7 else x for x in largest]
        sizes = [ops.cache_attention_workspace(batch, rows, heads * group, heads, d, max_new=new, max_context=context)
                 for batch, rows, new, context in (largest, smaller)]
        assert sizes[0] >= sizes[1], (heads, group, d, largest, smaller)
