"""The paged 8-bit cache on the GPU: plan, append and attention through `krn_b200.ops`, against 64-bit definitions."""

from __future__ import annotations

import math

import numpy as np
import pytest

from krn_b200 import ops
from krn_b200.runtime import calls, native
from tests import cache_reference as ref

pytestmark = pytest.mark.gpu

INT_MAX = 2 ** 31 - 1


# ---- plan --------------------------------------------------------------------------------------------------------------


def plan_case(rng, batch, page, prompts, chunk, done, context_high, spare=5, begin=0.3):
    context = rng.integers(0, context_high + 1, batch)
    new = rng.integers(0, 2, batch)
    who = rng.permutation(batch)
    new[who[:prompts]] = rng.integers(1, chunk + 1, prompts)
    context[rng.random(batch) < begin] = 0
    new[who[prompts: prompts + done]] = -1
    have = -(-context // page)
    need = int((-(-(context + np.maximum(new, 0)) // page) - have).sum())
    held, free = int(have.sum()), need + spare
    order = rng.permutation(held + free).astype(np.int32)
    width = -(-(context_high + chunk) // page) + 1
    table = np.full((batch, width), -7, np.int32)
    table[np.arange(width)[None, :] < have[:, None]] = order[:held]
    capacity = held + free
    taken = int(rng.integers(0, 5 * capacity))
    ring = np.full(capacity, -9, np.int32)
    ring[(taken + np.arange(free)) % capacity] = order[held:]
    return dict(context=context.astype(np.int32), new=new.astype(np.int32), table=table, ring=ring,
                state=np.array([taken, taken + free, 0], np.int64), num_pages=capacity)


def run_plan(torch, case, page, rows, pitch_extra=0):
    t = {k: torch.from_numpy(v).cuda() for k, v in case.items() if isinstance(v, np.ndarray)}
    if pitch_extra:
        wide = torch.full((t["table"].shape[0], t["table"].shape[1] + pitch_extra), -3, dtype=torch.int32, device="cuda")
        wide[:, : t["table"].shape[1]] = t["table"]
        t["wide"], t["table"] = wide, wide[:, : t["table"].shape[1]]
    plan = ops.cache_plan(len(case["context"]), rows, page)
    for x in (plan.context_len, plan.row_start, plan.slot_map, plan.runs, plan.pool_state):
        x.fill_(12345)
    ops.plan_cache(t["context"], t["new"], t["table"], t["ring"], t["state"], plan, page_size=page, num_pages=case["num_pages"])
    torch.cuda.synchronize()
    got = [x.cpu().numpy() for x in (plan.context_len, plan.row_start, plan.slot_map, plan.runs, t["table"], t["ring"], plan.pool_state)]
    return got, plan, t


def check_plan(torch, case, page, rows, **more):
    got, plan, t = run_plan(torch, case, page, rows, **more)
    want = ref.plan(case["context"], case["new"], case["table"], case["ring"], case["state"], page=page, rows=rows,
                    runs_len=len(got[3]), num_pages=case["num_pages"])
    for name, g, w in zip(("context", "row_start", "slot_map", "runs", "table", "ring", "state"), got, want):
        np.testing.assert_array_equal(g, w, err_msg=name)
    return got, plan, t


@pytest.mark.parametrize("batch,page,prompts,chunk,done,high", [
    (1, 64, 0, 1, 0, 100), (1, 16, 1, 1000, 0, 1), (3, 16, 1, 40, 1, 17), (16, 64, 0, 1, 0, 8192), (70, 32, 9, 300, 11, 2000),
    (513, 16, 40, 129, 60, 700), (1025, 128, 100, 77, 100, 300), (8192, 256, 3, 500, 900, 600)])
def test_plan_against_reference(cuda, batch, page, prompts, chunk, done, high) -> None:
    rng = np.random.default_rng(batch)
    case = plan_case(rng, batch, page, prompts, chunk, done, high)
    total = int(np.maximum(case["new"], 0).sum())
    for rows in (total, total + 77):
        check_plan(cuda, case, page, rows)
    check_plan(cuda, case, page, total, pitch_extra=3)


def test_plan_repeats_itself(cuda) -> None:
    """The same inputs over the same table and ring give the same plan again: the tool for replaying a captured step."""
    case = plan_case(np.random.default_rng(5), 40, 16, 5, 100, 4, 300)
    got, plan, t = check_plan(cuda, case, 16, 600)
    ops.plan_cache(t["context"], t["new"], t["table"], t["ring"], t["state"], plan, page_size=16, num_pages=case["num_pages"])
    again = [x.cpu().numpy() for x in (plan.context_len, plan.row_start, plan.slot_map, plan.runs, t["table"], t["ring"], plan.pool_state)]
    for g, w in zip(again, got):
        np.testing.assert_array_equal(g, w)


def test_plan_without_new_tokens(cuda) -> None:
    case = plan_case(np.random.default_rng(6), 9, 32, 0, 1, 0, 100)
    case["new"][:] = 0
    check_plan(cuda, case, 32, 0)
    check_plan(cuda, case, 32, 13)


def test_plan_refuses_a_step_that_does_not_fit(cuda) -> None:
    """Too few free pages, a table row too short, more rows than the slot map: nothing is taken, finished requests still
    give their pages back."""
    rng = np.random.default_rng(7)
    case = plan_case(rng, 30, 16, 6, 90, 5, 200, spare=0)
    total = int(np.maximum(case["new"], 0).sum())
    got, _, _ = check_plan(cuda, case, 16, total)
    assert got[-1][2] == 0 and got[-1][0] == case["state"][1]  # the last free page is used
    short = dict(case, state=case["state"] - np.array([0, 1, 0]))
    got, _, _ = check_plan(cuda, short, 16, total)
    assert got[-1][2] == 1 and (got[2] == -1).all() and got[-1][1] > short["state"][1]
    got, _, _ = check_plan(cuda, case, 16, total - 1)
    assert got[-1][2] == 1
    narrow = dict(case, table=case["table"][:, : int((-(-(case["context"] + np.maximum(case["new"], 0)) // 16)).max()) - 1].copy())
    got, _, _ = check_plan(cuda, narrow, 16, total)
    assert got[-1][2] == 1


def test_plan_of_wild_lengths(cuda) -> None:
    """Lengths that overflow any 32-bit sum are refused, contexts are clamped to the table."""
    case = plan_case(np.random.default_rng(8), 12, 64, 2, 50, 2, 300)
    case["new"][case["new"] >= 0] = INT_MAX
    got, _, _ = check_plan(cuda, case, 64, 100)
    assert got[-1][2] & 1
    case = plan_case(np.random.default_rng(9), 12, 64, 0, 1, 0, 300)
    case["new"][:] = 0
    case["context"][3], case["context"][4] = INT_MAX, -5
    case["table"][3] = np.arange(case["table"].shape[1]) % case["num_pages"]
    check_plan(cuda, case, 64, 8)


def test_plan_refuses_pages_given_back_twice(cuda) -> None:
    case = plan_case(np.random.default_rng(10), 8, 16, 0, 1, 0, 200)
    case["new"][:] = -1
    case["ring"] = case["ring"][: int(case["state"][1] - case["state"][0])].copy()  # a ring with room for the free pages only
    got, _, _ = check_plan(cuda, case, 16, 4)
    assert got[-1][2] == 2 and got[-1][1] == case["state"][1]


def test_plan_reports_bad_page_ids(cuda) -> None:
    """An id outside the pool in the ring or in the table: no slot for its tokens, and the status word says so."""
    case = plan_case(np.random.default_rng(11), 20, 16, 3, 60, 0, 100, begin=0.0)
    case["new"][:] = np.maximum(case["new"], 1)
    case = dict(case, ring=np.where(np.arange(len(case["ring"])) % 3 == 0, case["num_pages"], case["ring"]).astype(np.int32))
    free = int(case["state"][1] - case["state"][0])
    need = int((-(-(case["context"] + case["new"]) // 16) - -(-case["context"] // 16)).sum())
    assert need <= free + 20
    case["state"][1] = max(case["state"][1], case["state"][0] + need)
    check_plan(cuda, case, 16, int(case["new"].sum()))
    code, site, _ = native.device_status()
    assert code == native.ERR_DEVICE_INDEX and site == 41


# ---- append ------------------------------------------------------------------------------------------------------------


def lay_out(rng, context, new, page, rows, batch=None):
    """slot_map, runs and page table of requests that hold `context` tokens and bring `new`, over a shuffled pool."""
    pages = -(-(context + new) // page)
    total = int(pages.sum()) + 2
    order = rng.permutation(total).astype(np.int32)
    width = max(1, int(pages.max()))
    table = np.full((len(new), width), -1, np.int32)
    table[np.arange(width)[None, :] < pages[:, None]] = order[: int(pages.sum())]
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    slot, runs = np.full(rows, -1, np.int64), []
    for b in range(len(new)):
        for i in range(int(new[b])):
            pos = int(context[b]) + i
            slot[start[b] + i] = int(table[b, pos // page]) * page + pos % page
            if i == 0 or pos % page == 0:
                runs.append(start[b] + i)
    runs_len = calls.cache_runs(rows, len(new), page)
    assert len(runs) <= runs_len
    return table, start, slot, np.array(runs + [-1] * (runs_len - len(runs)), np.int32), total


def to16(torch, x, dtype):
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda().to(getattr(torch, dtype))
    return t, t.double().cpu().numpy()


def pool(rng, pages, page, heads, d):
    codes = rng.integers(0, 256, (pages, page, heads, d), dtype=np.uint8)
    codes[(codes & 0x7F) == 0x7F] = 0x3A
    return codes, np.exp2(rng.integers(-9, 3, (pages, heads))).astype(np.float32)


def check_append(torch, rng, dtype, context, new, page, heads, d, padding=0, change=None, spread=6.0):
    rows = int(new.sum()) + padding
    table, start, slot, runs, total = lay_out(rng, context, new, page, rows)
    kx, vx = (rng.standard_normal((rows, heads, d)) * np.exp2(rng.uniform(-spread, spread, (rows, heads, 1))) for _ in range(2))
    if change is not None:
        change(kx, vx)
    k, kx = to16(torch, kx, dtype)
    v, vx = to16(torch, vx, dtype)
    kc, ks = pool(rng, total, page, heads, d)
    vc, vs = pool(rng, total, page, heads, d)
    cache = ops.PagedCache(*(torch.from_numpy(x).cuda() for x in (kc, vc, ks, vs)))
    ds, dr = torch.from_numpy(slot).cuda(), torch.from_numpy(runs).cuda()
    for _ in range(2):  # the second pass over the same rows changes nothing
        ops.append_cache(k, v, ds, dr, cache)
        torch.cuda.synchronize()
        for name, x, codes, scale, got_codes, got_scale in (("k", kx, kc, ks, cache.k_pages, cache.k_scale),
                                                            ("v", vx, vc, vs, cache.v_pages, cache.v_scale)):
            want_codes, want_scale = ref.append(x, slot, runs, codes, scale, page=page)
            np.testing.assert_array_equal(got_scale.double().cpu().numpy(), want_scale, err_msg=name)
            np.testing.assert_array_equal(ref.DECODE[got_codes.cpu().numpy()], ref.DECODE[want_codes], err_msg=name)
    return cache, table, start


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page,heads,context,new", [
    (64, 8, [0], [1]), (64, 2, [63, 64, 100, 0], [1, 1, 1, 1]), (16, 3, [5, 0, 31, 16], [0, 40, 2, 15]),
    (128, 1, [100, 0], [300, 129]), (256, 2, [3, 0], [255, 700]), (32, 5, [30], [1]), (64, 2, [10, 7], [200, 64])])
def test_append_against_reference(cuda, dtype, d, page, heads, context, new) -> None:
    rng = np.random.default_rng(page + heads + d)
    check_append(cuda, rng, dtype, np.array(context), np.array(new), page, heads, d, padding=len(new) - 1)


@pytest.mark.parametrize("dtype,d", [("bfloat16", 128), ("float16", 64)])
@pytest.mark.parametrize("batch,most,page", [(40, 64, 64), (25, 300, 64), (30, 200, 32), (12, 700, 256)])
def test_append_of_many_runs_of_all_lengths(cuda, dtype, d, batch, most, page) -> None:
    """More runs than the GPU holds blocks, short and longer than a warp or a block keeps in registers."""
    rng = np.random.default_rng(56)
    check_append(cuda, rng, dtype, rng.integers(0, 3 * page, batch), rng.integers(0, most + 1, batch), page, 9, d, padding=33)


def test_append_of_many_single_tokens(cuda) -> None:
    rng = np.random.default_rng(20)
    check_append(cuda, rng, "bfloat16", rng.integers(0, 500, 130), np.ones(130, np.int64), 64, 4, 128)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_append_of_infinities_nan_and_zeros(cuda, dtype) -> None:
    """Infinities saturate, NaN stays NaN, neither moves the scale; rows of zeros get the least scale; the largest and the
    least finite values of the type."""
    def change(k, v):
        k[0, 0, 3], k[1, 0, 5], k[2, 0, 7] = np.inf, -np.inf, np.nan
        k[3:, 1] = 0.0
        v[:, 0] = np.nan
        v[0, 1, 0] = 6e4 if dtype == "float16" else 3e38
        v[20:, 1] = 0.0
        v[25, 1, 1] = 6e-8 if dtype == "float16" else 1e-39
    rng = np.random.default_rng(21)
    check_append(cuda, rng, dtype, np.array([0, 3]), np.array([20, 30]), 16, 2, 128, change=change, spread=0.0)


def test_append_at_the_borders_of_a_scale(cuda) -> None:
    """Peaks of exactly 448 * 2^k, one bit above and one below; every e4m3 midpoint."""
    middle = (ref.DECODE[0:126] + ref.DECODE[1:127]) / 2

    def change(k, v):
        k[:, 0] = 0.0
        k[:16, 0, 0], k[16:32, 0, 0], k[32:48, 0, 0] = 448.0, 450.0, 446.0
        v[:, 0] = 0.0
        v[:, 0, 0] = 448.0
        v[:, 0, 1:127] = middle
    check_append(cuda, np.random.default_rng(22), "float16", np.array([0]), np.array([48]), 16, 1, 128, change=change, spread=0.0)


def test_append_into_strided_pools_and_from_strided_rows(cuda) -> None:
    """Rows cut from a fused projection, pools kept head by head and as halves of one allocation."""
    torch, rng = cuda, np.random.default_rng(23)
    page, heads, d = 16, 3, 64
    context, new = np.array([7, 0]), np.array([30, 18])
    rows = int(new.sum())
    table, start, slot, runs, total = lay_out(rng, context, new, page, rows)
    fused = torch.randn(rows, (4 + 2 * heads) * d, device="cuda").to(torch.bfloat16)
    k = fused[:, 4 * d: (4 + heads) * d].view(rows, heads, d)
    v = fused[:, (4 + heads) * d:].view(rows, heads, d)
    (kc, ks), (vc, vs) = pool(rng, total, page, heads, d), pool(rng, total, page, heads, d)
    both = torch.empty(total, heads, 2, page, d, dtype=torch.uint8, device="cuda")
    kp, vp = both[:, :, 0].permute(0, 2, 1, 3), both[:, :, 1].permute(0, 2, 1, 3)
    kp.copy_(torch.from_numpy(kc))
    vp.copy_(torch.from_numpy(vc))
    cache = ops.PagedCache(kp, vp, torch.from_numpy(ks).cuda(), torch.from_numpy(vs).cuda())
    ops.append_cache(k, v, torch.from_numpy(slot).cuda(), torch.from_numpy(runs).cuda(), cache)
    for x, codes, scale, got, got_scale in ((k, kc, ks, kp, cache.k_scale), (v, vc, vs, vp, cache.v_scale)):
        want, want_scale = ref.append(x.double().cpu().numpy(), slot, runs, codes, scale, page=page)
        np.testing.assert_array_equal(ref.DECODE[got.cpu().numpy()], ref.DECODE[want])
        np.testing.assert_array_equal(got_scale.double().cpu().numpy(), want_scale)


def test_append_skips_what_lies_outside(cuda) -> None:
    """Runs and slots beyond the rows and the pool are skipped; a slot beyond the pool is reported."""
    torch, rng = cuda, np.random.default_rng(24)
    (kc, ks), (vc, vs) = pool(rng, 3, 16, 2, 64), pool(rng, 3, 16, 2, 64)
    cache = ops.PagedCache(*(torch.from_numpy(x).cuda() for x in (kc, vc, ks, vs)))
    x = torch.ones(4, 2, 64, dtype=torch.float16, device="cuda")
    slot = torch.tensor([48, -1, 2 ** 40, 5], dtype=torch.int64, device="cuda")
    runs = torch.tensor([0, 1, 2, 4, -1, 2 ** 30], dtype=torch.int32, device="cuda")
    ops.append_cache(x, x, slot, runs, cache)
    torch.cuda.synchronize()
    assert native.device_status()[:2] == (native.ERR_DEVICE_INDEX, 42)
    np.testing.assert_array_equal(cache.k_pages.cpu().numpy(), kc)
    np.testing.assert_array_equal(cache.v_pages.cpu().numpy(), vc)
    np.testing.assert_array_equal(cache.k_scale.cpu().numpy(), ks)


# ---- attention ---------------------------------------------------------------------------------------------------------


def attention_case(torch, rng, dtype, context, new, page, heads, group, d, padding=2, spread=2.0):
    context, new = np.array(context), np.array(new)
    rows = int(new.sum()) + padding
    table, start, _, _, total = lay_out(rng, np.maximum(context, 1), np.zeros_like(new), page, rows)
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    codes, scales = [], []
    for _ in range(2):
        x = rng.standard_normal((total, page, heads, d))
        s = np.abs(x).max(axis=(1, 3)) / 448.0
        codes.append(ref.encode(x / s[:, None, :, None]))
        scales.append((s * np.exp2(rng.uniform(-spread, spread, s.shape))).astype(np.float32))
    q, _ = to16(torch, rng.standard_normal((rows, heads * group, d)), dtype)
    return dict(q=q, codes=codes, scales=scales, table=table, context=context.astype(np.int32), start=start, page=page)


def run_attention(torch, case, max_new=None, max_context=None, scale=None, workspace_fill=0xFF):
    c = case
    q = c["q"]
    batch, (rows, q_heads, d), heads = len(c["context"]), q.shape, c["codes"][0].shape[2]
    cache = ops.PagedCache(*(torch.from_numpy(x).cuda() for x in (*c["codes"], *c["scales"])))
    max_new = max_new or max(1, int(np.diff(c["start"]).max()))
    max_context = max_context or c["table"].shape[1] * c["page"]
    out = torch.full(q.shape, 7.0, device="cuda", dtype=q.dtype)
    need = ops.cache_attention_workspace(batch, rows, q_heads, heads, d, max_new=max_new, max_context=max_context)
    workspace = torch.full((need + 256,), workspace_fill, dtype=torch.uint8, device="cuda")
    ops.cache_attention(q, cache, torch.from_numpy(c["table"]).cuda(), torch.from_numpy(c["context"]).cuda(),
                        torch.from_numpy(c["start"]).cuda(), out, max_new=max_new, max_context=max_context,
                        workspace=workspace[:need], scale=scale)
    torch.cuda.synchronize()
    assert bool((workspace[need:] == workspace_fill).all())
    return out


def check_attention(torch, case, scale=None, table=None, codes=None, scales=None, context=None, **more):
    out = run_attention(torch, case, scale=scale, **more)
    q = case["q"]
    codes, scales = codes or case["codes"], scales or case["scales"]
    want, bound = ref.attention(q.double().cpu().numpy(), *codes, *(s.astype(np.float64) for s in scales),
                                case["table"] if table is None else table, case["context"] if context is None else context, case["start"],
                                page=case["page"], scale=scale or 1.0 / math.sqrt(q.shape[2]), untouched=np.full(q.shape, 7.0))
    got = out.double().cpu().numpy()
    half_step = torch.finfo(out.dtype).eps / 2
    least = 2.0 ** -25 if out.dtype == torch.float16 else 0.0
    wrong = np.abs(got - want) > bound * (1 + half_step) + np.abs(want) * half_step + least
    assert not wrong.any(), (int(wrong.sum()), np.argwhere(wrong)[:4].tolist(), got[wrong][:4], want[wrong][:4], bound[wrong][:4])
    assert np.isfinite(got).all()
    return out


LENGTHS = [
    ([1], [1]), ([64], [1]), ([65, 1, 300], [1, 1, 1]), ([700, 0, 33, 129], [1, 0, 1, 1]), ([2000], [1]),  # single tokens
    ([90, 4, 257], [3, 4, 2]), ([500, 31], [8, 1]),                                                          # a few rows
    ([200], [200]), ([130, 40, 1, 390], [70, 40, 1, 129]), ([1000], [33]), ([600, 700], [1, 260]),           # prompts and chunks
]


@pytest.mark.parametrize("context,new", LENGTHS)
@pytest.mark.parametrize("dtype,page,heads,group,d", [("bfloat16", 64, 2, 4, 128), ("float16", 16, 1, 8, 64), ("bfloat16", 32, 3, 1, 64),
                                                      ("float16", 128, 2, 3, 128), ("bfloat16", 256, 1, 5, 128)])
def test_attention_against_reference(cuda, context, new, dtype, page, heads, group, d) -> None:
    rng = np.random.default_rng(len(context) * 100 + page)
    check_attention(cuda, attention_case(cuda, rng, dtype, context, new, page, heads, group, d))


@pytest.mark.parametrize("group", [2, 6, 7, 12, 16, 20, 32, 40, 128])
@pytest.mark.parametrize("new", [1, 3])
def test_attention_of_head_groups(cuda, group, new) -> None:
    rng = np.random.default_rng(group)
    check_attention(cuda, attention_case(cuda, rng, "bfloat16", [77, 200], [new, 1], 16, 1, group, 128))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("new,group,d", [(8, 4, 128), (9, 4, 128), (5, 6, 128), (1, 33, 128), (16, 4, 64), (17, 4, 64), (5, 12, 64),
                                         (9, 7, 64), (1, 64, 64), (1, 65, 64), (2, 33, 64)])
def test_attention_at_the_border_of_the_paths(cuda, dtype, new, group, d) -> None:
    """As many rows a request as are streamed, and the next more."""
    rng = np.random.default_rng(57)
    check_attention(cuda, attention_case(cuda, rng, dtype, [new, 300, 0, 1500], [new, new, 1, max(1, new - 1)], 32, 2, group, d), max_new=new)


def test_attention_of_a_long_context(cuda) -> None:
    """One request over thousands of keys: the work is split over the keys and joined."""
    rng = np.random.default_rng(31)
    check_attention(cuda, attention_case(cuda, rng, "bfloat16", [20001], [1], 64, 2, 4, 128))
    check_attention(cuda, attention_case(cuda, rng, "float16", [9000, 3], [20, 3], 32, 1, 4, 64))


def test_attention_of_rows_that_see_nothing(cuda) -> None:
    """A context shorter than the request's rows: rows before the first key get zeros; so does a context of zero."""
    rng = np.random.default_rng(32)
    for new in ([3, 2, 1], [40, 60, 1]):
        case = attention_case(cuda, rng, "bfloat16", [1, 0, 5], new, 16, 2, 4, 128)
        out = check_attention(cuda, case)
        assert not out[: new[0] - 1].any() and not out[new[0]: new[0] + new[1]].any()


@pytest.mark.parametrize("new", [1, 5, 100])
def test_attention_ignores_what_lies_behind_the_context(cuda, new) -> None:
    """NaN codes, infinite and NaN scales and wild page ids past the context."""
    rng = np.random.default_rng(33)
    context = [70, 129, 200]
    case = attention_case(cuda, rng, "bfloat16", context, [min(new, c) for c in context], 64, 2, 4, 128)
    clean = check_attention(cuda, case)
    dirty = dict(case, table=case["table"].copy(), codes=[x.copy() for x in case["codes"]], scales=[x.copy() for x in case["scales"]])
    used = np.zeros(len(case["codes"][0]), bool)
    for b, c in enumerate(context):
        last = c // 64
        if c % 64:
            for codes in dirty["codes"]:
                codes[case["table"][b, last], c % 64:] = 0x7F
        used[case["table"][b, : -(-c // 64)]] = True
        dirty["table"][b, -(-c // 64):] = 2 ** 31 - 1 if b % 2 else -5
    for i in range(2):
        dirty["codes"][i][~used] = 0xFF
        dirty["scales"][i][~used] = np.nan
    np.testing.assert_array_equal(run_attention(cuda, dirty).view(cuda.int16).cpu().numpy(), clean.view(cuda.int16).cpu().numpy())


@pytest.mark.parametrize("new", [1, 6, 90])
def test_attention_never_fetches_pages_outside_the_pool(cuda, new) -> None:
    """A bad id inside the context reads as a page of zeros, and the status word reports it."""
    rng = np.random.default_rng(34)
    case = attention_case(cuda, rng, "bfloat16", [100, 333], [new, 1], 64, 2, 4, 128)
    pages = len(case["codes"][0])
    broken, zeroed = case["table"].copy(), case["table"].copy()
    broken[0, 1], broken[1, 2] = pages, -1
    zeroed[0, 1] = zeroed[1, 2] = pages
    codes = [np.concatenate([c, np.zeros((1,) + c.shape[1:], np.uint8)]) for c in case["codes"]]
    scales = [np.concatenate([s, np.zeros((1,) + s.shape[1:], np.float32)]) for s in case["scales"]]
    check_attention(cuda, dict(case, table=broken), table=zeroed, codes=codes, scales=scales)
    assert native.device_status()[0] == native.ERR_DEVICE_INDEX


def test_attention_clamps_contexts(cuda) -> None:
    rng = np.random.default_rng(35)
    for new in (1, 50):
        case = attention_case(cuda, rng, "bfloat16", [128, 100, 60], [new, 1, 1], 64, 2, 4, 128)
        wild = dict(case, context=np.array([2 ** 31 - 1, 100, -9], np.int32))
        out = check_attention(cuda, wild, context=np.array([128, 100, 0], np.int32), max_context=128)
        assert not out[new + 1].any()


def test_attention_reports_more_rows_than_announced(cuda) -> None:
    rng = np.random.default_rng(36)
    for announced in (1, 40):
        case = attention_case(cuda, rng, "bfloat16", [100, 90], [announced + 1, 1], 16, 1, 4, 128)
        out = run_attention(cuda, case, max_new=announced)
        assert native.device_status()[:2] == (native.ERR_DEVICE_INDEX, 52)
        assert bool((out[: announced + 1] == 7).all()) and not bool((out[announced + 1] == 7).any())


@pytest.mark.parametrize("new,group", [(3, 4), (40, 4), (40, 1), (5, 40)])
def test_attention_refuses_rows_that_q_does_not_have(cuda, new, group) -> None:
    """A request whose rows reach behind q's last one is left out whole and reported; the others are computed."""
    rng = np.random.default_rng(53)
    case = attention_case(cuda, rng, "bfloat16", [100, 90], [2, new], 16, 1, group, 128)
    whole = run_attention(cuda, case, max_new=new)
    for missing in (1, new - 1):
        out = run_attention(cuda, dict(case, q=case["q"][: 2 + new - missing].contiguous()), max_new=new)
        assert native.device_status()[:2] == (native.ERR_DEVICE_INDEX, 52)
        assert bool((out[2:] == 7).all()) and not bool((out[:2] == 7).all(-1).any())
        # fewer rows may choose other kernels: each rounds its result by 2^-8 of it, and weights, values and scales to f16 (four
        # times 2^-11 of the largest value)
        assert cuda.allclose(out[:2].float(), whole[:2].float(), rtol=2 ** -7, atol=2 ** -8 * 448 * float(case["scales"][1].max()))


def test_bad_rows_of_late_requests_are_reported(cuda) -> None:
    """Requests behind those that the first block of a grid belongs to."""
    rng = np.random.default_rng(54)
    case = attention_case(cuda, rng, "bfloat16", [20] * 1200, [1] * 1199 + [2], 16, 1, 40, 64)
    out = run_attention(cuda, case, max_new=1)
    assert native.device_status()[:2] == (native.ERR_DEVICE_INDEX, 52)
    # whole rows: one of three million results may well round to 7
    assert bool((out[1199:] == 7).all()) and not bool((out[:1199] == 7).all(-1).any())


@pytest.mark.parametrize("new", [1, 64])
def test_attention_with_scales_far_apart(cuda, new) -> None:
    """Page scales from 2^-12 to 2^12 for both pools, and sharp softmaxes that settle on single keys."""
    rng = np.random.default_rng(37)
    case = attention_case(cuda, rng, "bfloat16", [300, 64], [new, 1], 16, 2, 4, 128)
    case["scales"][1] = np.exp2(rng.integers(-12, 13, case["scales"][1].shape)).astype(np.float32) / 100
    check_attention(cuda, case)
    check_attention(cuda, case, scale=2.0)
    case["scales"][1][...] = 0.0
    assert not check_attention(cuda, case)[:-2].any()


@pytest.mark.parametrize("new", [1, 4, 70])
def test_attention_of_large_and_small_queries(cuda, new) -> None:
    """Queries near the ends of bf16's range, balanced by the softmax scale; a row of zeros."""
    rng = np.random.default_rng(38)
    case = attention_case(cuda, rng, "bfloat16", [150, 80], [new, 1], 16, 1, 4, 128)
    q = case["q"]
    q[0] = 0
    for power in (-100, 80):
        check_attention(cuda, dict(case, q=q * 2.0 ** power), scale=2.0 ** -power / math.sqrt(128))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("new", [2, 70])
def test_attention_of_rows_with_nan_and_infinities(cuda, dtype, new) -> None:
    """A query row that holds a NaN or an infinity is NaN, and no other row is touched by it."""
    rng = np.random.default_rng(45)
    case = attention_case(cuda, rng, dtype, [150, 80], [new, 1], 16, 1, 4, 128)
    clean = run_attention(cuda, case)
    q = case["q"].clone()
    q[0, 1, 5], q[1, 3, 0], q[new, 2, 127] = math.nan, math.inf, -math.inf
    got = run_attention(cuda, dict(case, q=q))
    for row, head in ((0, 1), (1, 3), (new, 2)):
        assert bool(got[row, head].isnan().all())
        got[row, head] = clean[row, head]
    assert cuda.equal(got, clean)


@pytest.mark.parametrize("new", [1, 40])
def test_attention_with_a_negative_scale(cuda, new) -> None:
    rng = np.random.default_rng(46)
    check_attention(cuda, attention_case(cuda, rng, "bfloat16", [150, 80], [new, 1], 32, 1, 4, 64), scale=-0.2)


def test_pools_beyond_four_gigabytes(cuda) -> None:
    """Pages whose byte offsets do not fit 32 bits: the same bits as in a small pool."""
    torch, rng = cuda, np.random.default_rng(47)
    page, heads, d, far = 64, 8, 128, 70000
    context, new = np.array([100, 0, 77]), np.array([1, 130, 1])
    rows = int(new.sum())
    table, start, slot, runs, total = lay_out(rng, context, new, page, rows)
    (kc, ks), (vc, vs) = pool(rng, total, page, heads, d), pool(rng, total, page, heads, d)
    k, v, q = (torch.randn(rows, h, d, device="cuda").to(torch.bfloat16) for h in (heads, heads, 4 * heads))
    results = []
    for base, pages in ((0, total), (far, far + total)):
        cache = ops.PagedCache(*(torch.empty((pages, page, heads, d), dtype=torch.uint8, device="cuda") for _ in range(2)),
                               *(torch.empty((pages, heads), device="cuda") for _ in range(2)))
        for held, values in zip(cache, (kc, vc, ks, vs)):
            held[base:].copy_(torch.from_numpy(values))
        ids = torch.from_numpy(np.where(table >= 0, table + base, -1).astype(np.int32)).cuda()
        ops.append_cache(k, v, torch.from_numpy(slot + base * page).cuda(), torch.from_numpy(runs).cuda(), cache)
        out = torch.zeros_like(q)
        longest = table.shape[1] * page
        workspace = torch.empty(ops.cache_attention_workspace(3, rows, 4 * heads, heads, d, max_new=130, max_context=longest),
                                dtype=torch.uint8, device="cuda")
        ops.cache_attention(q, cache, ids, torch.from_numpy((context + new).astype(np.int32)).cuda(), torch.from_numpy(start).cuda(),
                            out, max_new=130, max_context=longest, workspace=workspace)
        results.append([x[base:].clone() for x in cache] + [out])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_attention_of_more_heads_than_warps(cuda) -> None:
    """More kv heads than the grid has warps: each takes several in turn."""
    rng = np.random.default_rng(48)
    check_attention(cuda, attention_case(cuda, rng, "bfloat16", [40], [1], 16, 1300, 1, 64))
    check_attention(cuda, attention_case(cuda, rng, "float16", [33, 5], [2, 1], 32, 1200, 2, 64))


@pytest.mark.parametrize("batch,new,group", [(1500, 1, 2), (700, 12, 4)])
def test_attention_of_many_requests(cuda, batch, new, group) -> None:
    """More requests than a block has threads, some without rows, some without keys."""
    rng = np.random.default_rng(49)
    rows = rng.integers(0, new + 1, batch)
    context = np.where(rng.random(batch) < 0.1, 0, rng.integers(0, 70, batch))
    check_attention(cuda, attention_case(cuda, rng, "bfloat16", context, rows, 16, 1, group, 64), max_new=new)


@pytest.mark.parametrize("batch,at,dtype,d,page", [(21, 20, "bfloat16", 128, 32), (4, 0, "float16", 128, 64), (700, 600, "bfloat16", 64, 16)])
def test_attention_of_a_chunk_among_decode_requests(cuda, batch, at, dtype, d, page) -> None:
    """One long request's keys are split over the blocks that the others leave, whatever the rows and requests would allow."""
    rng = np.random.default_rng(55)
    context, rows = rng.integers(1, 100, batch), np.ones(batch, int)
    context[at], rows[at] = 2900, 150
    rows[(at + 1) % batch], context[(at + 1) % batch] = 20, 700
    case = attention_case(cuda, rng, dtype, context, rows, page, 2, 4, d, padding=400)
    check_attention(cuda, case, max_new=200)
    check_attention(cuda, case, max_new=200, max_context=case["table"].shape[1] * page - 3)


def test_attention_announced_larger_than_it_is(cuda) -> None:
    """`max_new` and `max_context` only bound: any that hold give the same numbers within the kernels' roundings."""
    rng = np.random.default_rng(50)
    case = attention_case(cuda, rng, "bfloat16", [100, 37, 260], [2, 1, 5], 32, 2, 4, 128)
    for max_new in (5, 8, 9, 1000, 2 ** 40):
        check_attention(cuda, case, max_new=max_new)
    check_attention(cuda, case, max_context=260)


def test_device_tensors_and_streams_of_the_package(cuda) -> None:
    """The package's own tensors and streams in place of torch's."""
    import krn_b200
    from krn_b200.runtime.device import DeviceTensor

    torch, rng = cuda, np.random.default_rng(51)
    case = attention_case(torch, rng, "bfloat16", [100, 37], [1, 3], 32, 2, 4, 128)
    want = run_attention(torch, case)
    cache = ops.PagedCache(*(DeviceTensor(torch.from_numpy(x).cuda()) for x in (*case["codes"], *case["scales"])))
    table, context, start = (DeviceTensor(torch.from_numpy(case[x]).cuda()) for x in ("table", "context", "start"))
    out = DeviceTensor(torch.full_like(case["q"], 7.0))
    longest = case["table"].shape[1] * 32
    workspace = DeviceTensor(torch.empty(ops.cache_attention_workspace(2, case["q"].shape[0], 8, 2, 128, max_new=3, max_context=longest),
                                         dtype=torch.uint8, device="cuda"))
    stream = krn_b200.host.Device.current().default_stream
    torch.cuda.synchronize()
    assert ops.cache_attention(DeviceTensor(case["q"]), cache, table, context, start, out, max_new=3, max_context=longest,
                               workspace=workspace, stream=stream) is out
    stream.record().wait(60)
    assert torch.equal(out.data, want)


def test_attention_of_strided_tensors(cuda) -> None:
    """q cut from a fused projection, out head by head, pools as halves of one head-major allocation, a table with a pitch."""
    torch, rng = cuda, np.random.default_rng(39)
    for new in ([1, 1], [50, 3]):
        case = attention_case(torch, rng, "bfloat16", [100, 70], new, 32, 2, 4, 128)
        want = run_attention(torch, case)
        rows, q_heads, d = case["q"].shape
        fused = torch.zeros(rows, (q_heads + 4) * d, dtype=torch.bfloat16, device="cuda")
        q = fused[:, : q_heads * d].view(rows, q_heads, d)
        q.copy_(case["q"])
        out = torch.full((q_heads, rows, d), 7.0, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
        pages, page, heads, _ = case["codes"][0].shape
        both = torch.empty(pages, heads, 2, page, d, dtype=torch.uint8, device="cuda")
        kp, vp = both[:, :, 0].permute(0, 2, 1, 3), both[:, :, 1].permute(0, 2, 1, 3)
        kp.copy_(torch.from_numpy(case["codes"][0]))
        vp.copy_(torch.from_numpy(case["codes"][1]))
        cache = ops.PagedCache(kp, vp, *(torch.from_numpy(x).cuda() for x in case["scales"]))
        wide = torch.full((2, case["table"].shape[1] + 5), -1, dtype=torch.int32, device="cuda")
        wide[:, : case["table"].shape[1]] = torch.from_numpy(case["table"])
        most, longest = max(new), case["table"].shape[1] * page
        workspace = torch.empty(ops.cache_attention_workspace(2, rows, q_heads, heads, d, max_new=most, max_context=longest),
                                dtype=torch.uint8, device="cuda")
        ops.cache_attention(q, cache, wide[:, : case["table"].shape[1]], torch.from_numpy(case["context"]).cuda(),
                            torch.from_numpy(case["start"]).cuda(), out, max_new=most, max_context=longest, workspace=workspace)
        assert torch.equal(out, want)


# ---- together ----------------------------------------------------------------------------------------------------------


class Server:
    """A few requests served step by step through plan, append and attention, and the keys and values they brought."""

    def __init__(self, torch, batch, rows, page=16, heads=2, group=4, d=128, pages=64, width=20, max_new=64):
        self.torch, self.page, self.heads, self.group, self.d, self.max_new = torch, page, heads, group, d, max_new
        self.cache = ops.paged_cache(pages, page, heads, d)
        self.table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
        self.ring = torch.randperm(pages, device="cuda").int()
        self.plans = [ops.cache_plan(batch, rows, page) for _ in range(2)]
        self.plans[1].context_len.zero_()
        self.plans[1].pool_state.copy_(torch.tensor([0, pages, 0]))
        self.new = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.q = torch.zeros(rows, heads * group, d, dtype=torch.bfloat16, device="cuda")
        self.k, self.v = (torch.zeros(rows, heads, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        self.out = torch.full_like(self.q, 7.0)
        self.longest = width * page
        self.workspace = torch.empty(ops.cache_attention_workspace(batch, rows, heads * group, heads, d, max_new=max_new,
                                                                   max_context=self.longest), dtype=torch.uint8, device="cuda")
        self.turn = 0
        self.held = [[] for _ in range(batch)]  # (k, v) rows of each request, as quantised when it is checked

    def step(self):
        before, plan = self.plans[1 - self.turn % 2], self.plans[self.turn % 2]
        ops.plan_cache(before.context_len, self.new, self.table, self.ring, before.pool_state, plan, page_size=self.page,
                       num_pages=self.cache.num_pages)
        ops.append_cache(self.k, self.v, plan.slot_map, plan.runs, self.cache)
        ops.cache_attention(self.q, self.cache, self.table, plan.context_len, plan.row_start, self.out, max_new=self.max_new,
                            max_context=self.longest, workspace=self.workspace)
        self.turn += 1
        return plan

    def inputs(self, rng, new):
        torch = self.torch
        self.new.copy_(torch.tensor(new, dtype=torch.int32))
        for x in (self.q, self.k, self.v):
            x.copy_(torch.from_numpy(rng.standard_normal(tuple(x.shape)).astype(np.float32) * 2.0 ** rng.integers(-2, 3)))
        row = 0
        k, v = self.k.double().cpu().numpy(), self.v.double().cpu().numpy()
        for b, n in enumerate(new):
            if n < 0:
                self.held[b] = []
            for i in range(max(n, 0)):
                self.held[b].append((k[row], v[row]))
                row += 1

    def check(self, new):
        """The outputs against attention over the rows themselves: off by the cache's rounding and attention's."""
        out, q = self.out.double().cpu().numpy(), self.q.double().cpu().numpy()
        row = 0
        worst = 0.0
        for b, n in enumerate(new):
            n = max(n, 0)
            if n == 0:
                continue
            k, v = (np.stack([r[i] for r in self.held[b]]) for i in range(2))
            for i in range(n):
                c = len(k) - n + i + 1
                for h in range(q.shape[1]):
                    g = h // self.group
                    s = k[:c, g] @ q[row + i, h] / math.sqrt(self.d)
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    want = w @ v[:c, g]
                    worst = max(worst, np.linalg.norm(out[row + i, h] - want) / np.linalg.norm(v[:c, g], axis=1).max())
            row += n
        assert worst < 0.25, worst  # keys and values are kept in 3 mantissa bits
        assert (out[row:] == 7).all()


STEPS = [[40, 3, 0, 1], [1, 1, 17, 1], [1, 4, 1, 1], [-1, 1, 1, 1], [30, 1, -1, 2], [1, 1, 50, 1]]


def exact_check(server, plan, new):
    """The outputs against 64-bit attention over the cache as it stands."""
    q = server.q.double().cpu().numpy()
    arrays = [x.cpu().numpy() for x in (server.cache.k_pages, server.cache.v_pages, server.cache.k_scale, server.cache.v_scale)]
    want, bound = ref.attention(q, arrays[0], arrays[1], arrays[2].astype(np.float64), arrays[3].astype(np.float64),
                                server.table.cpu().numpy(), plan.context_len.cpu().numpy(), plan.row_start.cpu().numpy(),
                                page=server.page, scale=1.0 / math.sqrt(server.d), untouched=np.full(q.shape, 7.0))
    got = server.out.double().cpu().numpy()
    assert (np.abs(got - want) <= bound * (1 + 2.0 ** -8) + np.abs(want) * 2.0 ** -8).all()


@pytest.mark.parametrize("max_new", [64, 200])
def test_steps_of_a_server(cuda, max_new) -> None:
    """Prompts, chunks, single tokens, idle and finished requests over a pool whose pages are reused, padded rows."""
    rng = np.random.default_rng(40)
    server = Server(cuda, 4, 64, max_new=max_new)
    for new in STEPS:
        server.inputs(rng, new)
        server.out.fill_(7.0)
        plan = server.step()
        cuda.cuda.synchronize()
        assert plan.pool_state[2].item() == 0
        assert plan.context_len.tolist() == [len(h) for h in server.held]
        server.check(new)
        exact_check(server, plan, new)


def test_steps_captured_and_replayed(cuda) -> None:
    """Two steps (the two plans change places) in one CUDA graph on its own stream, replayed with new inputs: the same bits
    as eager calls."""
    torch, rng = cuda, np.random.default_rng(41)
    eager, graphed = Server(torch, 4, 64), Server(torch, 4, 64)
    graphed.ring.copy_(eager.ring)
    first = [12, 0, 5, 1]
    for s in (eager, graphed):
        s.inputs(np.random.default_rng(1), first)
        s.step()
        s.inputs(np.random.default_rng(2), [1, 1, 1, 1])
        s.step()
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    kept = [x.clone() for x in (graphed.plans[1].context_len, graphed.plans[1].pool_state)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        graphed.step()
        graphed.step()
    torch.cuda.synchronize()
    for a, b in zip(kept, (graphed.plans[1].context_len, graphed.plans[1].pool_state)):
        assert torch.equal(a, b)  # capturing runs nothing
    for n in range(4):
        new = [1, 2, 1, 1]
        seed = 10 + n
        for s in (eager, graphed):
            s.inputs(np.random.default_rng(seed), new)
        eager.step()
        eager.step()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in ((eager.out, graphed.out), (eager.cache.k_pages, graphed.cache.k_pages), (eager.cache.v_scale, graphed.cache.v_scale),
                     (eager.table, graphed.table), (eager.plans[1].context_len, graphed.plans[1].context_len)):
            assert torch.equal(a, b)


def test_calls_on_another_stream(cuda) -> None:
    torch = cuda
    rng = np.random.default_rng(42)
    case = attention_case(torch, rng, "bfloat16", [500, 80], [1, 3], 64, 2, 4, 128)
    want = run_attention(torch, case)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        got = run_attention(torch, case)
    stream.synchronize()
    assert torch.equal(got, want)


def test_two_calls_at_once_with_workspaces_of_their_own(cuda) -> None:
    torch, rng = cuda, np.random.default_rng(43)
    cases = [attention_case(torch, rng, "bfloat16", [3000 + 100 * i, 50], [1, 30], 64, 2, 4, 128) for i in range(2)]
    want = [run_attention(torch, c) for c in cases]
    streams = [torch.cuda.Stream() for _ in range(2)]
    held = []
    for c in cases:
        cache = ops.PagedCache(*(torch.from_numpy(x).cuda() for x in (*c["codes"], *c["scales"])))
        rows, q_heads, d = c["q"].shape
        need = ops.cache_attention_workspace(2, rows, q_heads, 2, d, max_new=30, max_context=c["table"].shape[1] * 64)
        held.append((c["q"], cache, torch.from_numpy(c["table"]).cuda(), torch.from_numpy(c["context"]).cuda(),
                     torch.from_numpy(c["start"]).cuda(), torch.full_like(c["q"], 7.0),
                     torch.empty(need, dtype=torch.uint8, device="cuda")))
    torch.cuda.synchronize()
    for _ in range(20):
        for h, s in zip(held, streams):
            q, cache, table, context, start, out, workspace = h
            ops.cache_attention(q, cache, table, context, start, out, max_new=30, max_context=table.shape[1] * 64,
                                workspace=workspace, stream=s)
    torch.cuda.synchronize()
    for h, w in zip(held, want):
        assert torch.equal(h[5], w)


def test_refusals_on_the_device(cuda) -> None:
    torch, rng = cuda, np.random.default_rng(44)
    case = attention_case(torch, rng, "bfloat16", [100], [1], 64, 2, 4, 128)
    cache = ops.PagedCache(*(torch.from_numpy(x).cuda() for x in (*case["codes"], *case["scales"])))
    table, context, start = (torch.from_numpy(case[x]).cuda() for x in ("table", "context", "start"))
    q = case["q"]
    workspace = torch.empty(1 << 26, dtype=torch.uint8, device="cuda")

    def call(q=q, out=None, table=table, context=context, start=start, **more):
        given = dict(max_new=1, max_context=100, workspace=workspace) | more
        ops.cache_attention(q, cache, table, context, start, torch.empty_like(q) if out is None else out, **given)

    call()
    with pytest.raises(TypeError, match="same element type"):
        call(out=q.half())
    with pytest.raises(TypeError, match="`context_len` must be int32"):
        call(context=context.long())
    with pytest.raises(ValueError, match="2 expected"):
        call(start=torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="do not match a pool"):
        call(q=q[..., :64].contiguous())
    with pytest.raises(ValueError, match="must not overlap"):
        call(out=q[:1].expand(q.shape))
    with pytest.raises(Exception, match="does not fit"):
        call(max_context=10 ** 6)
    with pytest.raises(Exception, match="KRN_B200_ERR_WORKSPACE"):
        call(workspace=workspace[:8])
    with pytest.raises(Exception, match="16-byte aligned"):
        call(workspace=workspace[8:])
    with pytest.raises(Exception, match="16 bits"):
        call(q=q.float())
    plan = ops.cache_plan(1, 4, 64)
    ring, state = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(Exception, match="share memory"):
        ops.plan_cache(plan.context_len, context, table, ring, state, plan, page_size=64, num_pages=4)
    with pytest.raises(ValueError, match="3 expected"):
        ops.plan_cache(context, context, table, ring, state[:2], plan, page_size=64, num_pages=4)
    with pytest.raises(ValueError, match="do not match a pool"):
        ops.append_cache(q[:, :3], q[:, :3], plan.slot_map, plan.runs, cache)
