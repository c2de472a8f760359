"""The paged 8-bit cache from its definitions, in Python integers and 64-bit floats (test infrastructure)."""

from __future__ import annotations

import math

import numpy as np

LEAST_EXPONENT = -100


def _decode_table() -> np.ndarray:
    values = np.empty(256)
    for code in range(256):
        e, m = code >> 3 & 15, code & 7
        size = math.nan if e == 15 and m == 7 else m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        values[code] = math.copysign(size, -1.0 if code >> 7 else 1.0)
    return values


DECODE = _decode_table()


def encode(x: np.ndarray) -> np.ndarray:
    """e4m3 codes of 64-bit values: nearest, ties to even, saturated at 448; NaN is 0x7f."""
    x = np.asarray(x, np.float64)
    nan = np.isnan(x)
    size = np.minimum(np.abs(np.where(nan, 0.0, x)), 448.0)
    _, e = np.frexp(size)
    exponent = np.maximum(e - 1, -6)
    steps = np.round(size * np.exp2(3.0 - exponent)).astype(np.int64)  # np.round: halves to even
    exponent, steps = np.where(steps == 16, exponent + 1, exponent), np.where(steps == 16, 8, steps)
    code = np.where(steps < 8, steps, (exponent + 7) * 8 + steps - 8) | np.where(np.signbit(x), 128, 0)
    return np.where(nan, 0x7F, code).astype(np.uint8)


def least_scale(peak: float) -> float:
    k = LEAST_EXPONENT
    while peak > 448.0 * 2.0 ** k:
        k += 1
    return 2.0 ** k


def plan(context, new, table, ring, state, *, page, rows, runs_len, num_pages):
    """(context, row_start, slot_map, runs, table, ring, state) after a step; arguments are left alone."""
    table, ring = table.copy(), ring.copy()
    batch, width = table.shape
    capacity, (taken, given) = len(ring), (int(state[0]), int(state[1]))
    context = [min(max(int(c), 0), width * page) for c in context]
    brings = [max(int(n), 0) for n in new]
    have = [-(-c // page) for c in context]
    after = [-(-(c + n) // page) for c, n in zip(context, brings)]
    need = sum(a - h for a, h in zip(after, have))
    refused = need > given - taken or max(after) > width or sum(brings) > rows
    back = [(b, j) for b in range(batch) if new[b] < 0 for j in range(have[b])]
    overfull = given - taken + len(back) > capacity
    slot, runs, start, spot = np.full(rows, -1, np.int64), [], [0], taken
    out = []
    row = 0
    for b in range(batch):
        n = 0 if refused else brings[b]
        for pos in range(context[b], context[b] + n):
            at = pos // page
            if at >= have[b] and pos % page == 0:
                table[b, at] = ring[spot % capacity]
                spot += 1
            if pos == context[b] or pos % page == 0:
                runs.append(row)
            good = 0 <= table[b, at] < num_pages
            slot[row] = int(table[b, at]) * page + pos % page if good else -1
            row += 1
        start.append(row)
        out.append((context[b] if overfull else 0) if new[b] < 0 else context[b] + n)
    if not overfull:
        for i, (b, j) in enumerate(back):
            ring[(given + i) % capacity] = table[b, j]
        given += len(back)
    runs = np.array(runs + [-1] * (runs_len - len(runs)), np.int32)
    return (np.array(out, np.int32), np.array(start, np.int32), slot, runs, table, ring,
            np.array([spot, given, (1 if refused else 0) | (2 if overfull else 0)], np.int64))


def append(x, slot, runs, codes, scale, *, page):
    """One pool (codes [pages, page, heads, d], scale [pages, heads]) with 64-bit rows x put in; arguments are left alone."""
    codes, scale = codes.copy(), scale.astype(np.float64)
    for row in runs:
        if row < 0 or row >= len(x) or slot[row] < 0 or slot[row] // page >= len(codes):
            continue
        where, offset = divmod(int(slot[row]), page)
        count = 1
        while offset + count < page and row + count < len(x) and slot[row + count] == slot[row] + count:
            count += 1
        for h in range(codes.shape[2]):
            new = x[row: row + count, h]
            finite = np.abs(new[np.isfinite(new)])
            need = least_scale(finite.max() if finite.size else 0.0)
            old = scale[where, h] if offset else 0.0
            now = max(old, need)
            if offset and now != old:
                codes[where, :offset, h] = encode(DECODE[codes[where, :offset, h]] * (old / now))
            codes[where, offset: offset + count, h] = encode(new / now)
            scale[where, h] = now
    return codes, scale


def attention(q, k_codes, v_codes, k_scale, v_scale, table, context, start, *, page, scale, untouched):
    """(out, bound): 64-bit attention of packed rows, and for each output the largest error that the kernels' roundings
    allow before the last one. With w the softmax weights and A = sum w |v|:

    * the query is used as f16 or as two e4m3 parts, off by at most 2^-8 of each element, so a score moves by at most
      delta = scale * 2^-8 * sum |q k| (largest over the keys) and a weight by exp(2 delta) - 1;
    * f32 sums of up to a few hundred products and the exponential: below 2^-14 of delta's sum and 2^-20 of a weight;
    * a weight is rounded to f16, at most 2^-11 of it, or 2^-25 of the largest: 2^-11 A, and with up to 2^17 keys of
      equal weight 2^-8 ulp-sized terms stay below another 2^-11 A;
    * a page's value scale, relative to the largest, is rounded to f16 and so is its product with a value: 2^-11 A each."""
    rows, q_heads, d = q.shape
    heads = k_codes.shape[2]
    out = np.array(untouched, np.float64)
    bound = np.zeros_like(out)
    for b in range(len(context)):
        n, c = int(start[b + 1] - start[b]), int(context[b])
        if n == 0:
            continue
        ids = table[b, : -(-c // page)]
        for h in range(q_heads):
            g = h // (q_heads // heads)
            k = (DECODE[k_codes[ids, :, g]] * k_scale[ids, g][:, None, None]).reshape(-1, d)[:c]
            v = (DECODE[v_codes[ids, :, g]] * v_scale[ids, g][:, None, None]).reshape(-1, d)[:c]
            x = q[start[b]: start[b + 1], h].astype(np.float64)
            seen = np.arange(c)[None, :] <= (c - n + np.arange(n))[:, None]
            with np.errstate(invalid="ignore"):
                s = np.where(seen, x @ k.T * scale, -np.inf)
                moved = np.where(seen, np.abs(x) @ np.abs(k).T * scale, 0.0).max(axis=1, initial=0.0)
            for i in range(n):
                if not seen[i].any():
                    out[start[b] + i, h] = 0.0
                    continue
                w = np.exp(s[i] - s[i].max())
                w /= w.sum()
                a = w[seen[i]] @ np.abs(v[seen[i]])
                out[start[b] + i, h] = w[seen[i]] @ v[seen[i]]
                delta = moved[i] * (2.0 ** -8 + 2.0 ** -14)
                bound[start[b] + i, h] = a * (math.expm1(2 * delta) + 4 * 2.0 ** -11 + 2.0 ** -17)
    return out, bound
