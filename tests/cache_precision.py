"""How far attention over the paged 8-bit cache may be from its definition, as the sum of what the kernels round (test
infrastructure). `cache_reference.attention` bounds single results by the worst case of every rounding at once; here the errors of
a row are taken together, as the independent errors that they are, so that a lost part of the query or results that are off by a
fiftieth are seen.

With u_j = exp(s_j - max s), L = sum u_j, w_j = u_j / L and o = sum w_j v_j, what a kernel does to a row of d results is

    e = sum_j eps_j v_j + sum_j w_j delta_j (v_j - o) + rho,

* eps_j: a weight is rounded to f16, whose half step is 2^-11 of it, and 2^-25 below f16's normal range. Weights are lifted by
  `lift` octaves before that, the largest being 2^lift at least, so the error is max(2^-11 u_j, 2^-25 - lift) / L. A page's value
  scale is rounded to f16 and so is its product with a value: 2^-11 w_j each;
* delta_j: the score's error. The query is held to 2^-21 of its row's largest magnitude (e4m3 parts, the last of them e5m2:
  see `query_parts`; the streamed kernel's f16 copy is finer), which meets the key's d values with signs of their own; sums of
  256 products in f32 are taken as 2^-20 of sum |q_i k_i|;
* rho: the result's own rounding, half a step of its type.

A rounding within half a step h has a variance of h^2 / 3 at most. Adding variances gives E |e|^2 <= T^2 with

    T^2 = sum_j |v_j|^2 (max(2^-11 u_j, 2^-25 - lift)^2 / L^2 + 2 (2^-11 w_j)^2) / 3 + sum_j w_j^2 delta_j^2 |v_j - o|^2 + sum h^2 / 3.

A row where one key has all the weight has a single eps, which may reach sqrt(3) of its deviation; where many have, |e| lies close
to T. So |e| <= 3 T for each row. Summed over the rows of a case, hundreds of errors, |e| <= 1.25 T."""

from __future__ import annotations

import numpy as np

from tests.cache_reference import DECODE, encode

ROW, ALL = 3.0, 1.25
LIFT = {"bfloat16": 7, "float16": 6}       # of the tiled kernel; the streamed one lifts by 15
HALF_STEP = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
LEAST_HALF_STEP = {"bfloat16": 0.0, "float16": 2.0 ** -25}


def requests(q, k_codes, v_codes, k_scale, v_scale, table, context, start, *, page):
    """(rows, q head, queries [n, d], keys [c, d], values [c, d], keys seen [n, c]) of every request and q head."""
    q_heads, heads = q.shape[1], k_codes.shape[2]
    for b in range(len(context)):
        first, n, c = int(start[b]), int(start[b + 1] - start[b]), int(context[b])
        if n == 0 or c == 0:
            continue
        ids = table[b, : -(-c // page)]
        seen = np.arange(c)[None, :] <= (c - n + np.arange(n))[:, None]
        for g in range(heads):
            k = (DECODE[k_codes[ids, :, g]] * k_scale[ids, g].astype(np.float64)[:, None, None]).reshape(-1, q.shape[2])[:c]
            v = (DECODE[v_codes[ids, :, g]] * v_scale[ids, g].astype(np.float64)[:, None, None]).reshape(-1, q.shape[2])[:c]
            for h in range(g * q_heads // heads, (g + 1) * q_heads // heads):
                yield slice(first, first + n), h, q[first: first + n, h], k, v, seen


def softmax(scores, seen):
    """(u, L) of every row; a row that sees nothing has u = 0 and L = 1."""
    s = np.where(seen, scores, -np.inf)
    top = s.max(axis=1, keepdims=True)
    u = np.exp(s - np.where(np.isfinite(top), top, 0.0))
    total = u.sum(axis=1, keepdims=True)
    return u, np.where(total > 0, total, 1.0)


def expected(dtype, q, *cache, page, scale):
    """(out, T): 64-bit attention, and for every row and q head the deviation that the kernels' roundings allow."""
    out, spread = np.zeros(q.shape), np.zeros(q.shape[:2])
    step, least = HALF_STEP[dtype], LEAST_HALF_STEP[dtype]
    for rows, h, x, k, v, seen in requests(q, *cache, page=page):
        u, total = softmax(x @ k.T * scale, seen)
        w = u / total
        o = w @ v
        v2 = (v * v).sum(axis=1)
        weight = np.where(seen, np.maximum(2.0 ** -11 * u, 2.0 ** (-25 - LIFT[dtype])), 0.0) / total
        squares = (weight ** 2 + 2 * (2.0 ** -11 * w) ** 2) @ v2 / 3
        query = 2.0 ** -21 * np.abs(x).max(axis=1, keepdims=True) * np.sqrt((k * k).sum(axis=1))[None, :] / np.sqrt(3.0)
        delta = scale * (query + 2.0 ** -20 * (np.abs(x) @ np.abs(k).T))
        away = v2[None, :] - 2 * o @ v.T + (o * o).sum(axis=1, keepdims=True)  # |v_j - o|^2
        squares += ((w * delta) ** 2 * np.maximum(away, 0.0)).sum(axis=1)
        squares += (np.maximum(step * np.abs(o), least) ** 2).sum(axis=1) / 3
        out[rows, h], spread[rows, h] = o, np.sqrt(squares)
    return out, spread


def deviations(got, out, spread):
    """(the worst row's error in units of T, all rows' error in units of all rows' T)."""
    wrong = np.sqrt(((got - out) ** 2).sum(axis=2))
    rows = np.divide(wrong, spread, out=np.where(wrong > 0, np.inf, 0.0), where=spread > 0)
    return float(rows.max()), float(np.linalg.norm(wrong) / (np.linalg.norm(spread) or 1.0))  # outputs may be zeros, exactly


def holds(worst, together) -> bool:
    return worst <= ROW and together <= ALL


# ---- a model of the tiled kernel's roundings, for the checks themselves -------------------------------------------------


def e5m2(x):
    """x rounded to the nearest e5m2 value."""
    _, e = np.frexp(x)
    step = np.exp2(np.maximum(e - 1, -14) - 2.0)
    return np.round(x / step) * step


def query_parts(x, parts, last=e5m2):
    """The query as the sum of `parts` 8-bit parts, each the rounded remainder of those before: e4m3, the last one e5m2."""
    size = np.abs(x).max(axis=-1, keepdims=True)
    factor = np.exp2(7 - np.floor(np.log2(np.where(size > 0, size, 1.0))))
    held = np.zeros_like(x)
    for part in range(parts):
        rest = x * factor - held
        held = held + (last(rest) if part + 1 == parts else DECODE[encode(rest)])
    return held / factor


def modelled(dtype, q, *cache, page, scale, parts=None, last=e5m2, lift=None, by=1.0):
    """Attention with the tiled kernel's roundings (two of them together for the values); `parts`, `last`, `lift` and `by` plant
    mistakes."""
    import torch

    parts = parts or (2 if dtype == "bfloat16" else 3)
    lift = LIFT[dtype] if lift is None else lift
    out = np.zeros(q.shape)
    for rows, h, x, k, v, seen in requests(q, *cache, page=page):
        u, total = softmax(query_parts(x, parts, last) @ k.T * scale, seen)
        weight = (u * 2.0 ** lift).astype(np.float16).astype(np.float64) / 2.0 ** lift
        size = np.exp2(np.floor(np.log2(np.abs(v).max())) - 14)
        out[rows, h] = weight / total @ ((v / size).astype(np.float16).astype(np.float64) * size) * by
    return torch.from_numpy(out).to(getattr(torch, dtype)).double().numpy()
