"""Page summaries, block selection, block attention, key weights and eviction from their definitions (numpy)."""

from __future__ import annotations

import numpy as np


def summary_ref(k, table, query_start, kv_len, bounds, scale):
    """Updates bounds int8 [pages, heads, 2, dim] and scale float32 [pages, heads] in place; k [pages, page, heads, dim]."""
    pages, page, heads, dim = k.shape
    for b in range(len(kv_len)):
        n, c = int(query_start[b + 1]) - int(query_start[b]), int(kv_len[b])
        if n <= 0 or c <= 0:
            continue
        for x in range(max(0, c - n) // page, (c - 1) // page + 1):
            if x >= table.shape[1] or not 0 <= table[b, x] < pages:
                continue
            pg = table[b, x]
            rows = k[pg, :min(page, c - x * page)].astype(np.float64)  # [n, heads, dim]
            for h in range(heads):
                r = rows[:, h]
                if not np.isfinite(r).all():
                    bounds[pg, h], scale[pg, h] = 0, np.inf
                    continue
                hi, lo = r.max(0), r.min(0)
                top = max(np.abs(hi).max(), np.abs(lo).max())
                scale[pg, h] = np.float32(top) * (np.float32(1) / np.float32(127))
                if top == 0:
                    bounds[pg, h] = 0
                else:
                    bounds[pg, h, 0], bounds[pg, h, 1] = np.floor(127 * lo / top), np.ceil(127 * hi / top)


def select_ref(q, bounds, scale, table, query_start, kv_len, count, page, window, sinks):
    """int32 [T, kv_heads, count]; rows that no request has are -7."""
    T, heads, dim = q.shape
    pages, kv_heads = scale.shape
    group = heads // kv_heads
    out = np.full((T, kv_heads, count), -7, np.int32)
    for b in range(len(kv_len)):
        n = int(query_start[b + 1]) - int(query_start[b])
        for i in range(n):
            t, p = int(query_start[b]) + i, int(kv_len[b]) - n + i
            if t >= T:
                continue
            cand = [x for x in range(table.shape[1]) if 0 <= table[b, x] < pages
                    and x * page <= p - window and (x + 1) * page > sinks]
            for h in range(kv_heads):
                score = []
                whole, steps = [], []
                for g in range(group):
                    v = q[t, h * group + g].astype(np.float64)
                    top = np.abs(v).max()
                    if not np.isfinite(top) or top == 0:
                        whole.append(np.zeros(dim, np.int64))
                        steps.append(np.float32(0))
                    else:
                        whole.append(np.rint(127 * v / top).astype(np.int64))
                        steps.append(np.float32(top) * (np.float32(1) / np.float32(127)))
                whole, steps = np.array(whole), np.array(steps, np.float32)
                pg = table[b, cand].astype(np.int64)
                lo, hi = bounds[pg, h, 0].astype(np.int64), bounds[pg, h, 1].astype(np.int64)
                dots = lo @ np.minimum(whole, 0).T + hi @ np.maximum(whole, 0).T  # [cand, group]
                best = (dots.astype(np.float32) * steps).max(1) if len(cand) else np.zeros(0, np.float32)
                s = scale[pg, h]
                with np.errstate(all="ignore"):
                    score = np.where(np.isinf(s), np.float32(np.inf), best * s)
                order = sorted(range(len(cand)), key=lambda x: (-score[x], cand[x]))[:count]
                got = sorted(cand[x] for x in order)
                out[t, h] = got + [-1] * (count - len(got))
    return out


def block_ids(blocks, page, heads, width):
    """The positions of blocks [T, kv_heads, count] as ids [T, heads, count * page], -1 where there are none."""
    T, kv_heads, count = blocks.shape
    ok = (blocks >= 0) & (blocks < width)  # past the table: past the context
    ids = np.where(ok, blocks, 0).astype(np.int64)[..., None] * page + np.arange(page)
    ids = np.where(ok[..., None], ids, -1).reshape(T, kv_heads, count * page)
    return np.repeat(ids, heads // kv_heads, 1)


def weights_ref(q, k, table, query_start, kv_len, lse, weights, *, window=-1, sinks=0, scale=None, held=None):
    """(weights in 64 bits after the step, tolerance of each): weights float32 [pages, heads, page] before it.  A term
    e^x is off by (|x| + 2) 2^-22 of itself (two 32-bit roundings of x, the exponential's 2^-22), a sum of n terms by
    n 2^-24 of itself."""
    T, heads, dim = q.shape
    pages, page, kv_heads, _ = k.shape
    group = heads // kv_heads
    scale = np.float32(dim ** -0.5 if scale is None else scale)
    w, tol = weights.astype(np.float64), np.zeros(weights.shape)
    for b in range(len(kv_len)):
        s, n, c = int(query_start[b]), int(query_start[b + 1]) - int(query_start[b]), int(kv_len[b])
        if n <= 0:
            continue
        from_zero = max(0, c - n) if held is None else max(0, int(held[b]))
        for j in range(c):
            if j // page >= table.shape[1] or not 0 <= table[b, j // page] < pages:
                continue
            pg, r = table[b, j // page], j % page
            p = np.arange(c - n, c)
            see = j <= p
            if window >= 0:
                see = see & ((p - j < window) | (j < sinks))
            t = s + np.flatnonzero(see)
            for h in range(kv_heads):
                old = 0.0 if j >= from_zero else float(weights[pg, h, r])
                if len(t) == 0 and j < from_zero:
                    continue
                l = lse[t, h * group:(h + 1) * group].astype(np.float64)
                with np.errstate(all="ignore"):
                    x = q[t, h * group:(h + 1) * group].astype(np.float64) @ k[pg, r, h].astype(np.float64) * float(scale) - l
                x = x[np.isfinite(l)]
                e = np.exp(x)
                w[pg, h, r] = old + e.sum()
                tol[pg, h, r] = (e * (np.abs(x) + 2)).sum() * 2.0 ** -22 + (n * group + 2) * 2.0 ** -24 * w[pg, h, r] + 1e-30
    return w, tol


def evict_ref(k, v, w, table, kv_len, budget, recent, sinks):
    """(kv_len, kept [R, heads, budget]); k, v [pages, page, heads, dim] and w [pages, heads, page] are updated in place."""
    pages, page, heads, _ = k.shape
    lens = np.minimum(np.maximum(kv_len, 0), table.shape[1] * page)
    kept = np.full((len(lens), heads, budget), -1, np.int32)
    for b, c in enumerate(lens):
        there = lambda j: 0 <= table[b, j // page] < pages  # noqa: E731
        for h in range(heads):
            if c <= budget:
                kept[b, h, :c] = np.arange(c)
                continue
            mid = list(range(sinks, c - recent))

            def rank(j):
                if not there(j):
                    return (1, 0.0, j)
                x = float(w[table[b, j // page], h, j % page])
                return (0, np.inf if np.isnan(x) else -x, j)
            mid = sorted(sorted(mid, key=rank)[:budget - sinks - recent])
            kept[b, h] = list(range(sinks)) + mid + list(range(c - recent, c))
            rows = [(k[table[b, j // page], j % page, h].copy(), v[table[b, j // page], j % page, h].copy(),
                     w[table[b, j // page], h, j % page]) if there(j) else None for j in kept[b, h]]
            for i, row in enumerate(rows):
                if row is not None and there(i):
                    at = table[b, i // page]
                    k[at, i % page, h], v[at, i % page, h], w[at, h, i % page] = row
    return np.minimum(lens, budget).astype(np.int32), kept
