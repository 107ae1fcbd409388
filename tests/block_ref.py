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
