"""The cache and attention operators from their definitions, row by row in 64
bits (numpy), and the inputs that their tests share."""

from __future__ import annotations

import math

import numpy as np


def plan_ref(ctx, new, table, free, head, page, tokens):
    """(query_start, kv_len, position, slot, free_head, refused); table is updated in place."""
    up = lambda n: -(-n // page)  # noqa: E731
    query_start, kv_len, refused = [0], [], []
    position, slot = [-1] * tokens, [-1] * tokens
    at, wanted = 0, 0  # pages taken, and pages wanted up to here
    left = max(0, len(free) - head)
    for b, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(0, c), max(0, n)
        wide = up(c + n) > table.shape[1]
        need = 0 if wide else up(c + n) - up(c)
        wanted += need
        no = wide or (need > 0 and wanted > left)
        refused.append(int(no))
        kv_len.append(0 if no else c + n)
        if not no:
            for i in range(need):
                table[b, up(c) + i] = free[head + at]
                at += 1
            for i in range(n):
                t = query_start[-1] + i
                if t < tokens:
                    position[t] = c + i
                    pg = int(table[b, (c + i) // page])
                    slot[t] = pg * page + (c + i) % page if pg >= 0 else -1
        query_start.append(query_start[-1] + n)
    return query_start, kv_len, position, slot, head + at, refused


def visible(p, window, sinks, ids=None):
    """Positions that a row at position p sees, ascending."""
    if p < 0:
        return []
    see = set(range(p + 1)) if window < 0 else {j for j in range(p + 1) if p - j < window or j < sinks}
    if ids is not None:
        see |= {int(j) for j in ids if 0 <= j <= p}
    return sorted(see)


def attention_ref(q, k_cache, v_cache, table, query_start, kv_len, *, window=-1, sinks=0, scale=None, ids=None):
    """(out [T, heads, dim], lse [T, heads], vmax [T, heads]) in float64; arrays in, page and head orders as the
    operators take them.  vmax: the largest |v| that the row sees, for tolerances.  Keys whose page is missing are
    not there; rows past the last request stay NaN."""
    T, heads, dim = q.shape
    pages, page, kv_heads, _ = k_cache.shape
    group = heads // kv_heads
    scale = dim ** -0.5 if scale is None else scale
    out = np.full((T, heads, dim), np.nan)
    lse = np.full((T, heads), np.nan)
    vmax = np.zeros((T, heads))
    for b in range(len(kv_len)):
        n = query_start[b + 1] - query_start[b]
        for i in range(n):
            t, p = query_start[b] + i, int(kv_len[b]) - n + i
            for h in range(heads):
                js = np.array([j for j in visible(p, window, sinks, None if ids is None else ids[t, h])
                               if j // page < table.shape[1] and 0 <= table[b, j // page] < pages], dtype=np.int64)
                out[t, h], lse[t, h] = 0.0, -np.inf
                if not len(js):
                    continue
                pg = table[b, js // page]
                with np.errstate(all="ignore"):
                    s = (k_cache[pg, js % page, h // group].astype(np.float64) @ q[t, h].astype(np.float64)) * scale
                    m = s.max()
                    if m == -np.inf:
                        continue
                    e = np.exp(s - m)
                    v = v_cache[pg, js % page, h // group].astype(np.float64)
                    out[t, h] = (e[:, None] * v).sum(0) / e.sum()
                    lse[t, h] = m + math.log(e.sum()) if e.sum() == e.sum() else np.nan
                vmax[t, h] = np.abs(v).max()
    return out, lse, vmax


def make(rng, *, ctx, new, heads, kv_heads, dim, page, spare=3, spread=1.0):
    """Queries, caches and a table with pages in no order, for requests of ctx + new tokens (float32 numpy, already
    rounded to what 16 bits hold in either type)."""
    total = [c + n for c, n in zip(ctx, new)]
    used = [-(-x // page) for x in total]
    width = max(used) + 1
    pages = sum(used) + spare
    perm = rng.permutation(pages)
    table = np.full((len(ctx), width), -1, dtype=np.int32)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = perm[at:at + u]
        at += u
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    T = int(start[-1])

    def draw(*shape):  # multiples of 1/32 up to +-4: exact in bfloat16 and float16
        return np.clip(np.round(rng.standard_normal(shape) * spread * 32) / 32, -3.96875, 3.96875).astype(np.float32)

    return dict(q=draw(T, heads, dim), k=draw(pages, page, kv_heads, dim), v=draw(pages, page, kv_heads, dim),
                table=table, start=start, kv_len=np.array(total, dtype=np.int32))
