"""Cases of the key/value cache and attention operators: what each has to compute, in plain torch operations and
through the package's own entry points.

Four operators, as a serving loop calls them for each step of a batch of requests: the step's plan (block tables and
slot maps from request lengths), the append of the new tokens' keys and values to the paged cache, the attention of
the new tokens over the cache (causal, with an optional sliding window and first tokens that stay visible), and the
attention over window, first tokens and the ids that a graph search returned for each query head.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one decode step of a small batch: every call costs little more than its launch
        dict(name="plan decode 8", op="plan", batch=8, ctx_lo=1, ctx_hi=4000, new_lo=1, new_hi=1, page=16, lens=1),
        # a step that admits many prompts beside running requests, chunks of up to 128 tokens
        dict(name="plan mixed 1000", op="plan", batch=1000, ctx_lo=0, ctx_hi=8000, new_lo=0, new_hi=128, page=32,
             lens=2),
        # the new tokens of a decode step
        dict(name="append decode 64", op="append", tokens=64, kv_heads=8, dim=128, page=16, pages=2048, fused=False,
             dtype="bf16", lens=3),
        # a prompt's chunk whose keys and values are slices of one fused projection, head size of the 96-d datasets
        dict(name="append chunk 16001", op="append", tokens=16001, kv_heads=4, dim=96, page=64, pages=640,
             fused=True, dtype="fp16", lens=4),
        # the smallest attention call: one user, one new token, a short context
        dict(name="decode 1 short", op="attend", batch=1, heads=8, kv_heads=2, dim=64, page=16, ctx_lo=200,
             ctx_hi=500, new_lo=1, new_hi=1, window=-1, sinks=0, dtype="bf16", lens=5),
        # a decode step of a busy server, ragged contexts
        dict(name="decode 64 ragged", op="attend", batch=64, heads=32, kv_heads=8, dim=128, page=16, ctx_lo=100,
             ctx_hi=8000, new_lo=1, new_hi=1, window=-1, sinks=0, dtype="bf16", lens=6),
        # one user with a very long context: few rows, one long axis
        dict(name="decode 1 long", op="attend", batch=1, heads=32, kv_heads=8, dim=128, page=64, ctx_lo=100001,
             ctx_hi=131071, new_lo=1, new_hi=1, window=-1, sinks=0, dtype="bf16", lens=7),
        # a prompt's chunk over the part of the prompt already in the cache
        dict(name="chunk 2048 on 8192", op="attend", batch=1, heads=32, kv_heads=8, dim=128, page=64, ctx_lo=8192,
             ctx_hi=8192, new_lo=2048, new_hi=2048, window=-1, sinks=0, dtype="bf16", lens=8),
        # prompts' chunks and decodes in one call, a layer with a sliding window and sinks, odd group of heads
        dict(name="mixed window sinks", op="attend", batch=24, heads=20, kv_heads=4, dim=96, page=32, ctx_lo=0,
             ctx_hi=5000, new_lo=1, new_hi=700, window=1000, sinks=4, dtype="fp16", lens=9),
        # one token of one user with ten retrieved ids for each head
        dict(name="retrieved 1x10", op="retrieve", batch=1, heads=8, kv_heads=2, dim=64, page=16, ctx_lo=2000,
             ctx_hi=3000, new_lo=1, new_hi=1, window=128, sinks=4, k=10, dtype="bf16", lens=10),
        # a decode step with the 100 ids that the search returns for each query head
        dict(name="retrieved 64x100", op="retrieve", batch=64, heads=32, kv_heads=8, dim=128, page=16, ctx_lo=4000,
             ctx_hi=16000, new_lo=1, new_hi=1, window=256, sinks=4, k=100, dtype="bf16", lens=11),
        # a few tokens per request (drafted ones), many ids, 96-d heads
        dict(name="retrieved few x512", op="retrieve", batch=9, heads=12, kv_heads=4, dim=96, page=32, ctx_lo=1000,
             ctx_hi=9000, new_lo=1, new_hi=5, window=64, sinks=16, k=512, dtype="fp16", lens=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "retrieve"])
    seed = rng.randrange(1 << 30)
    page = rng.choice([16, 32, 64])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "plan":
        new = rng.choice([1, _log(rng, 2, 128)])
        return dict(op=op, batch=_log(rng, 1, 1000), ctx_lo=0, ctx_hi=_log(rng, 10, 8000), new_lo=min(1, new),
                    new_hi=new, page=page, lens=seed)
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8])
    dim = rng.choice([64, 96, 128])
    if op == "append":
        tokens = _log(rng, 1, 16000)
        return dict(op=op, tokens=tokens, kv_heads=kv_heads, dim=dim, page=page, pages=tokens * 2 // page + 8,
                    fused=rng.random() < 0.5, dtype=dtype, lens=seed)
    base = dict(op=op, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, lens=seed)
    if op == "retrieve":
        batch = _log(rng, 1, 48)
        ctx = _log(rng, 200, 12000)
        return dict(base, batch=batch, ctx_lo=ctx // 3, ctx_hi=ctx, new_lo=1, new_hi=rng.choice([1, 1, 4]),
                    window=_log(rng, 1, 256), sinks=rng.choice([0, 1, 4, 16]),
                    k=_log(rng, 1, 100 if batch * group > 64 else 512))
    window = rng.choice([-1, -1, _log(rng, 1, 2000)])
    sinks = 0 if window < 0 else rng.choice([0, 4, 16])
    if rng.random() < 0.5:  # decode, or a few drafted tokens
        batch = _log(rng, 1, 64)
        ctx = _log(rng, 10, min(100000, 400000 // batch))
        return dict(base, batch=batch, ctx_lo=ctx // 4, ctx_hi=ctx, new_lo=1, new_hi=rng.choice([1, 1, 1, 4]),
                    window=window, sinks=sinks)
    batch = _log(rng, 1, 16)
    new = _log(rng, 8, 2048 // batch)
    ctx = _log(rng, 1, 8000)
    return dict(base, batch=batch, ctx_lo=ctx // 4, ctx_hi=ctx, new_lo=max(1, new // 4), new_hi=new, window=window,
                sinks=sinks)


def _lengths(case):
    """(tokens in the cache, new tokens) of each request: a fixed ragged set of the case, not of the seed."""
    r = random.Random(case["lens"])
    ctx = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["batch"])]
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["batch"])]
    if sum(new) == 0:
        new[0] = 1
    return ctx, new


def _pages(n, page):
    return -(-n // page)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    op, page = case["op"], case["page"]

    def ints(v, dtype=torch.int32):
        return torch.tensor(v, dtype=dtype, device=dev)

    if op == "append":
        dt, T, H, D = DTYPES[case["dtype"]], case["tokens"], case["kv_heads"], case["dim"]
        s = dict(op=op, page=page)
        shape = (case["pages"], page, H, D)
        s["k_cache"] = torch.randn(shape, generator=g, device=dev).to(dt)
        s["v_cache"] = torch.randn(shape, generator=g, device=dev).to(dt)
        if case["fused"]:  # [query | key | value] of one projection, two query heads for each key head
            qkv = torch.randn((T, 4 * H, D), generator=g, device=dev).to(dt)
            s["k"], s["v"] = qkv[:, 2 * H:3 * H], qkv[:, 3 * H:]
        else:
            s["k"] = torch.randn((T, H, D), generator=g, device=dev).to(dt)
            s["v"] = torch.randn((T, H, D), generator=g, device=dev).to(dt)
        # runs of consecutive slots in pages in no order; one token in 50 was refused
        order = torch.randperm(case["pages"], generator=g, device=dev)
        t = torch.arange(T, device=dev)
        slot = order[t // page] * page + t % page
        drop = torch.rand(T, generator=g, device=dev) < 0.02
        s["slot"] = torch.where(drop, torch.full_like(slot, -1), slot)
        return s

    ctx, new = _lengths(case)
    batch = case["batch"]
    had = [_pages(c, page) for c in ctx]
    will = [_pages(c + n, page) for c, n in zip(ctx, new)]
    width = max(will) + 3
    held = [had, will][op != "plan"]
    total = sum(will) + 32
    perm = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    taken = sum(held)
    # the pages that the requests hold, row by row; -1 beyond them
    hold = ints(held, torch.int64)
    start = torch.cumsum(hold, 0) - hold
    col = torch.arange(width, device=dev)
    table = torch.where(col[None, :] < hold[:, None], perm[(start[:, None] + col[None, :]).clamp(max=total - 1)], -1)
    s = dict(op=op, page=page, tokens=sum(new), max_new=max(new), max_kv=max(c + n for c, n in zip(ctx, new)))
    if op == "plan":
        # a pool nearly used up: an eighth of the pages that the step needs are missing, so its last requests wait
        need = sum(will) - sum(had)
        s.update(ctx=ints(ctx), new=ints(new), table=table.to(torch.int32).contiguous(),
                 free=perm[taken:taken + max(1, need - need // 8)].contiguous())
        return s
    dt, H, D = DTYPES[case["dtype"]], case["kv_heads"], case["dim"]
    T = sum(new)
    s["q"] = torch.randn((T, case["heads"], D), generator=g, device=dev).to(dt)
    s["k_cache"] = torch.randn((total, page, H, D), generator=g, device=dev).to(dt)
    s["v_cache"] = torch.randn((total, page, H, D), generator=g, device=dev).to(dt)
    s["table"] = table.to(torch.int32).contiguous()
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s["query_start"] = ints(starts)
    s["kv_len"] = ints([c + n for c, n in zip(ctx, new)])
    s["window"], s["sinks"], s["scale"] = case["window"], case["sinks"], D ** -0.5
    if op == "retrieve":
        # ids as a search returns them: positions of the context in order of distance, some repeated, some missing
        row_ctx = torch.repeat_interleave(ints(ctx), ints(new, torch.int64))
        u = torch.rand((T, case["heads"], case["k"]), generator=g, device=dev)
        ids = (u * row_ctx[:, None, None]).to(torch.int32)
        s["ids"] = torch.where(torch.rand(u.shape, generator=g, device=dev) < 0.02, torch.full_like(ids, -1), ids)
    return s


def run(s):
    if own:
        return _own(s)
    return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend, "retrieve": _plain_retrieve}[s["op"]](s)


def _own(s):
    import flashgann_b200 as fg
    if s["op"] == "plan":
        p = fg.kv_plan(s["ctx"], s["new"], s["table"], s["free"], tokens=s["tokens"], page_size=s["page"])
        return dict(query_start=p.query_start, kv_len=p.kv_len, position=p.position, slot=p.slot, head=p.free_head,
                    refused=p.refused, table=s["table"])
    if s["op"] == "append":
        fg.kv_append(s["k_cache"], s["v_cache"], s["k"], s["v"], s["slot"])
        return dict(k=s["k_cache"], v=s["v_cache"])
    if s["op"] == "attend":
        out, lse = fg.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["query_start"], s["kv_len"],
                                      s["max_new"], window=s["window"], sinks=s["sinks"], scale=s["scale"],
                                      return_lse=True)
    else:
        out, lse = fg.retrieved_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["query_start"],
                                          s["kv_len"], s["ids"], window=s["window"], sinks=s["sinks"],
                                          scale=s["scale"], return_lse=True)
    return dict(out=out, lse=lse)


def _plain_plan(s):
    ctx, new, table, free, page = s["ctx"].long(), s["new"].long(), s["table"], s["free"], s["page"]
    width, T = table.shape[1], s["tokens"]
    dev = table.device
    had = (ctx + page - 1) // page
    will = (ctx + new + page - 1) // page
    wide = will > width
    need = torch.where(wide, 0, will - had)
    first = torch.cumsum(need, 0) - need
    refused = wide | ((need > 0) & (first + need > free.numel()))
    take = torch.where(refused, 0, need)
    col = torch.arange(width, device=dev)
    fresh = (col >= had[:, None]) & (col < (had + take)[:, None])
    pick = (first[:, None] + col - had[:, None]).clamp(0, free.numel() - 1)
    table.copy_(torch.where(fresh, free[pick], table))
    end = torch.cumsum(new, 0)
    query_start = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), end])
    t = torch.arange(T, device=dev)
    r = torch.searchsorted(end, t, right=True).clamp(max=ctx.numel() - 1)
    gone = refused[r]
    pos = ctx[r] + t - query_start[r]
    slot = table[r, (pos // page).clamp(max=width - 1)].long() * page + pos % page
    return dict(query_start=query_start.int(), kv_len=torch.where(refused, 0, ctx + new).int(),
                position=torch.where(gone, -1, pos).int(), slot=torch.where(gone, -1, slot),
                head=take.sum().int().reshape(1), refused=refused.int(), table=table)


def _plain_append(s):
    page, ok = s["page"], s["slot"] >= 0
    at = s["slot"][ok]
    s["k_cache"][at // page, at % page] = s["k"][ok]
    s["v_cache"][at // page, at % page] = s["v"][ok]
    return dict(k=s["k_cache"], v=s["v_cache"])


def _softmax_times(scores, values, visible):
    """(weights @ values, log of the sum) over the visible scores; a row that sees nothing gives 0 and -inf."""
    scores = torch.where(visible, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    lse = (torch.log(total) + top).squeeze(-1)
    return torch.matmul(e, values) / torch.where(total == 0, 1.0, total), lse


def _plain_attend(s):
    q, table, page = s["q"], s["table"], s["page"]
    T, heads, D = q.shape
    H = s["k_cache"].shape[2]
    G, N, S = heads // H, s["max_new"], s["max_kv"]
    start, kv_len = s["query_start"].long(), s["kv_len"].long()
    B, dev = kv_len.numel(), q.device
    j = torch.arange(S, device=dev)
    at = table[:, j // page].long().clamp(min=0)
    k = s["k_cache"][at, j % page].float().permute(0, 2, 1, 3)  # [B, H, S, D]
    v = s["v_cache"][at, j % page].float().permute(0, 2, 1, 3)
    i = torch.arange(N, device=dev)
    new = start[1:] - start[:-1]
    row = (start[:-1, None] + i).clamp(max=T - 1)
    qp = q[row].float().view(B, N, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, N * G, D)
    p = (kv_len - new)[:, None] + i  # position of each new token
    see = j <= p[:, :, None]
    if s["window"] >= 0:
        see = see & ((j > p[:, :, None] - s["window"]) | (j < s["sinks"]))
    see = see.repeat_interleave(G, 1)[:, None]
    o, lse = _softmax_times(torch.matmul(qp, k.transpose(2, 3)) * s["scale"], v, see)
    t = torch.arange(T, device=dev)
    r = torch.searchsorted(start[1:], t, right=True)
    o = o.view(B, H, N, G, D).permute(0, 2, 1, 3, 4)[r, t - start[r]].reshape(T, heads, D)
    lse = lse.view(B, H, N, G).permute(0, 2, 1, 3)[r, t - start[r]].reshape(T, heads)
    return dict(out=o.to(q.dtype), lse=lse)


def _plain_retrieve(s):
    q, table, page, ids = s["q"], s["table"], s["page"], s["ids"].long()
    T, heads, D = q.shape
    H = s["k_cache"].shape[2]
    G, W, sinks, n = heads // H, s["window"], s["sinks"], ids.shape[2]
    start, kv_len = s["query_start"].long(), s["kv_len"].long()
    dev = q.device
    t = torch.arange(T, device=dev)
    r = torch.searchsorted(start[1:], t, right=True)
    p = kv_len[r] - start[r + 1] + t
    near = p[:, None] - torch.arange(W, device=dev)
    first = torch.arange(sinks, device=dev).expand(T, sinks)
    fixed = torch.cat([first, near], 1)[:, None].expand(T, heads, sinks + W)
    ok_first = first <= p[:, None]
    ok_near = near >= sinks
    ok_fixed = torch.cat([ok_first, ok_near], 1)[:, None].expand(T, heads, sinks + W)
    earlier = torch.ones((n, n), dtype=torch.bool, device=dev).tril(-1)
    again = ((ids[..., :, None] == ids[..., None, :]) & earlier).any(-1)
    ok_ids = (ids >= sinks) & (ids <= (p - W)[:, None, None]) & ~again
    j = torch.cat([fixed, ids], 2).clamp(min=0)
    see = torch.cat([ok_fixed, ok_ids], 2)
    at = table[r[:, None, None], (j // page).clamp(max=table.shape[1] - 1)].long().clamp(min=0)
    h = torch.arange(heads, device=dev)[None, :, None] // G
    k = s["k_cache"][at, j % page, h].float()
    v = s["v_cache"][at, j % page, h].float()
    o, lse = _softmax_times(torch.matmul(q.float()[:, :, None], k.transpose(2, 3)) * s["scale"], v, see[:, :, None])
    return dict(out=o[:, :, 0].to(q.dtype), lse=lse[:, :, 0])


def _visible_counts(case):
    """For each request: (sum over its new tokens of the keys that each sees, keys that any of them sees)."""
    ctx, new = _lengths(case)
    W, sinks, got = case["window"], case["sinks"], []
    for c, n in zip(ctx, new):
        if W < 0:
            got.append((n * c + n * (n + 1) // 2, c + n if n else 0))
            continue
        pairs = sum(min(p + 1, W) + min(sinks, max(0, p + 1 - W)) for p in range(c, c + n))
        low = max(0, c - W + 1)
        got.append((pairs, (c + n - low + min(sinks, low)) if n else 0))
    return got


def work(case):
    if case["op"] == "append":
        row = case["kv_heads"] * case["dim"] * 2
        return dict(bytes=case["tokens"] * (4 * row + 8), flops=0)
    ctx, new = _lengths(case)
    T, page, B = sum(new), case["page"], case["batch"]
    if case["op"] == "plan":
        need = sum(_pages(c + n, page) - _pages(c, page) for c, n in zip(ctx, new))
        # lengths and the pages taken in; starts, lengths, marks, new table entries, positions and slots out
        return dict(bytes=4 * (2 * B + need) + 4 * (3 * B + 1 + need) + 12 * T, flops=0)
    heads, H, D = case["heads"], case["kv_heads"], case["dim"]
    seen = _visible_counts(case)
    table = 4 * sum(_pages(c + n, page) for c, n in zip(ctx, new))
    bytes_ = T * heads * (2 * D * 2 + 4) + 4 * (2 * B + 1) + table
    if case["op"] == "attend":
        return dict(bytes=bytes_ + sum(u for _, u in seen) * H * D * 4, flops=4 * D * heads * sum(n for n, _ in seen))
    ids = T * heads * case["k"]
    pairs = heads * sum(n for n, _ in seen) + ids
    return dict(bytes=bytes_ + 4 * ids + (sum(n for n, _ in seen) * H + ids) * D * 4, flops=4 * D * pairs)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return None
    if case["op"] == "append":
        kept = torch.nonzero(s["slot"] >= 0)[:, 0]
        return {n: s[n + "_cache"].double().flatten(0, 1).index_copy_(0, s["slot"][kept], s[n][kept].double())
                .view(s[n + "_cache"].shape) for n in ("k", "v")}
    dev = s["q"].device
    ctx, new = _lengths(case)
    heads, H, page = case["heads"], case["kv_heads"], case["page"]
    outs, lses, at = [], [], 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        if n == 0:
            continue
        L = c + n
        pos = torch.arange(L, device=dev)
        rows = s["table"][b].long()[pos // page] * page + pos % page
        K = s["k_cache"].flatten(0, 1)[rows].double()
        V = s["v_cache"].flatten(0, 1)[rows].double()
        for lo in range(0, n, 256):
            hi = min(n, lo + 256)
            Q = s["q"][at + lo:at + hi].double()
            p = torch.arange(c + lo, c + hi, device=dev)[:, None]
            seen = pos[None, :] <= p
            if case["window"] >= 0:
                seen = seen & ((p - pos[None, :] < case["window"]) | (pos[None, :] < case["sinks"]))
            o = torch.zeros((hi - lo, heads, Q.shape[2]), dtype=torch.float64, device=dev)
            l = torch.zeros((hi - lo, heads), dtype=torch.float64, device=dev)
            for h in range(heads):
                see = seen
                if case["op"] == "retrieve":
                    ids = s["ids"][at + lo:at + hi, h].long()
                    mark = torch.zeros((hi - lo, L + 1), dtype=torch.bool, device=dev)
                    mark.scatter_(1, torch.where(ids < 0, L, ids), True)
                    see = seen | (mark[:, :L] & (pos[None, :] <= p))
                x = (Q[:, h] @ K[:, h * H // heads].T) * s["scale"]
                x = x.masked_fill(~see, -math.inf)
                l[:, h] = torch.logsumexp(x, 1)
                o[:, h] = torch.softmax(x, 1).nan_to_num(0.0) @ V[:, h * H // heads]
            outs.append(o)
            lses.append(l)
        at += n
    return dict(out=torch.cat(outs), lse=torch.cat(lses))
