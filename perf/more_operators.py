"""Cases of the operators that bound what a step of decoding reads from the key/value cache: what each has to compute,
in plain torch operations and through the package's own entry points.

Five operators, as a serving loop calls them.  Three attend over chosen pages of a long context: the summary of each
page's keys (bounds in 8 bits with a scale), the choice of the pages whose bound on the scores is highest, and the
attention over window, first tokens and those pages.  Two keep the cache short: the weight that each key was given so
far, and the eviction of the lightest keys of each kv head.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # the pages that a decode step of 64 requests wrote to
        dict(name="summarize decode 64", op="summarize", batch=64, ctx_lo=16, ctx_hi=500, new_lo=1, new_hi=1,
             kv_heads=8, dim=128, page=16, dtype="bf16", lens=1),
        # a prompt's pages, head size of the 96-d datasets
        dict(name="summarize prompt 16001", op="summarize", batch=1, ctx_lo=0, ctx_hi=0, new_lo=16001, new_hi=16001,
             kv_heads=4, dim=96, page=64, dtype="fp16", lens=2),
        # the smallest choice: one user, one new token
        dict(name="select 1 short", op="select", batch=1, heads=8, kv_heads=2, dim=64, page=16, ctx_lo=1000,
             ctx_hi=2000, new_lo=1, new_hi=1, window=128, sinks=4, count=16, dtype="bf16", lens=3),
        # a decode step of a busy server, ragged contexts
        dict(name="select 64 ragged", op="select", batch=64, heads=32, kv_heads=8, dim=128, page=16, ctx_lo=2000,
             ctx_hi=16000, new_lo=1, new_hi=1, window=256, sinks=4, count=64, dtype="bf16", lens=4),
        # one user with a very long context
        dict(name="select 1 long", op="select", batch=1, heads=32, kv_heads=8, dim=128, page=16, ctx_lo=100001,
             ctx_hi=131071, new_lo=1, new_hi=1, window=256, sinks=4, count=128, dtype="bf16", lens=5),
        # the attention after the smallest choice
        dict(name="blocks 1x16", op="blocks", batch=1, heads=8, kv_heads=2, dim=64, page=16, ctx_lo=1000, ctx_hi=2000,
             new_lo=1, new_hi=1, window=128, sinks=4, count=16, dtype="bf16", lens=6),
        # and after that of the busy server
        dict(name="blocks 64x64", op="blocks", batch=64, heads=32, kv_heads=8, dim=128, page=16, ctx_lo=2000,
             ctx_hi=16000, new_lo=1, new_hi=1, window=256, sinks=4, count=64, dtype="bf16", lens=7),
        # a few drafted tokens to a request, pages of 32, odd group
        dict(name="blocks drafted x33", op="blocks", batch=9, heads=12, kv_heads=4, dim=96, page=32, ctx_lo=1000,
             ctx_hi=9000, new_lo=1, new_hi=5, window=64, sinks=16, count=33, dtype="fp16", lens=8),
        # the weights of a decode step
        dict(name="weights decode 64", op="weights", batch=64, heads=32, kv_heads=8, dim=128, page=16, ctx_lo=100,
             ctx_hi=8000, new_lo=1, new_hi=1, window=-1, sinks=0, dtype="bf16", lens=9),
        # the weights that a prompt's last 64 tokens give to all of it
        dict(name="weights last 64 of 8192", op="weights", batch=1, heads=32, kv_heads=8, dim=128, page=64,
             ctx_lo=8128, ctx_hi=8128, new_lo=64, new_hi=64, window=-1, sinks=0, dtype="bf16", lens=10),
        # one request a little over its budget
        dict(name="evict 1 to 512", op="evict", batch=1, kv_heads=2, dim=64, page=16, ctx_lo=576, ctx_hi=576,
             budget=512, recent=128, sinks=4, dtype="bf16", lens=11),
        # a batch of prompts that are cut to the same budget
        dict(name="evict 32 to 1024", op="evict", batch=32, kv_heads=8, dim=128, page=16, ctx_lo=900, ctx_hi=8000,
             budget=1024, recent=256, sinks=4, dtype="bf16", lens=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["summarize", "select", "select", "blocks", "blocks", "weights", "weights", "evict"])
    seed = rng.randrange(1 << 30)
    page = rng.choice([16, 32, 64])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8])
    dim = rng.choice([64, 96, 128])
    base = dict(op=op, kv_heads=kv_heads, dim=dim, page=page, dtype=rng.choice(["bf16", "fp16"]), lens=seed)
    if op == "summarize":
        if rng.random() < 0.5:  # decode, or a few drafted tokens
            return dict(base, batch=_log(rng, 1, 64), ctx_lo=0, ctx_hi=_log(rng, 10, 2000), new_lo=1,
                        new_hi=rng.choice([1, 1, 4]))
        batch = _log(rng, 1, 8)
        new = _log(rng, 10, 16000 // batch)
        return dict(base, batch=batch, ctx_lo=0, ctx_hi=_log(rng, 1, 2000), new_lo=max(1, new // 3), new_hi=new)
    if op == "evict":
        batch = _log(rng, 1, 32)
        ctx = _log(rng, 20, min(32000, 150000 // batch))
        budget = max(2, int(ctx * rng.choice([0.1, 0.25, 0.5, 0.9])))
        recent = rng.randint(0, budget // 2)
        return dict(base, batch=batch, ctx_lo=ctx // 2, ctx_hi=ctx, budget=budget, recent=recent,
                    sinks=rng.choice([0, 1, 4]) if budget - recent > 8 else 0)
    base["heads"] = kv_heads * group
    window, sinks = _log(rng, 1, 1000), rng.choice([0, 1, 4, 16])
    if op == "weights":
        if rng.random() < 0.5:
            window, sinks = -1, 0
        if rng.random() < 0.5:  # decode
            batch = _log(rng, 1, 64)
            ctx = _log(rng, 10, min(100000, 400000 // batch))
            return dict(base, batch=batch, ctx_lo=ctx // 4, ctx_hi=ctx, new_lo=1, new_hi=rng.choice([1, 1, 4]),
                        window=window, sinks=sinks)
        batch = _log(rng, 1, 4)
        new = _log(rng, 8, 64 // batch)
        ctx = _log(rng, 1, 8000)
        return dict(base, batch=batch, ctx_lo=ctx // 4, ctx_hi=ctx, new_lo=max(1, new // 4), new_hi=new, window=window,
                    sinks=sinks)
    batch = _log(rng, 1, 64)
    new = rng.choice([1, 1, 1, 4]) if batch <= 12 else 1
    if op == "select":  # contexts with more pages than are chosen
        ctx = _log(rng, 64 * page, min(130000, max(65 * page, 500000 // batch)))
        window = min(window, ctx // 8)
        count = _log(rng, 1, min(128, (ctx // 4 - window) // page // 2))
    else:  # at most as many keys to a request as the largest listed case reads
        ctx = _log(rng, 50, min(60000, 500000 // batch))
        count = _log(rng, 1, 1024 // page)
    return dict(base, batch=batch, ctx_lo=ctx // 4, ctx_hi=ctx, new_lo=1, new_hi=new, window=min(window, 256),
                sinks=sinks, count=count)


def _lengths(case):
    """(tokens in the cache, new tokens) of each request: a fixed ragged set of the case, not of the seed."""
    r = random.Random(case["lens"])
    ctx = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["batch"])]
    new = [r.randint(case.get("new_lo", 0), case.get("new_hi", 0)) for _ in range(case["batch"])]
    return ctx, new


def _pages(n, page):
    return -(-n // page)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    op, page, H, D, dt = case["op"], case["page"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    ctx, new = _lengths(case)
    used = [_pages(c + n, page) for c, n in zip(ctx, new)]
    width, total = max(used) + 3, sum(used) + 8

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev)

    # pages in no order; -1 beyond those that a request holds
    perm = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    hold = ints(used).long()
    col = torch.arange(width, device=dev)
    at = ((torch.cumsum(hold, 0) - hold)[:, None] + col).clamp(max=total - 1)
    table = torch.where(col < hold[:, None], perm[at], -1).contiguous()
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s = dict(op=op, page=page, table=table, query_start=ints(starts), tokens=starts[-1], max_new=max(new),
             max_kv=max(c + n for c, n in zip(ctx, new)), kv_len=ints([c + n for c, n in zip(ctx, new)]))
    # the keys of a page have something in common, and channels differ in size
    size = 0.5 + torch.rand((H, D), generator=g, device=dev)
    s["k_cache"] = ((0.7 * randn(total, 1, H, D) + 0.7 * randn(total, page, H, D)) * size).to(dt)
    if op in ("summarize", "select"):
        if op == "select":
            s["bounds"], s["scale"] = _bounds(s["k_cache"].float(), torch.ones((total, page), dtype=torch.bool, device=dev))
            del s["k_cache"]
        else:
            s["bounds"] = torch.zeros((total, H, 2, D), dtype=torch.int8, device=dev)
            s["scale"] = torch.zeros((total, H), device=dev)
    if op in ("blocks", "evict"):
        s["v_cache"] = randn(total, page, H, D).to(dt)
    if op == "evict":
        # a few keys get most of the weight
        s["weights"] = torch.exp(2 * randn(total, H, page))
        s.update(budget=case["budget"], recent=case["recent"], sinks=case["sinks"])
        return s
    if op == "summarize":
        return s
    T = starts[-1]
    s["q"] = randn(T, case["heads"], D).to(dt)
    s["window"], s["sinks"], s["softmax_scale"] = case["window"], case["sinks"], D ** -0.5
    if op == "select":
        s["count"] = case["count"]
    if op == "blocks":
        # as a choice leaves them: pages with keys outside of window and first tokens, ascending, then -1
        row_new = ints(new).long()
        pos = torch.repeat_interleave(ints(ctx).long(), row_new) + torch.arange(T, device=dev) - torch.repeat_interleave(
            s["query_start"][:-1].long(), row_new)
        can = (col >= s["sinks"] // page) & (col <= ((pos - s["window"]) // page)[:, None])
        u = torch.where(can[:, None], torch.rand((T, H, width), generator=g, device=dev), 2.0)
        got, which = torch.sort(u, dim=2)
        which = torch.where(got < 2.0, which, width)[:, :, :case["count"]]
        which = torch.nn.functional.pad(which, (0, case["count"] - which.shape[2]), value=width)
        which = torch.sort(which, dim=2).values
        s["blocks"] = torch.where(which < width, which, -1).int().contiguous()
    if op == "weights":
        s["weights"] = torch.rand((total, H, page), generator=g, device=dev)
        s["lse"] = _lse(s, ctx, new)
    return s


def _lse(s, ctx, new):
    """What the attention of the step left: log of each row's sum."""
    heads, H, page = s["q"].shape[1], s["k_cache"].shape[2], s["page"]
    got, at = [], 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        j = torch.arange(c + n, device=s["q"].device)
        k = s["k_cache"][s["table"][b, j // page].long(), j % page].float().repeat_interleave(heads // H, 1)
        x = torch.einsum("nhd,jhd->nhj", s["q"][at:at + n].float(), k) * s["softmax_scale"]
        see = _sees(c + torch.arange(n, device=j.device)[:, None], j, s["window"], s["sinks"])
        got.append(torch.logsumexp(x.masked_fill(~see[:, None], -math.inf), -1))
        at += n
    return torch.cat(got).contiguous()


def _sees(p, j, window, sinks):
    see = j <= p
    return see if window < 0 else see & ((p - j < window) | (j < sinks))


def run(s):
    if own:
        return _own(s)
    return {"summarize": _plain_summarize, "select": _plain_select, "blocks": _plain_blocks, "weights": _plain_weights,
            "evict": _plain_evict}[s["op"]](s)


def _values(s):
    """The bounds as the values that they stand for."""
    return dict(bounds=s["bounds"] * s["scale"][:, :, None, None], scale=s["scale"])


def _own(s):
    import flashgann_b200 as fg
    if s["op"] == "summarize":
        fg.kv_summarize(s["k_cache"], s["bounds"], s["scale"], s["table"], s["query_start"], s["kv_len"],
                        tokens=s["tokens"])
        return _values(s)
    if s["op"] == "select":
        return fg.select_blocks(s["q"], s["bounds"], s["scale"], s["table"], s["query_start"], s["kv_len"], s["count"],
                                page_size=s["page"], window=s["window"], sinks=s["sinks"])
    if s["op"] == "blocks":
        out, lse = fg.block_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["query_start"], s["kv_len"],
                                      s["blocks"], window=s["window"], sinks=s["sinks"], scale=s["softmax_scale"],
                                      return_lse=True)
        return dict(out=out, lse=lse)
    if s["op"] == "weights":
        fg.attention_weights(s["q"], s["k_cache"], s["weights"], s["table"], s["query_start"], s["kv_len"], s["lse"],
                             window=s["window"], sinks=s["sinks"], scale=s["softmax_scale"])
        return s["weights"]
    e = fg.kv_evict(s["k_cache"], s["v_cache"], s["weights"], s["table"], s["kv_len"], s["budget"],
                    recent=s["recent"], sinks=s["sinks"])
    return dict(k=s["k_cache"], v=s["v_cache"], weights=s["weights"], kv_len=e.kv_len, kept=e.kept)


def _bounds(k, valid):
    """(bounds int8 [.., heads, 2, dim] (lower, upper), scale [.., heads]) of pages of keys [.., page, heads, dim]."""
    hi = torch.where(valid[..., None, None], k, -math.inf).amax(-3)
    lo = torch.where(valid[..., None, None], k, math.inf).amin(-3)
    top = torch.maximum(hi.abs(), lo.abs()).amax(-1)
    fine = torch.isfinite(top)
    scale = torch.where(fine, top / 127, math.inf)
    # 127 x / top with a product that is exact, so that what is rounded up or down is the quotient itself
    by = torch.where(fine & (top > 0), top / 128, 1.0)[..., None]
    up = torch.where(fine[..., None], torch.ceil(hi * (127 / 128) / by), 0.0)
    down = torch.where(fine[..., None], torch.floor(lo * (127 / 128) / by), 0.0)
    return torch.stack([down, up], -2).to(torch.int8), scale


def _plain_summarize(s):
    page, table, kv_len, start = s["page"], s["table"], s["kv_len"].long(), s["query_start"].long()
    dev = table.device
    new = start[1:] - start[:-1]
    first = (kv_len - new) // page
    most = (s["max_new"] + page - 2) // page + 1  # pages that new tokens of a request can lie in
    col = first[:, None] + torch.arange(most, device=dev)
    pages = torch.gather(table.long(), 1, col.clamp(max=table.shape[1] - 1))
    ok = (col <= ((kv_len - 1) // page)[:, None]) & (new > 0)[:, None] & (pages >= 0)
    valid = col[..., None] * page + torch.arange(page, device=dev) < kv_len[:, None, None]
    bounds, scale = _bounds(s["k_cache"][pages.clamp(min=0)].float(), valid)
    s["bounds"][pages[ok]] = bounds[ok]
    s["scale"][pages[ok]] = scale[ok]
    return _values(s)


def _plain_select(s):
    q, table, page, window, sinks, count = s["q"].float(), s["table"], s["page"], s["window"], s["sinks"], s["count"]
    T, heads, D = q.shape
    H, W, dev = s["bounds"].shape[1], table.shape[1], q.device
    G, N, R = heads // H, s["max_new"], table.shape[0]
    start, kv_len = s["query_start"].long(), s["kv_len"].long()
    top = q.abs().amax(-1)
    top = torch.where(torch.isfinite(top), top, 0.0)
    step = top / 127
    whole = torch.where((top > 0)[..., None], torch.round(q * (127 / 128) / torch.where(top > 0, top / 128, 1.0)[..., None]), 0.0)
    # rows of a request beside each other, so that its pages are read once
    i = torch.arange(N, device=dev)
    row = (start[:-1, None] + i).clamp(max=T - 1)
    x = whole[row].view(R, N, H, G, D).permute(0, 2, 1, 3, 4).reshape(R, H, N * G, D)
    sides = s["bounds"][table.long().clamp(min=0)].float().permute(0, 2, 3, 4, 1)  # [R, H, 2, D, W]
    dots = torch.matmul(x.clamp(max=0), sides[:, :, 0]) + torch.matmul(x.clamp(min=0), sides[:, :, 1])  # whole numbers
    t = step[row].view(R, N, H, G).permute(0, 2, 1, 3)
    best = (dots.view(R, H, N, G, W) * t[..., None]).amax(3)
    scale = s["scale"][table.long().clamp(min=0)].permute(0, 2, 1)[:, :, None]  # [R, H, 1, W]
    score = torch.where(scale == math.inf, math.inf, best * torch.where(scale == math.inf, 1.0, scale))
    p = (kv_len - (start[1:] - start[:-1]))[:, None] + i
    col = torch.arange(W, device=dev)
    can = (col >= sinks // page) & (col <= ((p - window) // page)[..., None]) & (table >= 0)[:, None]  # [R, N, W]
    # candidates first, by score, ties to the lowest page
    order = torch.sort(torch.where(can[:, None], score, -math.inf), dim=-1, descending=True, stable=True).indices
    picked = torch.where(torch.gather(can[:, None].expand(R, H, N, W), 3, order), order, W)[..., :count]
    picked = torch.nn.functional.pad(picked, (0, count - picked.shape[-1]), value=W)
    picked = torch.sort(picked, dim=-1).values
    picked = torch.where(picked < W, picked, -1).permute(0, 2, 1, 3)  # [R, N, H, count]
    t = torch.arange(T, device=dev)
    r = torch.searchsorted(start[1:], t, right=True)
    return picked[r, t - start[r]].int()


def _plain_blocks(s):
    q, table, page, blocks = s["q"], s["table"], s["page"], s["blocks"].long()
    T, heads, D = q.shape
    H, n = blocks.shape[1], blocks.shape[2]
    G, W, sinks, dev = heads // H, s["window"], s["sinks"], q.device
    start, kv_len = s["query_start"].long(), s["kv_len"].long()
    t = torch.arange(T, device=dev)
    r = torch.searchsorted(start[1:], t, right=True)
    p = kv_len[r] - start[r + 1] + t
    near = p[:, None] - torch.arange(W, device=dev)
    first = torch.arange(sinks, device=dev).expand(T, sinks)
    fixed = torch.cat([first, near], 1)[:, None].expand(T, H, sinks + W)
    ok_fixed = torch.cat([first <= p[:, None], near >= sinks], 1)[:, None].expand(T, H, sinks + W)
    earlier = torch.ones((n, n), dtype=torch.bool, device=dev).tril(-1)
    again = ((blocks[..., :, None] == blocks[..., None, :]) & earlier).any(-1)
    chosen = (blocks[..., None] * page + torch.arange(page, device=dev))  # [T, H, n, page]
    ok = ((blocks >= 0) & ~again)[..., None] & (chosen >= sinks) & (chosen <= (p - W)[:, None, None, None])
    j = torch.cat([fixed, chosen.flatten(2)], 2).clamp(min=0)
    see = torch.cat([ok_fixed, ok.flatten(2)], 2)
    at = table[r[:, None, None], (j // page).clamp(max=table.shape[1] - 1)].long().clamp(min=0)
    h = torch.arange(H, device=dev)[None, :, None]
    k = s["k_cache"][at, j % page, h].float()
    v = s["v_cache"][at, j % page, h].float()
    x = torch.matmul(q.float().view(T, H, G, D), k.transpose(2, 3)) * s["softmax_scale"]
    x = torch.where(see[:, :, None], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e, v) / torch.where(total == 0, 1.0, total)
    lse = (torch.log(total) + top).squeeze(-1)
    return dict(out=out.view(T, heads, D).to(q.dtype), lse=lse.view(T, heads))


def _plain_weights(s):
    q, table, page = s["q"], s["table"], s["page"]
    T, heads, D = q.shape
    H = s["k_cache"].shape[2]
    G, N, S, dev = heads // H, s["max_new"], s["max_kv"], q.device
    start, kv_len = s["query_start"].long(), s["kv_len"].long()
    B = kv_len.numel()
    j = torch.arange(S, device=dev)
    at = table[:, j // page].long().clamp(min=0)
    k = s["k_cache"][at, j % page].float().permute(0, 2, 1, 3)  # [B, H, S, D]
    i = torch.arange(N, device=dev)
    new = start[1:] - start[:-1]
    row = (start[:-1, None] + i).clamp(max=T - 1)
    x = q[row].float().view(B, N, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, N * G, D)
    lse = s["lse"][row].view(B, N, H, G).permute(0, 2, 1, 3).reshape(B, H, N * G, 1)
    p = (kv_len - new)[:, None] + i
    see = _sees(p[:, :, None], j, s["window"], s["sinks"]) & (i < new[:, None])[:, :, None]
    see = see.repeat_interleave(G, 1)[:, None] & torch.isfinite(lse)
    e = torch.exp(torch.matmul(x, k.transpose(2, 3)) * s["softmax_scale"] - torch.where(torch.isfinite(lse), lse, 0.0))
    got = torch.where(see, e, 0.0).sum(2)  # [B, H, S]
    held = s["weights"][at[:, None], torch.arange(H, device=dev)[None, :, None], (j % page)[None, None]]
    got = got + torch.where(j < (kv_len - new)[:, None, None], held, 0.0)
    b, jj = torch.nonzero((j < kv_len[:, None]) & (table[:, j // page] >= 0), as_tuple=True)
    s["weights"][at[b, jj], :, jj % page] = got[b, :, jj]
    return s["weights"]


def _plain_evict(s):
    table, page, kv_len, budget = s["table"], s["page"], s["kv_len"].long(), s["budget"]
    H, S, dev = s["weights"].shape[1], s["max_kv"], table.device
    j = torch.arange(S, device=dev)
    h = torch.arange(H, device=dev)[:, None]
    at = table[:, j // page].long().clamp(min=0)
    w = s["weights"][at[:, None], h, j % page].double()  # [B, H, S]
    w = torch.where(torch.isnan(w), -math.inf, w).clamp(max=1e300)
    always = (j < s["sinks"]) | (j >= (kv_len - s["recent"])[:, None])
    inside = j < kv_len[:, None]
    w = torch.where(always[:, None], math.inf, w)
    w = torch.where(inside[:, None], w, -math.inf)
    order = torch.sort(w, dim=2, descending=True, stable=True).indices[:, :, :budget]
    order = torch.where(order < kv_len[:, None, None], order, S)
    order = torch.nn.functional.pad(order, (0, budget - order.shape[2]), value=S)
    kept = torch.sort(order, dim=2).values  # [B, H, budget]
    kept = torch.where(kept < S, kept, -1)
    src, to = kept.clamp(min=0), torch.arange(budget, device=dev)
    b = torch.arange(table.shape[0], device=dev)[:, None, None]
    here = table[b, src // page].long().clamp(min=0)
    there = table[b, (to // page).clamp(max=table.shape[1] - 1)].long().expand(kept.shape)
    rows = to.expand(kept.shape) % page
    heads = h.expand(kept.shape)
    ok = (kept >= 0) & (kv_len > budget)[:, None, None]
    for name in ("k_cache", "v_cache"):
        s[name][there[ok], rows[ok], heads[ok]] = s[name][here, src % page, heads][ok]
    s["weights"][there[ok], heads[ok], rows[ok]] = s["weights"][here, heads, src % page][ok]
    return dict(k=s["k_cache"], v=s["v_cache"], weights=s["weights"], kv_len=kv_len.clamp(max=budget).int(), kept=kept.int())


def _seen(case, p):
    """Keys that a token at position p sees by window and first tokens."""
    W, sinks = case["window"], case["sinks"]
    return p + 1 if W < 0 else min(p + 1, W) + min(sinks, max(0, p + 1 - W))


def _candidates(case, p):
    """Pages that hold a key outside of window and first tokens."""
    return max(0, (p - case["window"]) // case["page"] - case["sinks"] // case["page"] + 1) if p >= case["window"] else 0


def work(case):
    ctx, new = _lengths(case)
    op, page, H, D, B = case["op"], case["page"], case["kv_heads"], case["dim"], case["batch"]
    T = sum(new)
    if op == "evict":
        kept = sum(min(c, case["budget"]) for c in ctx if c > case["budget"])
        table = 4 * sum(_pages(c, page) for c in ctx)
        return dict(bytes=H * (4 * sum(c for c in ctx if c > case["budget"]) + kept * (2 * 4 * D + 4) + 4 * case["budget"] * B)
                    + table + 8 * B, flops=0)
    if op == "summarize":
        rows = pages = 0
        for c, n in zip(ctx, new):
            if n:
                rows += c + n - c // page * page
                pages += _pages(c + n, page) - c // page
        return dict(bytes=H * (rows * D * 2 + pages * (2 * D + 4)) + 4 * (2 * B + 1 + pages), flops=2 * H * D * rows)
    heads = case["heads"]
    positions = [range(c, c + n) for c, n in zip(ctx, new)]
    if op == "select":
        read = sum(max([_candidates(case, p) for p in r], default=0) for r in positions)
        dots = sum(_candidates(case, p) for r in positions for p in r)
        return dict(bytes=T * heads * D * 2 + read * (4 + H * (2 * D + 4)) + 4 * T * H * case["count"] + 4 * (2 * B + 1),
                    flops=2 * heads * D * dots)
    if op == "blocks":
        keys = [_seen(case, p) + min(case["count"], _candidates(case, p)) * page for r in positions for p in r]
        return dict(bytes=T * heads * (4 * D + 4) + 4 * T * H * case["count"] + sum(keys) * (4 * D * H + 4 // page)
                    + 4 * (2 * B + 1), flops=4 * D * heads * sum(keys))
    pairs = sum(_seen(case, p) for r in positions for p in r)
    keys = 0  # that any of a request's new tokens sees
    for c, n in zip(ctx, new):
        low = max(0, c - case["window"] + 1) if case["window"] >= 0 else 0
        keys += (c + n - low + min(case["sinks"], low)) if n else 0
    return dict(bytes=T * heads * (2 * D + 4) + H * keys * (2 * D + 8) + 4 * (keys // page + 2 * B + 1),
                flops=2 * D * heads * pairs)


def exact(case, seed):
    if case["op"] == "select":
        return None
    s = prepare(case, seed)
    ctx, new = _lengths(case)
    page, H, table = case["page"], case["kv_heads"], s["table"].long()
    if case["op"] == "summarize":
        bounds, scale = s["bounds"].double(), s["scale"].double()
        for b, (c, n) in enumerate(zip(ctx, new)):
            for x in range(c // page, _pages(c + n, page)):
                k = s["k_cache"][table[b, x], :min(page, c + n - x * page)].double()
                a = k.abs().amax((0, 2))[:, None]
                bounds[table[b, x], :, 0] = torch.floor(127 * k.amin(0) / a) * a / 127
                bounds[table[b, x], :, 1] = torch.ceil(127 * k.amax(0) / a) * a / 127
                scale[table[b, x]] = a[:, 0] / 127
        return dict(bounds=bounds, scale=scale)
    if case["op"] == "evict":
        k, v, w = s["k_cache"].double(), s["v_cache"].double(), s["weights"].double()
        kept = torch.full((len(ctx), H, case["budget"]), -1, dtype=torch.int32, device=k.device)
        for b, c in enumerate(ctx):
            for h in range(H):
                pos = torch.arange(c, device=k.device)
                if c > case["budget"]:
                    mid = torch.arange(case["sinks"], c - case["recent"], device=k.device)
                    best = torch.argsort(w[table[b, mid // page], h, mid % page], descending=True, stable=True)
                    mid = mid[best[:case["budget"] - case["sinks"] - case["recent"]]]
                    pos = torch.cat([pos[:case["sinks"]], torch.sort(mid).values, pos[c - case["recent"]:]])
                    to = torch.arange(case["budget"], device=k.device)
                    for x in (k, v):
                        x[table[b, to // page], to % page, h] = x[table[b, pos // page], pos % page, h]
                    w[table[b, to // page], h, to % page] = w[table[b, pos // page], h, pos % page]
                kept[b, h, :len(pos)] = pos.int()
        return dict(k=k, v=v, weights=w, kept=None, kv_len=None)
    heads = case["heads"]
    outs, lses, at = [], [], 0
    w = s["weights"].double() if case["op"] == "weights" else None
    for b, (c, n) in enumerate(zip(ctx, new)):
        pos = torch.arange(c + n, device=table.device)
        pg, rows = table[b, pos // page], pos % page
        K = s["k_cache"][pg, rows].double()
        Q = s["q"][at:at + n].double()
        p = torch.arange(c, c + n, device=table.device)[:, None]
        seen = pos <= p
        if case["window"] >= 0:
            seen = seen & ((p - pos < case["window"]) | (pos < case["sinks"]))
        if case["op"] == "weights":
            for h in range(H):
                x = torch.einsum("ngd,jd->ngj", Q[:, h * heads // H:(h + 1) * heads // H], K[:, h]) * s["softmax_scale"]
                e = torch.exp(x - s["lse"][at:at + n, h * heads // H:(h + 1) * heads // H, None].double())
                add = e.masked_fill(~seen[:, None], 0.0).sum((0, 1))
                w[pg, h, rows] = torch.where(pos < c, w[pg, h, rows], 0.0) + add
        else:
            V = s["v_cache"][pg, rows].double()
            o = torch.zeros((n, heads, Q.shape[2]), dtype=torch.float64, device=table.device)
            l = torch.zeros((n, heads), dtype=torch.float64, device=table.device)
            for h in range(H):
                mark = torch.zeros((n, _pages(c + n, page) + 1), dtype=torch.bool, device=table.device)
                mark.scatter_(1, s["blocks"][at:at + n, h].long() % mark.shape[1], True)  # -1: the last place, beyond all
                see = seen | (mark[:, pos // page] & (pos <= p))
                for y in range(h * heads // H, (h + 1) * heads // H):
                    x = ((Q[:, y] @ K[:, h].T) * s["softmax_scale"]).masked_fill(~see, -math.inf)
                    l[:, y] = torch.logsumexp(x, 1)
                    o[:, y] = torch.softmax(x, 1) @ V[:, h]
            outs.append(o)
            lses.append(l)
        at += n
    return w if w is not None else dict(out=torch.cat(outs), lse=torch.cat(lses))
