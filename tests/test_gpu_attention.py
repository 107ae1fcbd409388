"""The paged cache and its attention on the GPU against their definitions in
64 bits: types, head layouts, lengths, masks that leave rows empty, strides,
what masked places hold, streams, and repeatability.

Tolerances.  Inputs are exact in both 16-bit types.  The weights of the second
product are rounded to the type (unit roundoff u = 2^-8 or 2^-11) and sum to
one, and so is the result: |error| <= 2 u max|v| over the visible v; 32-bit
sums and exponentials of scores below about 30 add less than 2e-4 max|v|, and
less than 2e-4 to a log-sum-exp."""

from __future__ import annotations

import numpy as np
import pytest

from tests.attention_ref import attention_ref, make, plan_ref

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}


def _dt(name):
    import torch
    return {"bf16": torch.bfloat16, "fp16": torch.float16}[name]


def _cuda(a, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def _check(out, lse, ref, dtype, rows=None):
    o, l, vmax = ref
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    if rows is not None:
        o, l, vmax, out, lse = o[rows], l[rows], vmax[rows], out[rows], lse[rows]
    assert np.array_equal(np.isnan(o), np.isnan(out))
    fine = np.isfinite(o)
    assert np.array_equal(out[~fine & ~np.isnan(o)], o[~fine & ~np.isnan(o)])
    err = np.abs(np.where(fine, out - np.where(fine, o, 0), 0))
    tol = (2 * U[dtype] + 2e-4) * np.where(np.isfinite(vmax), vmax, 4.0)[..., None]
    assert (err <= tol).all(), f"worst {np.max(err / np.maximum(tol, 1e-30)):.2f} of the tolerance"
    fl = np.isfinite(l)
    assert np.array_equal(np.isneginf(l), np.isneginf(lse)) and np.array_equal(np.isnan(l), np.isnan(lse))
    assert (np.abs(lse[fl] - l[fl]) <= 2e-4).all()


def _run(x, dtype, *, window=-1, sinks=0, scale=None, ids=None, max_new=None, order="phd", **kw):
    """The operator on the arrays of make(); order: the cache's axes in memory (p page row, h head, d dim)."""
    import torch
    import flashgann_b200 as fg
    dt = _dt(dtype)
    k, v = _cuda(x["k"], dt), _cuda(x["v"], dt)
    if order == "hpd":
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    elif order == "joined":  # K and V of a page beside each other
        kv = torch.stack([k, v], 1)
        k, v = kv[:, 0], kv[:, 1]
    args = (_cuda(x["q"], dt), k, v, _cuda(x["table"]), _cuda(x["start"]), _cuda(x["kv_len"]))
    if ids is None:
        mn = int(np.max(np.diff(x["start"]))) if max_new is None else max_new
        return fg.paged_attention(*args, mn, window=window, sinks=sinks, scale=scale, return_lse=True, **kw)
    return fg.retrieved_attention(*args, _cuda(ids), window=window, sinks=sinks, scale=scale, return_lse=True, **kw)


def _ref(x, **kw):
    return attention_ref(x["q"], x["k"], x["v"], x["table"], x["start"], x["kv_len"], **kw)


# ---- plan and append ----

@pytest.mark.parametrize("R,page,width,short,seed", [
    (1, 16, 9, 0, 0), (2, 1, 60, 0, 1), (33, 8, 12, 0, 2), (33, 8, 12, 40, 3), (700, 16, 7, 300, 4),
    (257, 32, 4, 0, 5), (1, 16, 3, 99, 6), (3000, 64, 2, 500, 7)])
def test_plan(R, page, width, short, seed):
    import flashgann_b200 as fg
    rng = np.random.default_rng(seed)
    top = page * width
    ctx = rng.integers(0, top, R).astype(np.int32)
    new = (rng.integers(0, max(2, top // 3), R) * (rng.random(R) < 0.7)).astype(np.int32)
    ctx[rng.random(R) < 0.1] = 0
    new[rng.random(R) < 0.05] = top + 5  # never fits
    ctx[rng.random(R) < 0.02] = -3       # counts as none
    head = int(rng.integers(0, 4))
    table = np.full((R, width), -1, dtype=np.int32)
    for b in range(R):
        n = -(-max(0, int(ctx[b])) // page)
        table[b, :n] = rng.integers(0, 10000, n)
    need = sum(max(0, -(-(max(0, c) + n) // page) - -(-max(0, c) // page)) for c, n in zip(ctx.tolist(), new.tolist()))
    free = rng.permutation(50000)[:max(1, head + need - short)].astype(np.int32)
    for tokens in {int(new.sum()), int(new.sum()) + 7, max(0, int(new.sum()) - 3)}:
        want_table = table.copy()
        want = plan_ref(ctx.tolist(), new.tolist(), want_table, free, head, page, tokens)
        got_table = _cuda(table)
        p = fg.kv_plan(_cuda(ctx), _cuda(new), got_table, _cuda(free), tokens=tokens, page_size=page,
                       free_head=_cuda(np.array([head], np.int32)))
        assert np.array_equal(got_table.cpu().numpy(), want_table)
        for name, w in zip(("query_start", "kv_len", "position", "slot", "free_head", "refused"), want):
            assert np.array_equal(getattr(p, name).cpu().numpy().ravel(), np.array(w).ravel()), (name, tokens)


def test_plan_slots_pass_32_bits():
    import flashgann_b200 as fg
    table = _cuda(np.array([[2 ** 31 - 1]], np.int32))
    p = fg.kv_plan(_cuda(np.array([3], np.int32)), _cuda(np.array([2], np.int32)), table, _cuda(np.array([1], np.int32)),
                   tokens=2, page_size=16)
    assert p.slot.tolist() == [(2 ** 31 - 1) * 16 + 3, (2 ** 31 - 1) * 16 + 4]


@pytest.mark.parametrize("dim,heads,page,tokens,dtype,order,fused", [
    (64, 1, 1, 1, "bf16", "phd", False), (96, 3, 8, 77, "fp16", "hpd", True), (128, 8, 16, 300, "bf16", "joined", True),
    (128, 2, 64, 5000, "fp16", "phd", False), (96, 4, 32, 4097, "bf16", "joined", False)])
def test_append(dim, heads, page, tokens, dtype, order, fused):
    import torch
    import flashgann_b200 as fg
    dt = _dt(dtype)
    pages = -(-tokens // page) + 2
    g = torch.Generator(device="cuda").manual_seed(tokens)
    shape = (pages, page, heads, dim)
    k, v = torch.randn(shape, generator=g, device="cuda").to(dt), torch.randn(shape, generator=g, device="cuda").to(dt)
    if order == "hpd":
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    elif order == "joined":
        kv = torch.stack([k, v], 1)
        k, v = kv[:, 0], kv[:, 1]
    rows = torch.randn((tokens, 4 * heads, dim), generator=g, device="cuda").to(dt)
    nk, nv = rows[:, heads:2 * heads], rows[:, 3 * heads:]
    if not fused:
        nk, nv = nk.contiguous(), nv.contiguous()
    slot = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    slot[::7] = -1
    slot[3::11] = pages * page + 5
    want = [t.clone().reshape(pages * page, heads, dim) for t in (k, v)]
    ok = (slot >= 0) & (slot < pages * page)
    want[0][slot[ok]], want[1][slot[ok]] = nk[ok], nv[ok]
    fg.kv_append(k, v, nk, nv, slot)
    assert torch.equal(k.reshape(pages * page, heads, dim), want[0])
    assert torch.equal(v.reshape(pages * page, heads, dim), want[1])


def test_append_misaligned_rows():
    """Rows that do not start on 16 bytes are copied first, the result is the same."""
    import torch
    import flashgann_b200 as fg
    k, v = (torch.zeros((4, 8, 2, 64), dtype=torch.float16, device="cuda") for _ in range(2))
    flat = torch.arange(5 * 2 * 64 + 1, device="cuda").to(torch.float16)
    rows = flat[1:].view(5, 2, 64)
    fg.kv_append(k, v, rows, rows, torch.arange(5, device="cuda"))
    assert torch.equal(k[0, :5], rows) and torch.equal(v[0, :5], rows) and not k[1:].any()


# ---- attention ----

# (ctx, new, heads, kv_heads, dim, page, dtype, order)
SHAPES = [
    ([0], [1], 1, 1, 64, 16, "bf16", "phd"),                             # one token, nothing before it
    ([0, 5, 130, 1], [1, 1, 1, 1], 8, 2, 128, 16, "bf16", "phd"),
    ([15, 16, 17, 127, 128, 129], [1, 1, 1, 1, 1, 1], 6, 2, 96, 8, "fp16", "hpd"),
    ([700, 0, 3], [1, 0, 1], 5, 1, 64, 1, "fp16", "joined"),             # pages of one row, a request without tokens
    ([900], [1], 40, 1, 128, 64, "bf16", "joined"),                      # 40 heads on one kv head
    ([10, 200, 33], [4, 3, 5], 12, 4, 96, 32, "bf16", "hpd"),            # a few drafted tokens
    ([100], [60], 4, 4, 64, 16, "fp16", "phd"),                          # a chunk, one head each
    ([0, 70], [45, 33], 6, 2, 128, 16, "bf16", "phd"),                   # chunks, the first without context
    ([40, 300, 7], [1, 100, 17], 10, 2, 96, 8, "fp16", "joined"),        # chunks beside a decode
    ([0], [300], 7, 1, 128, 256, "bf16", "hpd"),                         # a page larger than a tile
    ([250, 3], [129, 128], 8, 2, 128, 16, "fp16", "phd"),
    ([513], [65], 16, 2, 64, 32, "bf16", "phd"),
]
MASKS = [(-1, 0), (0, 0), (0, 3), (1, 0), (17, 4), (64, 100), (100, 200), (5, 300), (1000, 16)]


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_paged_attention(shape, mask):
    ctx, new, heads, kv_heads, dim, page, dtype, order = SHAPES[shape]
    x = make(np.random.default_rng(shape), ctx=ctx, new=new, heads=heads, kv_heads=kv_heads, dim=dim, page=page)
    out, lse = _run(x, dtype, window=mask[0], sinks=mask[1], order=order)
    _check(out, lse, _ref(x, window=mask[0], sinks=mask[1]), dtype)


@pytest.mark.parametrize("max_new", [1, 100000])
def test_max_new_does_not_change_what_is_computed(max_new):
    """max_new picks the kernel; each of them takes every request."""
    x = make(np.random.default_rng(5), ctx=[0, 90, 300], new=[70, 1, 13], heads=6, kv_heads=2, dim=96, page=16)
    for mask in [(-1, 0), (33, 5)]:
        out, lse = _run(x, "bf16", window=mask[0], sinks=mask[1], max_new=max_new)
        _check(out, lse, _ref(x, window=mask[0], sinks=mask[1]), "bf16")


@pytest.mark.parametrize("new", [[1, 1], [9, 30]])
def test_broken_lengths_and_tables(new):
    """kv_len below the number of new tokens, 0, and past the table; missing and wrong pages; rows past the last
    request are left alone."""
    import torch
    import flashgann_b200 as fg
    rng = np.random.default_rng(3)
    for change in range(4):
        x = make(rng, ctx=[50, 60], new=new, heads=4, kv_heads=2, dim=64, page=16)
        if change == 0:
            x["kv_len"] = np.array([new[0] - 1, 0], np.int32)
        elif change == 1:
            x["kv_len"] = x["kv_len"] + np.array([5, 400], np.int32)
        elif change == 2:
            x["table"][0, 1], x["table"][1, 2] = -1, x["k"].shape[0]
        else:
            x["table"][:] = -7
        for window in (-1, 20):
            out, lse = _run(x, "fp16", window=window, sinks=2)
            _check(out, lse, _ref(x, window=window, sinks=2), "fp16")
    x = make(rng, ctx=[3], new=[2], heads=2, kv_heads=1, dim=64, page=16)
    x["q"] = np.concatenate([x["q"], x["q"]])
    out = torch.full((4, 2, 64), 7.0, dtype=torch.float16, device="cuda")
    got, _ = _run(x, "fp16", out=out)
    assert got is out and (out[2:] == 7).all() and (out[:2] != 7).any()
    # query_start past the tokens that there are
    x["start"] = np.array([0, 1000], np.int32)
    x["kv_len"] = np.array([1003], np.int32)
    got, _ = _run(x, "fp16", max_new=2)
    assert torch.isfinite(got.float()).all()
    assert fg.paged_attention(got[:0], got[None, :, :1], got[None, :, :1], _cuda(x["table"]), _cuda(x["start"]),
                              _cuda(x["kv_len"]), 0).shape == (0, 2, 64)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("new", [1, 5, 150])
def test_masked_places_may_hold_anything(new, value):
    """Keys and values that no row sees (free pages, page ends, outside of window and first tokens) and those that
    only later rows see must not touch a row; a row that sees them gets what the formula says."""
    rng = np.random.default_rng(new)
    for window, sinks in [(-1, 0), (40, 4)]:
        x = make(rng, ctx=[210], new=[new], heads=8, kv_heads=2, dim=128, page=16)
        kv_len, page = int(x["kv_len"][0]), 16
        seen = np.zeros(x["k"].shape[:2], bool)
        js = np.arange(kv_len)
        low = 0 if window < 0 else max(0, 210 - window + 1)
        js = js[(js >= low) | (js < sinks)]
        seen[x["table"][0, js // page], js % page] = True
        x["k"][~seen], x["v"][~seen] = value, value
        out, lse = _run(x, "bf16", window=window, sinks=sinks)
        _check(out, lse, _ref(x, window=window, sinks=sinks), "bf16")
        assert np.isfinite(out.float().cpu().numpy()).all()
        if new > 1:  # the last token's own value, in one element: the rows before it do not see it
            j = kv_len - 1
            x["v"][x["table"][0, j // page], j % page, 1, 5] = value
            out, lse = _run(x, "bf16", window=window, sinks=sinks)
            _check(out, lse, _ref(x, window=window, sinks=sinks), "bf16")
            assert np.isfinite(out[:-1].float().cpu().numpy()).all()
            x["k"][x["table"][0, j // page], j % page, 0, 7] = np.nan  # and its key: its own row is NaN
            out, lse = _run(x, "bf16", window=window, sinks=sinks)
            assert np.isfinite(out[:-1].float().cpu().numpy()).all()
            assert np.isnan(out[-1, :4].float().cpu().numpy()).all()


def test_large_scores_and_scales():
    """Scores far apart: the running maximum moves at every chunk, forwards and backwards."""
    rng = np.random.default_rng(8)
    for new in (1, 40):
        x = make(rng, ctx=[600], new=[new], heads=4, kv_heads=1, dim=64, page=32)
        ramp = np.round(np.linspace(-3.5, 3.5, 20) * 32) / 32  # one value for each page of 32 positions
        for sign in (1, -1):
            for pos in range(600 + new):
                x["k"][x["table"][0, pos // 32], pos % 32] = sign * ramp[pos // 32]
            x["q"][:] = 1.0
            for scale in (0.125, -0.125, 0.0, 0.5):
                out, lse = _run(x, "fp16", scale=scale)
                o, l, vmax = _ref(x, scale=scale)
                # scores up to 112: their 32-bit rounding times the sum's length adds 2^-17 * 112 to an exponent
                err = np.abs(out.double().cpu().numpy() - o)
                assert (err <= (2 * U["fp16"] + 2e-3) * vmax[..., None]).all()
                assert (np.abs(lse.double().cpu().numpy() - l) <= 2e-3).all()


def test_offsets_past_32_bits():
    """Pages that lie more than 2^32 bytes and 2^31 elements into the cache."""
    import torch
    import flashgann_b200 as fg
    pages, page, heads, dim = 70000, 64, 4, 128  # 2.3e9 elements, 4.6 GB each
    k = torch.zeros((pages, page, heads, dim), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    rng = np.random.default_rng(1)
    for new in (1, 40):
        x = make(rng, ctx=[150], new=[new], heads=8, kv_heads=heads, dim=dim, page=page, spare=0)
        n = x["k"].shape[0]
        at = torch.arange(pages - n, pages, device="cuda")
        slot = (at[:, None] * page + torch.arange(page, device="cuda")).flatten()
        fg.kv_append(k, v, _cuda(x["k"], torch.bfloat16).view(-1, heads, dim),
                     _cuda(x["v"], torch.bfloat16).view(-1, heads, dim), slot)
        assert torch.equal(k[pages - n:].float().cpu(), torch.from_numpy(x["k"]))
        table = np.where(x["table"] >= 0, x["table"] + pages - n, -1).astype(np.int32)
        out, lse = fg.paged_attention(_cuda(x["q"], torch.bfloat16), k, v, _cuda(table), _cuda(x["start"]),
                                      _cuda(x["kv_len"]), new, return_lse=True)
        _check(out, lse, _ref(x), "bf16")


@pytest.mark.parametrize("ctx,new,heads,kv_heads", [([20000], [1], 8, 2), ([3000, 1, 6000, 500], [1, 1, 2, 1], 4, 4),
                                                    ([9000], [80], 8, 1), ([3000, 20, 100], [300, 1, 50], 4, 2)])
def test_long_axes_split_over_ctas(ctx, new, heads, kv_heads):
    """Long contexts with few rows: tiles that many CTAs share.  Against torch in 64 bits; equal on every run."""
    import torch
    rng = np.random.default_rng(len(ctx))
    x = make(rng, ctx=ctx, new=new, heads=heads, kv_heads=kv_heads, dim=128, page=16)
    for window, sinks in [(-1, 0), (2500, 8)]:
        out, lse = _run(x, "bf16", window=window, sinks=sinks)
        again, lse2 = _run(x, "bf16", window=window, sinks=sinks)
        assert torch.equal(out, again) and torch.equal(lse, lse2)
        for b in range(len(ctx)):
            s, e, L = x["start"][b], x["start"][b + 1], int(x["kv_len"][b])
            js = np.arange(L)
            pg = x["table"][b, js // 16]
            k = torch.from_numpy(x["k"][pg, js % 16]).cuda().double().repeat_interleave(heads // kv_heads, 1)
            v = torch.from_numpy(x["v"][pg, js % 16]).cuda().double().repeat_interleave(heads // kv_heads, 1)
            q = torch.from_numpy(x["q"][s:e]).cuda().double()
            p = torch.arange(L - (e - s), L, device="cuda")[:, None]
            j = torch.arange(L, device="cuda")[None]
            see = (j <= p) & ((p - j < window) | (j < sinks) if window >= 0 else True)
            sc = torch.einsum("thd,jhd->htj", q, k) * 128 ** -0.5
            sc = sc.masked_fill(~see, -np.inf)
            o = torch.einsum("htj,jhd->thd", torch.softmax(sc, -1), v)
            ref = (o.cpu().numpy(), torch.logsumexp(sc, -1).T.cpu().numpy(), np.full((e - s, heads), 4.0))
            _check(out[s:e], lse[s:e], ref, "bf16")


# ---- retrieved ----

@pytest.mark.parametrize("ctx,new,heads,kv_heads,dim,page,count,window,sinks,dtype", [
    ([50], [1], 2, 1, 64, 16, 5, 8, 0, "bf16"),
    ([500, 30, 0], [1, 1, 1], 8, 2, 128, 16, 100, 64, 4, "bf16"),
    ([300, 700], [3, 2], 6, 2, 96, 8, 33, 1, 16, "fp16"),
    ([400], [2], 40, 1, 64, 32, 17, 0, 0, "fp16"),          # three tiles of heads; no window
    ([900, 2], [1, 2], 12, 4, 128, 64, 512, 16, 1, "bf16"),
    ([10], [1], 4, 4, 96, 16, 200, 100, 4, "fp16"),         # the window holds all
    ([250], [1], 3, 1, 128, 1, 1, 5, 2, "bf16"),
    ([3000, 900], [1, 2], 6, 2, 64, 16, 1000, 30, 3, "fp16"),   # a tile to a head
    ([5000], [1], 4, 1, 128, 32, 500, 0, 0, "bf16"),            # two heads to a tile
    ([100, 40], [1, 1], 6, 1, 64, 16, 1024, 3, 0, "fp16"),      # as many ids as there may be, most of them repeats
    ([2000], [3], 8, 8, 96, 16, 40, 700, 0, "bf16"),
])
def test_retrieved_attention(ctx, new, heads, kv_heads, dim, page, count, window, sinks, dtype):
    rng = np.random.default_rng(count)
    x = make(rng, ctx=ctx, new=new, heads=heads, kv_heads=kv_heads, dim=dim, page=page)
    T = x["q"].shape[0]
    top = max(c + n for c, n in zip(ctx, new))
    ids = rng.integers(0, top + 20, (T, heads, count)).astype(np.int32)  # future ones and repeats among them
    ids[rng.random(ids.shape) < 0.1] = -1
    ids[rng.random(ids.shape) < 0.05] = 2 ** 31 - 1
    ids[:, -1, :] = ids[:, -1, :1]  # one id over and over
    if heads > 2:
        ids[:, 1, :] = -1           # nothing retrieved
    out, lse = _run(x, dtype, window=window, sinks=sinks, ids=ids)
    _check(out, lse, _ref(x, window=window, sinks=sinks, ids=ids), dtype)


def test_retrieved_rows_stay_apart():
    """A key that one head retrieved and that holds NaN or infinity touches that head alone."""
    rng = np.random.default_rng(4)
    x = make(rng, ctx=[400], new=[1], heads=8, kv_heads=2, dim=128, page=16)
    ids = rng.integers(0, 300, (1, 8, 40)).astype(np.int32)
    ids[ids == 77] = 78
    ids[0, 5, 11] = 77
    for value in (np.nan, np.inf):
        x["v"][x["table"][0, 77 // 16], 77 % 16, 1, 3] = value
        out, lse = _run(x, "fp16", window=32, sinks=4, ids=ids)
        _check(out, lse, _ref(x, window=32, sinks=4, ids=ids), "fp16")
        assert not np.isfinite(out[0, 5, 3].item()) and np.isfinite(out.float().cpu().numpy()).sum() == 8 * 128 - 1


def test_retrieved_strided_ids_and_empty_rows():
    import torch
    import flashgann_b200 as fg
    rng = np.random.default_rng(6)
    x = make(rng, ctx=[100, 200], new=[1, 1], heads=4, kv_heads=2, dim=64, page=16)
    ids = rng.integers(0, 100, (2, 4, 12)).astype(np.int32)
    ids[1, 2] = -1
    by_head = _cuda(ids.transpose(1, 0, 2))  # [heads, T, count], as one search for each head leaves them
    dt = torch.bfloat16
    out, lse = fg.retrieved_attention(_cuda(x["q"], dt), _cuda(x["k"], dt), _cuda(x["v"], dt), _cuda(x["table"]),
                                      _cuda(x["start"]), _cuda(x["kv_len"]), by_head.transpose(0, 1), window=0,
                                      return_lse=True)
    _check(out, lse, _ref(x, window=0, ids=ids), "bf16")
    assert (out[1, 2] == 0).all() and lse[1, 2].item() == float("-inf")
    none = fg.retrieved_attention(_cuda(x["q"], dt), _cuda(x["k"], dt), _cuda(x["v"], dt), _cuda(x["table"]),
                                  _cuda(x["start"]), _cuda(x["kv_len"]), by_head.transpose(0, 1)[:, :, :0], window=7)
    want = fg.paged_attention(_cuda(x["q"], dt), _cuda(x["k"], dt), _cuda(x["v"], dt), _cuda(x["table"]),
                              _cuda(x["start"]), _cuda(x["kv_len"]), 1, window=7)
    assert torch.allclose(none.float(), want.float(), atol=2 * U["bf16"] * 4)


# ---- streams, layouts of queries and outputs, graphs ----

def test_streams_strides_and_graph():
    import torch
    import flashgann_b200 as fg
    x = make(np.random.default_rng(12), ctx=[300, 40], new=[20, 1], heads=6, kv_heads=2, dim=128, page=16)
    ref = _ref(x, window=100, sinks=4)
    dt = torch.bfloat16
    T = x["q"].shape[0]
    qkv = torch.zeros((T, 10, 128), dtype=dt, device="cuda")
    qkv[:, :6] = _cuda(x["q"], dt)
    wide = torch.full((T, 9, 136), 3.0, dtype=dt, device="cuda")
    out = wide[:, 2:8, 8:]
    k, v, table, start, kv_len = (_cuda(x["k"], dt), _cuda(x["v"], dt), _cuda(x["table"]), _cuda(x["start"]),
                                  _cuda(x["kv_len"]))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for stream in (None, side, side.cuda_stream):
        out.fill_(3.0)
        torch.cuda.synchronize()
        got, lse = fg.paged_attention(qkv[:, :6], k, v, table, start, kv_len, 20, window=100, sinks=4, out=out,
                                      return_lse=True, stream=stream)
        torch.cuda.synchronize()
        _check(got, lse, ref, "bf16")
        assert (wide[:, :2] == 3).all() and (wide[:, 8:] == 3).all() and (wide[:, :, :8] == 3).all()
    # misaligned queries are copied
    flat = torch.zeros(T * 6 * 128 + 1, dtype=dt, device="cuda")
    flat[1:] = _cuda(x["q"], dt).flatten()
    got, lse = fg.paged_attention(flat[1:].view(T, 6, 128), k, v, table, start, kv_len, 20, window=100, sinks=4,
                                  return_lse=True)
    _check(got, lse, ref, "bf16")
    # captured once, replayed on other contents
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, lse = fg.paged_attention(qkv[:, :6], k, v, table, start, kv_len, 20, window=100, sinks=4, return_lse=True)
    k.mul_(-1)
    graph.replay()
    torch.cuda.synchronize()
    x["k"] = -x["k"]
    _check(got, lse, _ref(x, window=100, sinks=4), "bf16")


def test_step_of_a_batch():
    """plan, append and attention together: two steps of three requests against the definition on the whole
    sequences."""
    import torch
    import flashgann_b200 as fg
    rng = np.random.default_rng(20)
    dt, page, H, G, D = torch.float16, 16, 2, 3, 96
    cache = torch.full((2, 40, page, H, D), float("nan"), dtype=dt, device="cuda")
    free = _cuda(rng.permutation(40).astype(np.int32))
    table = torch.full((3, 12), -1, dtype=torch.int32, device="cuda")
    head = None
    ctx = np.zeros(3, np.int32)
    hist = [[np.zeros((0, H, D), np.float32)] * 2 for _ in range(3)]
    for new in ([100, 7, 30], [1, 1, 4], [1, 40, 1]):
        T = sum(new)
        q, k, v = (np.round(rng.standard_normal((T, n, D)) * 32).astype(np.float32) / 32 for n in (H * G, H, H))
        plan = fg.kv_plan(_cuda(ctx), _cuda(np.array(new, np.int32)), table, free, tokens=T, page_size=page,
                          free_head=head)
        fg.kv_append(cache[0], cache[1], _cuda(k, dt), _cuda(v, dt), plan.slot)
        out, lse = fg.paged_attention(_cuda(q, dt), cache[0], cache[1], table, plan.query_start, plan.kv_len, max(new),
                                      return_lse=True)
        head = plan.free_head
        at = 0
        for b, n in enumerate(new):
            hist[b] = [np.concatenate([h, r[at:at + n]]) for h, r in zip(hist[b], (k, v))]
            L = len(hist[b][0])
            one = attention_ref(q[at:at + n], hist[b][0][None], hist[b][1][None], np.zeros((1, 1), np.int64), [0, n],
                                [L])
            _check(out[at:at + n], lse[at:at + n], one, "fp16")
            at += n
        ctx = ctx + np.array(new, np.int32)
    assert plan.refused.sum().item() == 0


@pytest.mark.parametrize("new", [1, 60])
def test_expanded_tensors(new):
    """Axes of stride 0: one kv head's cache shown as four, one query shown as all."""
    import torch
    import flashgann_b200 as fg
    x = make(np.random.default_rng(30 + new), ctx=[70, 40], new=[new, new], heads=8, kv_heads=1, dim=64, page=16)
    x["q"][:] = x["q"][:, :1]
    dt = torch.float16
    k, v, q = _cuda(x["k"], dt).expand(-1, -1, 4, -1), _cuda(x["v"], dt).expand(-1, -1, 4, -1), _cuda(x["q"][:, :1], dt)
    rest = (_cuda(x["table"]), _cuda(x["start"]), _cuda(x["kv_len"]), new)
    for qq in (q.expand(-1, 8, -1), q.repeat(1, 8, 1)):
        for kk, vv in ((k, v), (k.contiguous(), v.contiguous())):
            out, lse = fg.paged_attention(qq, kk, vv, *rest, return_lse=True)
            _check(out, lse, _ref(x), "fp16")
    one = _cuda(x["q"][:1, :1], dt).expand(2 * new, 8, -1)
    x["q"][:] = x["q"][:1, :1]
    out, lse = fg.paged_attention(one, k, v, *rest, return_lse=True)
    _check(out, lse, _ref(x), "fp16")


def test_workspace_refusals():
    """A call whose rows may be split refuses a missing, misaligned or short workspace; a short table needs none."""
    import ctypes
    import torch
    import flashgann_b200 as fg
    from flashgann_b200 import _capi
    L = fg.lib()
    z = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    p = z.data_ptr()

    def args(width, **kw):
        cache = _capi.KVCacheArgs(k=p, v=p, page_stride=1024, token_stride=64, head_stride=64, pages=4, page_size=16,
                                  heads=1, dim=64, dtype=_capi.FG_DTYPE_F16)
        a = _capi.AttentionArgs(q=p, q_token_stride=64, q_head_stride=64, out=p + 4096, out_token_stride=64,
                                out_head_stride=64, block_table=p + 8192, table_stride=width, query_start=p + 16384,
                                kv_len=p + 16448, tokens=1, heads=1, requests=1, table_width=width, max_new=1, window=-1,
                                scale=0.125, **kw)
        return cache, a

    need = ctypes.c_uint64()
    c, a = args(1000)
    assert L.fg_attention_workspace_bytes(c, a, 0, ctypes.byref(need)) == fg.FG_OK and need.value > 0
    for kw in (dict(), dict(workspace=p + 16, workspace_bytes=1 << 40), dict(workspace=p, workspace_bytes=need.value - 1)):
        c, a = args(1000, **kw)
        assert L.fg_paged_attention_device(c, a, None) == fg.FG_ERR_ARG
        assert "workspace" in L.fg_last_error().decode()
    c, a = args(4)
    assert L.fg_attention_workspace_bytes(c, a, 0, ctypes.byref(need)) == fg.FG_OK and need.value == 0
    assert L.fg_paged_attention_device(c, a, None) == fg.FG_OK
    torch.cuda.synchronize()


def test_example_of_a_decode_over_retrieved_keys():
    """The example runs all four operators with the search; its last step's output is the formula's for the ids that
    the search returned, over the cache as plan and append left it."""
    import importlib.util
    import os
    from tests.common import ROOT
    spec = importlib.util.spec_from_file_location("retrieval_decode", os.path.join(ROOT, "examples", "retrieval_decode.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    r = m.run(context=4000, steps=2)
    assert r["refused"] == 0 and r["tokens"] == 4002 and 0 < r["weight_seen"] <= 1 + 1e-3
    x = {k: v.float().cpu().numpy() if hasattr(v, "cpu") and v.is_floating_point() else v for k, v in r["last"].items()}
    ref = attention_ref(x["q"], x["k_cache"], x["v_cache"], x["table"].cpu().numpy(), [0, 1], [4002],
                        window=x["window"], sinks=x["sinks"], ids=x["ids"].cpu().numpy())
    _check(r["last"]["out"], r["last"]["lse"], ref, "bf16")
