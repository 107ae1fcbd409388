"""The cache and attention operators on the GPU at the ends of what they promise: batches of thousands of requests,
sums that pass 32 bits, scores far apart in 16-bit weights.  References are the definitions in 64 bits; tolerances
are those of test_gpu_attention.py, and stated at the test where they differ."""

from __future__ import annotations

import numpy as np
import pytest

from tests.test_gpu_attention import _cuda, _dt, _run, U

pytestmark = pytest.mark.gpu


def _batch(rng, requests, *, heads, kv_heads, dim, page, new, ctx):
    """Requests with up to ctx tokens in the cache and up to new more each, a third of them without any; all pages are
    drawn from a small cache, so that requests share them (as prefixes do)."""
    pages = 97
    c = rng.integers(0, ctx + 1, requests)
    n = rng.integers(1, new + 1, requests) * (rng.random(requests) < 2 / 3)
    n[rng.integers(0, requests)] = 1
    start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    width = -(-(ctx + new) // page)

    def draw(*shape):  # multiples of 1/32 up to +-4: exact in both types
        return np.clip(np.round(rng.standard_normal(shape) * 32) / 32, -3.96875, 3.96875).astype(np.float32)

    return dict(q=draw(int(start[-1]), heads, dim), k=draw(pages, page, kv_heads, dim), v=draw(pages, page, kv_heads, dim),
                table=rng.integers(0, pages, (requests, width)).astype(np.int32), start=start,
                kv_len=(c + n).astype(np.int32))


def _ref64(x, *, window=-1, sinks=0, ids=None, at=4096):
    """(out, lse) of every row in 64 bits on the GPU, `at` rows at a time."""
    import torch
    q, k, v, table = (_cuda(x[n]) for n in ("q", "k", "v", "table"))
    start, kv_len = _cuda(x["start"]).long(), _cuda(x["kv_len"]).long()
    T, heads, dim = q.shape
    page, H = k.shape[1], k.shape[2]
    t = torch.arange(T, device="cuda")
    r = torch.searchsorted(start[1:].contiguous(), t, right=True)
    p = kv_len[r] - start[r + 1] + t
    j = torch.arange(int(kv_len.max()), device="cuda")
    outs, lses = [], []
    for lo in range(0, T, at):
        rr, pp = r[lo:lo + at], p[lo:lo + at, None]
        pg = table[rr[:, None], (j // page)[None, :]].long()
        see = j[None] <= pp
        if window >= 0:
            see = see & ((pp - j[None] < window) | (j[None] < sinks))
        see = see[:, None].expand(-1, heads, -1)
        if ids is not None:
            got = _cuda(ids[lo:lo + at]).long()
            mark = torch.zeros((*got.shape[:2], len(j) + 1), dtype=torch.bool, device="cuda")
            mark.scatter_(2, torch.where((got < 0) | (got > pp[:, None]), len(j), got), True)
            see = see | mark[..., :-1]
        kk = k[pg, j % page].double().repeat_interleave(heads // H, 2)
        s = torch.einsum("thd,tjhd->thj", q[lo:lo + at].double(), kk) * dim ** -0.5
        s = s.masked_fill(~see, -np.inf)
        vv = v[pg, j % page].double().repeat_interleave(heads // H, 2)
        outs.append(torch.einsum("thj,tjhd->thd", torch.softmax(s, -1).nan_to_num(0.0), vv))
        lses.append(torch.logsumexp(s, -1))
    return torch.cat(outs), torch.cat(lses)


def _close(got, want, dtype, vmax=4.0):
    import torch
    (out, lse), (o, l) = got, want
    assert torch.equal(torch.isneginf(lse.double()), torch.isneginf(l))
    fine = torch.isfinite(l)
    assert torch.isfinite(out.float()).all()
    assert ((out.double() - o).abs() <= (2 * U[dtype] + 2e-4) * vmax).all(), float((out.double() - o).abs().max())
    assert ((lse.double() - l)[fine].abs() <= 2e-4).all()


# ---- many requests: the scan over their lengths ----

@pytest.mark.parametrize("requests,dim,dtype", [(12224, 64, "bf16"), (12225, 64, "fp16"), (16384, 64, "bf16"),
                                                (16384, 96, "fp16"), (16384, 128, "bf16")])
def test_as_many_requests_as_there_may_be(requests, dim, dtype):
    """The sums over 16384 requests take 64 KB of shared memory, more than the keys of the smallest head size do."""
    rng = np.random.default_rng(requests + dim)
    x = _batch(rng, requests, heads=2, kv_heads=1, dim=dim, page=16, new=1, ctx=30)
    _close(_run(x, dtype), _ref64(x), dtype)
    ids = rng.integers(-1, 40, (x["q"].shape[0], 2, 6)).astype(np.int32)
    _close(_run(x, dtype, ids=ids, window=3, sinks=1), _ref64(x, ids=ids, window=3, sinks=1), dtype)
    # the kernel of many rows, for the same requests
    _close(_run(x, dtype, max_new=1000, window=9), _ref64(x, window=9), dtype)


def test_too_many_ids_are_refused():
    import flashgann_b200 as fg
    rng = np.random.default_rng(0)
    x = _batch(rng, 2, heads=2, kv_heads=1, dim=64, page=16, new=1, ctx=30)
    for count in (1025, 2000):
        with pytest.raises(fg.FlashGANNError, match=f"{count} ids"):
            _run(x, "fp16", ids=np.zeros((x["q"].shape[0], 2, count), np.int32), window=3)


@pytest.mark.parametrize("requests", [4, 5, 32, 33, 64, 65, 128, 129, 257, 513, 2000])
@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", [(6, 2, 96, 8, "fp16"), (4, 4, 64, 16, "bf16"), (8, 1, 128, 32, "bf16")])
def test_batches_around_the_scans_steps(requests, heads, kv_heads, dim, page, dtype):
    """One warp scans up to 32 requests (4 in the kernel of many rows), the block 128 (64) at a time: sizes at and past
    each of these, requests without tokens among them, in both kernels and with ids."""
    rng = np.random.default_rng(requests * heads)
    x = _batch(rng, requests, heads=heads, kv_heads=kv_heads, dim=dim, page=page, new=3, ctx=70)
    for window, sinks in [(-1, 0), (20, 3)]:
        want = _ref64(x, window=window, sinks=sinks)
        for max_new in (1, 1000):
            _close(_run(x, dtype, window=window, sinks=sinks, max_new=max_new), want, dtype)
    ids = rng.integers(-1, 90, (x["q"].shape[0], heads, 9)).astype(np.int32)
    _close(_run(x, dtype, ids=ids, window=5, sinks=2), _ref64(x, ids=ids, window=5, sinks=2), dtype)


@pytest.mark.parametrize("requests", [7, 65, 150])
def test_batches_of_chunks_and_long_contexts(requests):
    """Requests of up to 200 rows and contexts that are split over CTAs, beside short ones."""
    rng = np.random.default_rng(requests)
    x = _batch(rng, requests, heads=4, kv_heads=2, dim=64, page=16, new=50, ctx=20)
    long = rng.integers(0, requests, 2)
    x["kv_len"][long] += 900
    x["table"] = rng.integers(0, x["k"].shape[0], (requests, 70)).astype(np.int32)
    for window, sinks in [(-1, 0), (300, 20)]:
        want = _ref64(x, window=window, sinks=sinks, at=256)
        for max_new in (1, 1000):
            _close(_run(x, "fp16", window=window, sinks=sinks, max_new=max_new), want, "fp16")


# ---- weights in 16 bits ----

@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("depth", [12.0, 17.5, 20.0])
@pytest.mark.parametrize("kernel", ["rows", "tiles"])
def test_many_keys_far_below_the_maximum(kernel, depth, dtype):
    """Four keys with a score of `depth` before half a million with a score of 0: e^-17.5 is below half of float16's
    least number, but all of them together are 0.3 % of the sum, and the output is that share of their value.  One
    tile to a CTA, so that each warp (each row) meets a maximum first and the tail after it.  Beside the usual
    tolerances: a lane's running sum of about 1 takes up to 8192 addends, each rounded to 2^-24."""
    import torch
    import flashgann_b200 as fg
    n, page, dim = 1 << 19, 64, 64
    requests, heads, new = (37, 8, 1) if kernel == "rows" else (37, 4, 20)  # 296 or 148 tiles
    dt = _dt(dtype)
    k, v = (torch.zeros((2, page, heads, dim), dtype=dt, device="cuda") for _ in range(2))
    k[0, ::16, :, 0] = 1.0                  # the first page: every 16th key
    v[..., :32] = 1.0                       # half of the columns hold the tail's value and nothing of the four keys'
    v[0, ::16, :, :32] = 0.0
    v[0, ::16, :, 32:] = 1.0                # the others the reverse
    q = torch.zeros((requests * new, heads, dim), dtype=dt, device="cuda")
    q[..., 0] = 1.0
    table = torch.ones((requests, n // page), dtype=torch.int32, device="cuda")
    table[:, 0] = 0
    start = torch.arange(0, requests * new + 1, new, dtype=torch.int32, device="cuda")
    kv_len = torch.full((requests,), n, dtype=torch.int32, device="cuda")
    out, lse = fg.paged_attention(q, k, v, table, start, kv_len, new, scale=depth, return_lse=True)
    tail = (torch.arange(n - new, n, device="cuda").double() + 1 - 4).repeat(requests)[:, None, None] * np.exp(-depth)
    want = torch.cat([(tail / (4 + tail)).expand(-1, heads, 32), (4 / (4 + tail)).expand(-1, heads, 32)], 2)
    tol = 2 * U[dtype] + 2e-4
    assert ((out.double() - want).abs() <= tol).all(), float((out.double() - want).abs().max())
    assert ((lse.double() - (depth + torch.log(4 + tail[..., 0]))).abs() <= 2e-4 + 8192 * 2.0 ** -24).all()


# ---- sums of work past 32 bits ----

def test_more_than_2_to_the_31_units_of_work():
    """4096 requests of 35 million keys each, 2.2e9 units of 64 keys for a kv head; all but the first page of a request
    are missing, so that little is read.  (Eight seconds: every chunk is walked.)"""
    import torch
    import flashgann_b200 as fg
    requests, page, dim, n = 4096, 4096, 64, 35_000_000
    g = torch.Generator(device="cuda").manual_seed(9)
    k, v, q = ((torch.randn(s, generator=g, device="cuda").clamp(-3.9, 3.9) * 32).round().div(32).half()
               for s in ((1, page, 1, dim), (1, page, 1, dim), (requests, 1, dim)))
    table = torch.full((1, -(-n // page)), -1, dtype=torch.int32, device="cuda")
    table[0, 0] = 0
    start = torch.arange(requests + 1, dtype=torch.int32, device="cuda")
    kv_len = torch.full((requests,), n, dtype=torch.int32, device="cuda")
    out = torch.full((requests, 1, dim), 7.0, dtype=torch.float16, device="cuda")
    _, lse = fg.paged_attention(q, k, v, table.expand(requests, -1), start, kv_len, 1, out=out, return_lse=True)
    s = q[:, 0].double() @ k[0, :, 0].double().T * dim ** -0.5
    _close((out, lse), (torch.softmax(s, -1)[:, None] @ v[0, :, 0].double(), torch.logsumexp(s, -1)[:, None]), "fp16")


def test_calls_of_2_to_the_31_blocks_leave_the_kernel_of_many_rows():
    """Its sums of blocks are 32 bits: where the counts do not exclude more, the other kernel takes the call, as the
    size of the workspace shows."""
    import ctypes
    import flashgann_b200 as fg
    from tests.test_attention_args import _args, _cache

    def need(**kw):
        n = ctypes.c_uint64()
        kw = dict(dict(window=-1, heads=2, requests=16384, tokens=16384, table_width=1 << 20), **kw)
        assert fg.lib().fg_attention_workspace_bytes(_cache(page_size=16), _args(**kw), 0, ctypes.byref(n)) == fg.FG_OK
        return n.value

    few = need(max_new=1)
    assert need(max_new=1000, table_width=1 << 19) != few   # 16384 requests of 2^23 keys: 1.1e9 blocks
    assert need(max_new=1000) == few                        # twice as many
    # all positions that there are, for 100 and for 128 requests
    assert need(max_new=1000, table_width=1 << 30, requests=100, tokens=100) != few
    assert need(max_new=1000, table_width=1 << 30, requests=128, tokens=128) == few
    # one request, of 2^13 and of 2^14 tiles
    assert need(max_new=1000, tokens=1 << 21, requests=1) != few
    assert need(max_new=1000, tokens=1 << 22, requests=1) == few


# ---- waits inside the kernel of many rows ----

@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("fp16", 64)])
def test_a_wait_that_runs_out_shows_in_every_row_it_leaves(dtype, dim):
    """K tiles from some block of each CTA on are never loaded (a flag that nothing sets): the waits for them run out
    and the CTAs give up.  Their rows are NaN, whole tiles and parts that are joined alike, and no row keeps what the
    output held before.  The next call is not touched by it."""
    import torch
    import flashgann_b200 as fg
    rng = np.random.default_rng(dim)
    for requests, new, ctx, window, sinks in [(1, 300, 6000, -1, 0), (40, 70, 300, -1, 0), (40, 70, 300, 90, 9)]:
        x = _batch(rng, requests, heads=4, kv_heads=2, dim=dim, page=16, new=new, ctx=ctx)
        want, want_lse = _ref64(x, window=window, sinks=sinks, at=128)
        shares = []
        for first in (0, 1, 2, 3, 5, 9, 1000):
            out = torch.full(want.shape, 7.0, dtype=_dt(dtype), device="cuda")
            fg.lib().fg_test_attention_lose_blocks(first, 4)
            try:
                _, lse = _run(x, dtype, window=window, sinks=sinks, max_new=1000, out=out)
                torch.cuda.synchronize()
            finally:
                fg.lib().fg_test_attention_lose_blocks(-1, -1)
            lost = torch.isnan(lse)
            shares.append(float(lost.float().mean()))
            assert torch.equal(lost[..., None].expand_as(out), torch.isnan(out))
            _close((out[~lost][:, None], lse[~lost][:, None]), (want[~lost][:, None], want_lse[~lost][:, None]), dtype)
        assert shares[0] == 1.0 and shares[-1] == 0.0 and sorted(shares, reverse=True) == shares
        _close(_run(x, dtype, window=window, sinks=sinks, max_new=1000), (want, want_lse), dtype)


# ---- rows that are written must not overlap ----

def test_overlapping_tensors_are_refused():
    import torch
    import flashgann_b200 as fg
    x = _batch(np.random.default_rng(1), 3, heads=2, kv_heads=1, dim=64, page=16, new=2, ctx=30)
    T = x["q"].shape[0]
    flat = torch.full((T * 3 * 64,), 7.0, dtype=torch.float16, device="cuda")
    for strides in [(64, 64, 1), (64, 128, 1), (0, 64, 1), (96, 64, 1)]:
        with pytest.raises(fg.FlashGANNError, match="rows of out overlap"):
            _run(x, "fp16", out=flat.as_strided((T, 2, 64), strides))
    assert (flat == 7).all()
    by_head = flat.as_strided((T, 2, 64), (64, T * 64, 1))  # any order of axes that nest
    _close(_run(x, "fp16", out=by_head), _ref64(x), "fp16")
    assert (flat[T * 2 * 64:] == 7).all()
    ints = torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(fg.FlashGANNError, match="rows of the block table overlap"):
        fg.kv_plan(ints, ints + 1, ints[None, :1].expand(2, 4).contiguous()[:1].expand(2, 4), ints, tokens=2, page_size=16)


# ---- plan ----

def test_plan_refuses_lengths_past_31_bits():
    """Lengths and positions are 32 bits: a request that would pass them gets nothing, whatever its table holds."""
    import flashgann_b200 as fg
    top = 2 ** 31 - 1
    ctx, new = [top, top - 2, top, top - 1], [0, 2, 1, 5]
    table = np.arange(12, dtype=np.int32).reshape(4, 3)  # three pages of 2^30 rows each
    got = _cuda(table)
    p = fg.kv_plan(_cuda(np.array(ctx, np.int32)), _cuda(np.array(new, np.int32)), got, _cuda(np.array([40], np.int32)),
                   tokens=8, page_size=2 ** 30)
    assert p.refused.tolist() == [0, 0, 1, 1] and p.kv_len.tolist() == [top, top, 0, 0]
    assert p.query_start.tolist() == [0, 0, 2, 3, 8] and p.free_head.tolist() == [0]
    assert p.position.tolist() == [top - 2, top - 1] + [-1] * 6
    assert p.slot.tolist() == [(4 << 30) + 2 ** 30 - 3, (4 << 30) + 2 ** 30 - 2] + [-1] * 6
    assert np.array_equal(got.cpu().numpy(), table)


def test_plans_of_many_requests_from_threads():
    """Plans above 2048 requests need more shared memory than a kernel gets unasked; calls of different sizes from
    threads at the same time all get theirs."""
    import threading
    import torch
    import flashgann_b200 as fg
    L, bad = fg.lib(), []

    def plans(requests):
        z = torch.zeros(6 * requests + 64, dtype=torch.int32, device="cuda")
        p, stream = z.data_ptr(), torch.cuda.Stream()
        at = [p + 4 * requests * i for i in range(6)]
        for _ in range(3000):
            rc = L.fg_kv_plan_device(at[0], at[1], requests, None, 0, None, 16, None, 0, 0, 0, at[2], at[3] + 16, None, None,
                                     at[4] + 32, at[5] + 48, stream.cuda_stream)
            if rc != fg.FG_OK:
                bad.append((requests, L.fg_last_error().decode()))
                break
        stream.synchronize()

    threads = [threading.Thread(target=plans, args=(n,)) for n in (2100, 8192, 4000)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad


# ---- gradients and versions ----

def test_gradients_are_refused_and_writes_are_counted():
    """No call has a backward pass: under grad mode a tensor that requires a gradient is refused, and what a call
    writes in place gets a new version, so that autograd notices."""
    import torch
    import flashgann_b200 as fg
    x = _batch(np.random.default_rng(2), 3, heads=2, kv_heads=1, dim=64, page=16, new=2, ctx=30)
    dt = torch.float16
    q, k, v = (_cuda(x[n], dt) for n in ("q", "k", "v"))
    rest = (_cuda(x["table"]), _cuda(x["start"]), _cuda(x["kv_len"]))
    T = q.shape[0]
    new, slot = torch.zeros((T, 1, 64), dtype=dt, device="cuda"), torch.arange(T, device="cuda")
    ids = torch.zeros((T, 2, 4), dtype=torch.int32, device="cuda")
    calls = {
        "paged": lambda q, k, v, n, out: fg.paged_attention(q, k, v, *rest, 2, out=out),
        "retrieved": lambda q, k, v, n, out: fg.retrieved_attention(q, k, v, *rest, ids, window=3, out=out),
        "append": lambda q, k, v, n, out: fg.kv_append(k, v, n, n, slot)}
    for name, call in calls.items():
        for i, t in enumerate((q, k, v, new, torch.empty_like(q))):
            args = [q, k.clone(), v.clone(), new, None]
            args[i] = t.clone().requires_grad_()
            if (name == "append") == (i in (0, 4)) and i not in (1, 2):
                call(*args)  # not an argument of this call
                continue
            with pytest.raises(fg.FlashGANNError, match="requires a gradient"):
                call(*args)
            with torch.no_grad():
                call(*args)
            with torch.inference_mode():
                call(*args)
    versions = [t._version for t in (q, k, v, new)]
    fg.kv_append(k, v, new, new, slot)
    out = torch.empty_like(q)
    before = out._version
    fg.paged_attention(q, k, v, *rest, 2, out=out)
    assert out._version == before + 1
    assert [t._version for t in (q, k, v, new)] == [versions[0], versions[1] + 1, versions[2] + 1, versions[3]]
    one, table = torch.ones(3, dtype=torch.int32, device="cuda"), rest[0].clone()
    fg.kv_plan(one, one, table, one, tokens=3, page_size=16)
    assert table._version == 1
    with torch.inference_mode():
        kk = k.clone()
        fg.kv_append(kk, kk.clone(), new, new, slot)


# ---- axes of one entry ----

@pytest.mark.parametrize("new", [1, 30])
def test_axes_of_one_entry_have_any_stride(new):
    """One kv head, K with the pages' rows outside and V with the heads outside: the same layout, other strides of the
    axis of one entry; and one token, one page, one head with strides that no tensor core would take."""
    import torch
    import flashgann_b200 as fg
    dt = torch.float16
    x = _batch(np.random.default_rng(new), 3, heads=2, kv_heads=1, dim=64, page=16, new=new, ctx=30)
    q, k, v = (_cuda(x[n], dt) for n in ("q", "k", "v"))
    rest = (_cuda(x["table"]), _cuda(x["start"]), _cuda(x["kv_len"]))
    by_head = v.transpose(1, 2).contiguous().transpose(1, 2).as_strided(v.shape, (1024, 64, 1024, 1))
    odd = v.as_strided(v.shape, (1024, 64, 3, 1))
    for vv in (v, by_head, odd):
        for kk in (k, k.as_strided(k.shape, (1024, 64, 5, 1))):
            _close(fg.paged_attention(q, kk, vv, *rest, new, return_lse=True), _ref64(x), "fp16")
    T = q.shape[0]
    a, b = k.clone(), by_head.clone(memory_format=torch.preserve_format)
    slot = torch.randperm(k.shape[0] * 16, device="cuda")[:T]
    fg.kv_append(a, b.as_strided(b.shape, (1024, 64, 7, 1)), q[:, :1], q[:, 1:], slot)
    assert torch.equal(a.view(-1, 64)[slot], q[:, 0]) and torch.equal(b.reshape(-1, 64)[slot], q[:, 1])
    one = _batch(np.random.default_rng(7), 1, heads=1, kv_heads=1, dim=64, page=64, new=1, ctx=30)
    q, k, v = (_cuda(one[n], dt) for n in ("q", "k", "v"))
    one["table"][:] = 0
    one["k"], one["v"] = one["k"][:1], one["v"][:1]
    rest = (_cuda(one["table"]), _cuda(one["start"]), _cuda(one["kv_len"]))
    out = torch.zeros(100, dtype=dt, device="cuda").as_strided((1, 1, 64), (5, 3, 1))
    k, v = (t[:1].as_strided((1, 64, 1, 64), (9, 64, 11, 1)) for t in (k, v))
    for max_new in (1, 100):
        _, lse = fg.paged_attention(q.as_strided(q.shape, (3, 1, 1)), k, v, *rest, max_new, out=out, return_lse=True)
        _close((out, lse), _ref64(one), "fp16")


def test_waits_run_out_within_seconds():
    """With the limit that all calls have: a copy that never comes costs about a second, not the GPU."""
    import time
    import torch
    import flashgann_b200 as fg
    x = _batch(np.random.default_rng(3), 2, heads=4, kv_heads=2, dim=64, page=16, new=70, ctx=900)
    _run(x, "bf16", max_new=1000)
    torch.cuda.synchronize()
    fg.lib().fg_test_attention_lose_blocks(0, -1)
    try:
        t = time.monotonic()
        out, lse = _run(x, "bf16", max_new=1000)
        torch.cuda.synchronize()
        t = time.monotonic() - t
    finally:
        fg.lib().fg_test_attention_lose_blocks(-1, -1)
    assert 0.2 < t < 5, t
    assert torch.isnan(out).all() and torch.isnan(lse).all()
    _close(_run(x, "bf16", max_new=1000), _ref64(x), "bf16")
