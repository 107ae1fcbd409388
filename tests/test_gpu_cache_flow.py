"""Page summaries, block selection and attention, key weights and eviction together, as a decoder calls them: steps of a
batch against the definitions, captured in graphs, on other streams, over caches of more than 2^31 elements."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from tests.attention_ref import attention_ref, make
from tests.block_ref import block_ids, evict_ref, select_ref, summary_ref, weights_ref
from tests.test_gpu_attention import _check, _cuda, _dt

pytestmark = pytest.mark.gpu


def _host(t):
    return (t.float() if t.is_floating_point() else t).cpu().numpy()


@pytest.mark.parametrize("dtype,dim,page,group", [("bf16", 64, 8, 3), ("fp16", 96, 16, 4), ("bf16", 128, 4, 1)])
def test_steps_of_a_batch(dtype, dim, page, group):
    """Prompts, then steps of one and of two tokens with attention over chosen blocks; where a request passes its budget the
    cache is cut, summed up anew, and decoding goes on.  Every call against its definition on the state it was given."""
    import torch
    import flashgann_b200 as fg
    rng = np.random.default_rng(dim)
    H, R, budget, recent, sinks, window, count = 2, 3, 8 * page, 2 * page, 2, 5, 3
    dt = _dt(dtype)
    pages = 3 * R * budget // page
    k, v = (torch.zeros((pages, page, H, dim), dtype=dt, device="cuda") for _ in range(2))
    bounds = torch.zeros((pages, H, 2, dim), dtype=torch.int8, device="cuda")
    scale = torch.zeros((pages, H), device="cuda")
    weights = torch.full((pages, H, page), float("nan"), device="cuda")  # of pages that nobody used yet
    table = torch.full((R, pages), -1, dtype=torch.int32, device="cuda")
    free = list(range(pages))
    rng.shuffle(free)
    length = torch.zeros(R, dtype=torch.int32, device="cuda")

    def draw(n, heads):
        return _cuda(np.clip(np.round(rng.standard_normal((n, heads, dim)) * 32) / 32, -3.9, 3.9).astype(np.float32), dt)

    evictions = 0
    for step, new in enumerate([[6 * page + 3, 20, 5 * page]] + [[1, 1, 1], [2, 1, 0], [page, 2, 1]] * 4):
        T = sum(new)
        q, nk, nv = draw(T, H * group), draw(T, H), draw(T, H)
        pool = _cuda(np.array(free, np.int32))
        plan = fg.kv_plan(length, _cuda(np.array(new, np.int32)), table, pool, tokens=T, page_size=page)
        assert not plan.refused.any()
        free = free[int(plan.free_head):]
        fg.kv_append(k, v, nk, nv, plan.slot)
        where = (table, plan.query_start, plan.kv_len)
        state = [_host(t) for t in (k, v, table, plan.query_start, plan.kv_len)]
        hk, hv, htable, hstart, hlen = state
        # the whole attention, for the weights
        out, lse = fg.paged_attention(q, k, v, *where, max(new), return_lse=True)
        ref = attention_ref(_host(q), hk, hv, htable, hstart, hlen)
        _check(out, lse, ref, dtype)
        want, tol = weights_ref(_host(q), hk, htable, hstart, hlen, _host(lse), _host(weights))
        fg.attention_weights(q, k, weights, *where, lse)
        got = _host(weights).astype(np.float64)
        assert np.array_equal(np.isnan(got), np.isnan(want)) and (np.abs(np.nan_to_num(got - want)) <= tol).all()
        # the attention over chosen blocks
        summed = _host(bounds).copy(), _host(scale).copy()
        summary_ref(hk, htable, hstart, hlen, *summed)
        fg.kv_summarize(k, bounds, scale, *where, tokens=T)
        assert np.array_equal(_host(bounds), summed[0]) and np.array_equal(_host(scale), summed[1])
        blocks = fg.select_blocks(q, bounds, scale, *where, count, page_size=page, window=window, sinks=sinks)
        assert np.array_equal(_host(blocks), select_ref(_host(q), *summed, htable, hstart, hlen, count, page, window, sinks))
        out, lse = fg.block_attention(q, k, v, *where, blocks, window=window, sinks=sinks, return_lse=True)
        ids = block_ids(_host(blocks), page, H * group, htable.shape[1])
        _check(out, lse, attention_ref(_host(q), hk, hv, htable, hstart, hlen, window=window, sinks=sinks, ids=ids), dtype)
        length = plan.kv_len
        if int(length.max()) > budget:
            evictions += 1
            cut = [hk.copy(), hv.copy(), _host(weights).copy()]
            lens, kept = evict_ref(*cut, htable, hlen, budget, recent, sinks)
            e = fg.kv_evict(k, v, weights, table, length, budget, recent=recent, sinks=sinks)
            assert np.array_equal(_host(e.kv_len), lens) and np.array_equal(_host(e.kept), kept)
            for a, b in zip((k, v, weights), cut):
                assert np.array_equal(_host(a), b, equal_nan=True)
            # the pages behind the budget are free again
            for b in range(R):
                was, now = -(-int(hlen[b]) // page), -(-int(lens[b]) // page)
                free += htable[b, now:was].tolist()
                table[b, now:] = -1
            length = e.kv_len
            starts = torch.nn.functional.pad(torch.cumsum(length, 0), (1, 0)).int()
            fg.kv_summarize(k, bounds, scale, table, starts, length, tokens=R * budget)
            summed = _host(bounds).copy(), _host(scale).copy()
            again = summed[0].copy(), summed[1].copy()
            summary_ref(_host(k), _host(table), _host(starts), _host(length), *again)
            assert np.array_equal(summed[0], again[0]) and np.array_equal(summed[1], again[1])
    assert evictions >= 3


def _step(s):
    """One step's calls on the tensors of a dict; what they return."""
    import flashgann_b200 as fg
    where = (s["table"], s["start"], s["len"])
    fg.kv_summarize(s["k"], s["bounds"], s["scale"], *where, tokens=s["q"].shape[0])
    blocks = fg.select_blocks(s["q"], s["bounds"], s["scale"], *where, s["count"], page_size=s["k"].shape[1], window=9, sinks=2)
    out, lse = fg.block_attention(s["q"], s["k"], s["v"], *where, blocks, window=9, sinks=2, return_lse=True)
    full, sums = fg.paged_attention(s["q"], s["k"], s["v"], *where, 1, return_lse=True)
    fg.attention_weights(s["q"], s["k"], s["weights"], *where, sums)
    e = fg.kv_evict(s["k"], s["v"], s["weights"], s["table"], s["len"], s["budget"], recent=8, sinks=2)
    return [blocks, out, lse, full, sums, e.kv_len, e.kept]


def _state(seed, lens, *, heads=8, kv_heads=2, dim=64, page=16, count=4, budget=200, dtype="bf16"):
    import torch
    rng = np.random.default_rng(seed)
    x = make(rng, ctx=[n - 1 for n in lens], new=[1] * len(lens), heads=heads, kv_heads=kv_heads, dim=dim, page=page)
    dt = _dt(dtype)
    s = dict(q=_cuda(x["q"], dt), k=_cuda(x["k"], dt), v=_cuda(x["v"], dt), table=_cuda(x["table"]), start=_cuda(x["start"]),
             len=_cuda(x["kv_len"]), count=count, budget=budget)
    pages = x["k"].shape[0]
    s["bounds"] = torch.zeros((pages, kv_heads, 2, dim), dtype=torch.int8, device="cuda")
    s["scale"] = torch.zeros((pages, kv_heads), device="cuda")
    s["weights"] = _cuda(rng.random((pages, kv_heads, page)).astype(np.float32))
    all_pages = dict(s, start=_cuda(np.concatenate([[0], np.cumsum(x["kv_len"])]).astype(np.int32)))
    import flashgann_b200 as fg
    fg.kv_summarize(s["k"], s["bounds"], s["scale"], s["table"], all_pages["start"], s["len"], tokens=int(x["kv_len"].sum()))
    return s


WRITTEN = ("k", "v", "weights", "bounds", "scale")


@pytest.mark.parametrize("page,lens", [(16, [300, 17, 150]), (1, [700, 290, 1])])  # one kernel for the selection, and two
def test_captured_steps(page, lens):
    """Two graphs over states of their own, captured side by side and replayed in turn with other inputs, give what eager
    calls give."""
    import torch
    make_state = lambda seed: _state(seed, lens, page=page)  # noqa: E731
    states = [make_state(s) for s in (1, 2)]
    warm = make_state(3)
    _step(warm)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_step(s))
        graphs.append(g)
    for seeds in [(4, 5), (6, 7)]:
        fresh = [make_state(seed) for seed in seeds]
        for s, f in zip(states, fresh):
            for n in WRITTEN + ("q", "table", "len"):
                s[n].copy_(f[n])
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for s, f, got in zip(states, fresh, outs):
            want = _step(f)
            for a, b in zip(got, want):
                assert torch.equal(a, b)
            for n in WRITTEN:
                assert torch.equal(s[n], f[n])
    # shorter requests than those captured
    f = make_state(8)
    for t in (f, states[0]):
        t["len"].fill_(40)
    for n in WRITTEN + ("q", "table"):
        states[0][n].copy_(f[n])
    graphs[0].replay()
    torch.cuda.synchronize()
    for a, b in zip(outs[0], _step(f)):
        assert torch.equal(a, b)


def test_two_streams_at_once():
    """The same steps on two streams at a time, and on a stream that is not the current one."""
    import torch
    import flashgann_b200 as fg
    seeds = list(range(10, 18))
    want = []
    for seed in seeds:
        s = _state(seed, [260, 90, 31, 200] * 3)
        want.append(_step(s) + [s[n] for n in WRITTEN])
    states = [_state(seed, [260, 90, 31, 200] * 3) for seed in seeds]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i, s in enumerate(states):
        with torch.cuda.stream(streams[i % 2]):
            got.append(_step(s) + [s[n] for n in WRITTEN])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for a, b in zip(g, w):
            assert torch.equal(a, b)
    s, f = _state(20, [260, 90]), _state(20, [260, 90])
    where = lambda t: (t["table"], t["start"], t["len"])  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    fg.kv_summarize(s["k"], s["bounds"], s["scale"], *where(s), tokens=2, stream=side)
    blocks = fg.select_blocks(s["q"], s["bounds"], s["scale"], *where(s), 4, page_size=16, window=9, sinks=2, stream=side)
    full, sums = fg.paged_attention(s["q"], s["k"], s["v"], *where(s), 1, return_lse=True, stream=side)
    fg.attention_weights(s["q"], s["k"], s["weights"], *where(s), sums, stream=side)
    e = fg.kv_evict(s["k"], s["v"], s["weights"], s["table"], s["len"], 200, recent=8, sinks=2, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    w = _step(f)
    assert torch.equal(blocks, w[0]) and torch.equal(e.kv_len, w[5]) and torch.equal(e.kept, w[6])
    for n in WRITTEN:
        assert torch.equal(s[n], f[n])


def test_caches_of_more_than_2_31_elements():
    """Pages at the far end of caches, summaries and weights whose offsets pass 32 bits."""
    import torch
    small = _state(30, [300, 130], kv_heads=8, heads=16, dim=128, page=64)
    n = small["k"].shape[0]
    far = 2 ** 31 // small["k"][0].numel() + 10
    big = dict(small, table=torch.where(small["table"] >= 0, small["table"] + far, -1).int())
    for name in ("k", "v"):
        big[name] = torch.zeros((far + n,) + small[name].shape[1:], dtype=small[name].dtype, device="cuda")
        big[name][far:] = small[name]
    # page strides that put the last page past 2^31 and 2^32
    for name, stride in (("bounds", 2 ** 31 // far + 4096), ("weights", 2 ** 31 // far + 1024)):
        shape = (far + n,) + small[name].shape[1:]
        stride = (max(stride, small[name][0].numel()) + 15) // 16 * 16
        flat = torch.zeros(stride * (far + n), dtype=small[name].dtype, device="cuda")
        big[name] = flat.as_strided(shape, (stride,) + small[name].stride()[1:])
        big[name][far:] = small[name]
    big["scale"] = torch.zeros((far + n, 8), device="cuda")
    big["scale"][far:] = small["scale"]
    for a, b in zip(_step(big), _step(small)):
        assert torch.equal(a, b)
    for name in WRITTEN:
        assert torch.equal(big[name][far:], small[name])
        assert not big[name][:far].any()


def test_many_rows_of_one_request_beside_decodes():
    """A prompt's last tokens among many decodes: gone through a few rows at a time."""
    import torch
    import flashgann_b200 as fg
    rng = np.random.default_rng(31)
    x = make(rng, ctx=[30, 60, 7] * 10 + [300], new=[1] * 30 + [40], heads=12, kv_heads=3, dim=64, page=16)
    w = rng.random((x["k"].shape[0], 3, 16)).astype(np.float32)
    for kw in (dict(), dict(window=50, sinks=3)):
        lse = attention_ref(x["q"], x["k"], x["v"], x["table"], x["start"], x["kv_len"], **kw)[1].astype(np.float32)
        got = _cuda(w)
        held = np.where(np.arange(31) % 2, x["kv_len"], 0).astype(np.int32)
        fg.attention_weights(_cuda(x["q"], torch.bfloat16), _cuda(x["k"], torch.bfloat16), got, _cuda(x["table"]), _cuda(x["start"]),
                             _cuda(x["kv_len"]), _cuda(lse), held=_cuda(held), **kw)
        want, tol = weights_ref(x["q"], x["k"], x["table"], x["start"], x["kv_len"], lse, w, held=held, **kw)
        assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("new", [1, 40])  # the kernels of few and of many rows
def test_waits_that_run_out_leave_nan(new):
    """Products that are never issued: the weights that would have come from them are NaN, those before are right, and the
    next call is as ever."""
    import torch
    import flashgann_b200 as fg
    x = make(np.random.default_rng(32), ctx=[4000], new=[new], heads=4, kv_heads=1, dim=64, page=16)
    lse = attention_ref(x["q"], x["k"], x["v"], x["table"], x["start"], x["kv_len"])[1].astype(np.float32)
    args = (_cuda(x["q"], torch.bfloat16), _cuda(x["k"], torch.bfloat16))
    rest = (_cuda(x["table"]), _cuda(x["start"]), _cuda(x["kv_len"]), _cuda(lse))
    w = torch.zeros((x["k"].shape[0], 1, 16), device="cuda")
    good = w.clone()
    fg.attention_weights(*args, good, *rest)
    hook = fg.lib().fg_test_key_weights_lose_blocks
    hook.argtypes = [ctypes.c_int32, ctypes.c_int32]
    hook.restype = None
    try:
        hook(0, 3)
        bad = w.clone()
        fg.attention_weights(*args, bad, *rest)
        torch.cuda.synchronize()
    finally:
        hook(-1, -1)
    seen = torch.zeros_like(w, dtype=torch.bool)
    j = torch.arange(4000 + new, device="cuda")
    seen[rest[0][0, j // 16].long(), 0, j % 16] = True
    assert torch.isnan(bad[seen]).all() and not bad[~seen].any()
    again = w.clone()
    fg.attention_weights(*args, again, *rest)
    assert torch.equal(again, good)


def test_gradients_are_refused_and_writes_counted():
    import torch
    import flashgann_b200 as fg
    s = _state(40, [100, 30])
    where = (s["table"], s["start"], s["len"])
    lse = torch.zeros((2, 8), device="cuda")
    blocks = torch.zeros((2, 2, 3), dtype=torch.int32, device="cuda")

    def calls(q, k):
        return [lambda: fg.kv_summarize(k, s["bounds"], s["scale"], *where, tokens=2),
                lambda: fg.select_blocks(q, s["bounds"], s["scale"], *where, 3, page_size=16, window=4),
                lambda: fg.block_attention(q, k, s["v"], *where, blocks, window=4),
                lambda: fg.attention_weights(q, k, s["weights"], *where, lse),
                lambda: fg.kv_evict(k, s["v"], s["weights"], s["table"], s["len"], 64)]
    q, k = s["q"].clone().requires_grad_(), s["k"].clone().requires_grad_()
    for i, call in enumerate(calls(q, k)):
        with pytest.raises(fg.FlashGANNError, match="gradient"):
            call()
        with torch.no_grad():
            before = {n: s[n]._version for n in WRITTEN if n != "k"} | {"k": k._version}
            call()
            now = {n: s[n]._version for n in WRITTEN if n != "k"} | {"k": k._version}
            wrote = [("bounds", "scale"), (), (), ("weights",), ("k", "v", "weights")][i]
            assert {n for n in now if now[n] > before[n]} == set(wrote)


@pytest.mark.parametrize("call,kw,word", [
    ("kv_summarize", dict(bounds="scale"), "bounds must be int8"), ("kv_summarize", dict(scale="weights"), "scale must be float32"),
    ("kv_summarize", dict(table="scale"), "block_table must be"), ("kv_summarize", dict(k="q"), "caches must be"),
    ("select_blocks", dict(q="bounds"), "q must be"), ("select_blocks", dict(start="len"), "query_start entries"),
    ("block_attention", dict(blocks="start"), "blocks must be int32"), ("block_attention", dict(q="bounds"), "q must be"),
    ("attention_weights", dict(lse="q"), "lse must be float32"), ("attention_weights", dict(weights="scale"), "weights must be float32"),
    ("attention_weights", dict(held="start"), "held and kv_len"), ("kv_evict", dict(weights="bounds"), "weights must be float32"),
    ("kv_evict", dict(table="start2"), "table rows")])
def test_python_calls_refuse_other_tensors(call, kw, word):
    import torch
    import flashgann_b200 as fg
    s = _state(41, [100, 30])
    s["start2"] = s["start"].view(3, 1)
    s["lse"] = torch.zeros((2, 8), device="cuda")
    s["blocks"] = torch.zeros((2, 2, 3), dtype=torch.int32, device="cuda")
    s["held"] = s["len"]
    t = {n: s[kw.get(n, n)] for n in ("q", "k", "v", "bounds", "scale", "weights", "table", "start", "len", "lse", "blocks", "held")}
    where = (t["table"], t["start"], t["len"])
    with pytest.raises((fg.FlashGANNError, RuntimeError), match=word):
        {"kv_summarize": lambda: fg.kv_summarize(t["k"], t["bounds"], t["scale"], *where, tokens=2),
         "select_blocks": lambda: fg.select_blocks(t["q"], t["bounds"], t["scale"], *where, 3, page_size=16, window=4),
         "block_attention": lambda: fg.block_attention(t["q"], t["k"], t["v"], *where, t["blocks"], window=4),
         "attention_weights": lambda: fg.attention_weights(t["q"], t["k"], t["weights"], *where, t["lse"], held=t["held"]),
         "kv_evict": lambda: fg.kv_evict(t["k"], t["v"], t["weights"], t["table"], t["len"], 64)}[call]()
