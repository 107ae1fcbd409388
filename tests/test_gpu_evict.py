"""Key weights and eviction on the GPU against their definitions; the weights' tolerance is derived in weights_ref, the
eviction moves numbers and has to be equal."""

from __future__ import annotations

import numpy as np
import pytest

from tests.attention_ref import attention_ref, make
from tests.block_ref import evict_ref, weights_ref
from tests.test_gpu_attention import _cuda, _dt

pytestmark = pytest.mark.gpu


# ---- weights ----

def _lse(x, **kw):
    return attention_ref(x["q"], x["k"], x["v"], x["table"], x["start"], x["kv_len"], **kw)[1].astype(np.float32)


def _weights(rng, x):
    return rng.random((x["k"].shape[0], x["k"].shape[2], x["k"].shape[1])).astype(np.float32) * 3


def _add(x, w, lse, dtype, order="phd", held=None, **kw):
    import flashgann_b200 as fg
    k = _cuda(x["k"], _dt(dtype))
    if order == "hpd":
        k = k.transpose(1, 2).contiguous().transpose(1, 2)
    got = _cuda(w)
    fg.attention_weights(_cuda(x["q"], _dt(dtype)), k, got, _cuda(x["table"]), _cuda(x["start"]), _cuda(x["kv_len"]),
                         _cuda(lse), held=None if held is None else _cuda(held), **kw)
    return got.double().cpu().numpy()


def _check_weights(got, ref):
    want, tol = ref
    assert np.array_equal(np.isnan(got), np.isnan(want))
    err = np.abs(np.where(np.isnan(want), 0, got - want))
    assert (err <= tol).all(), f"worst {np.max(err / np.maximum(tol, 1e-30)):.2f} of the tolerance"


# (ctx, new, heads, kv_heads, dim, page, dtype, order)
WEIGHTS = [
    ([0], [1], 1, 1, 64, 16, "bf16", "phd"),
    ([0, 5, 130, 31], [1, 1, 1, 1], 8, 2, 128, 16, "bf16", "phd"),
    ([700, 0, 3], [1, 0, 1], 5, 1, 64, 1, "fp16", "hpd"),
    ([300], [1], 40, 1, 96, 64, "bf16", "phd"),              # 40 heads on one kv head
    ([10, 200, 33], [4, 3, 5], 12, 4, 96, 32, "fp16", "hpd"),
    ([500], [70], 6, 2, 128, 8, "bf16", "phd"),              # the last tokens of a prompt
    ([0, 90], [33, 1], 4, 4, 64, 256, "fp16", "phd"),        # a prompt beside a decode
    ([40] * 60, [1] * 60, 8, 4, 64, 16, "bf16", "phd"),
    ([170], [110], 12, 3, 96, 16, "bf16", "hpd"),            # more rows than are gone through at once
    ([33, 0], [64, 65], 2, 1, 128, 32, "fp16", "phd"),
]


@pytest.mark.parametrize("mask", [(-1, 0), (0, 0), (1, 0), (17, 4), (64, 100), (0, 3)])
@pytest.mark.parametrize("shape", range(len(WEIGHTS)))
def test_weights(shape, mask):
    ctx, new, heads, kv_heads, dim, page, dtype, order = WEIGHTS[shape]
    rng = np.random.default_rng(shape)
    x = make(rng, ctx=ctx, new=new, heads=heads, kv_heads=kv_heads, dim=dim, page=page)
    w = _weights(rng, x)
    kw = dict(window=mask[0], sinks=mask[1])
    lse = _lse(x, **kw)
    _check_weights(_add(x, w, lse, dtype, order, **kw), weights_ref(x["q"], x["k"], x["table"], x["start"], x["kv_len"], lse, w, **kw))
    # nothing there yet, some, and more than there are
    for held in ([0] * len(ctx), [c // 2 for c in ctx], [10000] * len(ctx), [-3] * len(ctx)):
        held = np.array(held, np.int32)
        got = _add(x, w, lse, dtype, order, held, **kw)
        _check_weights(got, weights_ref(x["q"], x["k"], x["table"], x["start"], x["kv_len"], lse, w, held=held, **kw))


def test_weights_of_a_step_sum_to_its_rows():
    """Every row gives 1 in all, whatever lay in the new pages."""
    x = make(np.random.default_rng(1), ctx=[0, 100], new=[50, 2], heads=6, kv_heads=2, dim=64, page=16)
    w = np.full((x["k"].shape[0], 2, 16), np.nan, np.float32)
    got = _add(x, w, _lse(x), "bf16", held=np.zeros(2, np.int32))
    assert np.allclose(np.nansum(got), 52 * 6, rtol=1e-5)
    assert np.isfinite(got).sum() == 2 * (50 + 102)


def test_weights_of_rows_without_a_sum():
    """lse of -inf, inf and NaN: the row adds nothing; keys that hold infinities or NaN and their rows."""
    rng = np.random.default_rng(2)
    for new in (1, 20):
        x = make(rng, ctx=[60, 30], new=[new, new], heads=6, kv_heads=2, dim=64, page=16)
        w = _weights(rng, x)
        lse = _lse(x)
        lse[0, 0], lse[0, 3], lse[-1, 5], lse[-1, 1] = -np.inf, np.nan, np.inf, np.nan
        _check_weights(_add(x, w, lse, "fp16"), weights_ref(x["q"], x["k"], x["table"], x["start"], x["kv_len"], lse, w))
        x["k"][x["table"][0, 1], 3, 0] = np.nan   # seen by all rows of request 0, kv head 0
        x["k"][x["table"][1, 0], 2, 1, 7] = np.inf
        x["v"][:] = 0
        lse = _lse(x)
        assert not np.isfinite(lse[:new, :3]).any()
        lse[new:, 3:] = np.nan
        got = _add(x, w, lse, "fp16")
        assert np.isfinite(got).all()
        _check_weights(got, weights_ref(x["q"], x["k"], x["table"], x["start"], x["kv_len"], lse, w))
        # outside of the window
        kw = dict(window=5, sinks=0)
        lse = _lse(x, **kw)
        assert np.isfinite(lse).all() or new > 1
        _check_weights(_add(x, w, lse, "fp16", **kw), weights_ref(x["q"], x["k"], x["table"], x["start"], x["kv_len"], lse, w, **kw))


def test_weights_of_broken_lengths_and_tables():
    rng = np.random.default_rng(3)
    for change in range(4):
        x = make(rng, ctx=[90, 120], new=[2, 3], heads=4, kv_heads=2, dim=64, page=8)
        if change == 0:
            x["kv_len"] = np.array([1, 0], np.int32)
        elif change == 1:
            x["kv_len"] = x["kv_len"] + np.array([5, 4000], np.int32)
        elif change == 2:
            x["table"][0, 3], x["table"][1, 5], x["table"][1, 6] = -1, x["k"].shape[0], 2 ** 31 - 1
        else:
            x["table"][:] = -7
        w = _weights(rng, x)
        for kw in (dict(), dict(window=9, sinks=3)):
            lse = np.where(np.isfinite(_lse(x, **kw)), _lse(x, **kw), 0).astype(np.float32)
            _check_weights(_add(x, w, lse, "bf16", **kw), weights_ref(x["q"], x["k"], x["table"], x["start"], x["kv_len"], lse, w, **kw))


def test_weights_scales_strides_and_repeats():
    """A scale of its own; weights as a slice of a larger buffer, lse with strides; the same bits on every run."""
    import torch
    import flashgann_b200 as fg
    rng = np.random.default_rng(4)
    x = make(rng, ctx=[200, 50], new=[3, 1], heads=8, kv_heads=2, dim=96, page=16)
    w = _weights(rng, x)
    for scale in (0.5, -0.125, 0.0):
        lse = _lse(x, scale=scale)
        _check_weights(_add(x, w, lse, "fp16", scale=scale), weights_ref(x["q"], x["k"], x["table"], x["start"], x["kv_len"], lse, w, scale=scale))
    lse = _lse(x)
    ref = weights_ref(x["q"], x["k"], x["table"], x["start"], x["kv_len"], lse, w)
    layers = torch.full((3, w.shape[0], 2, 16), 5.0, device="cuda")
    wide = torch.zeros((8, 4), device="cuda")
    wide[:] = _cuda(lse).T
    args = (_cuda(x["q"], torch.float16), _cuda(x["k"], torch.float16), layers[1], _cuda(x["table"]), _cuda(x["start"]), _cuda(x["kv_len"]), wide.T)
    first = None
    for _ in range(3):
        layers[1] = _cuda(w)
        fg.attention_weights(*args)
        _check_weights(layers[1].double().cpu().numpy(), ref)
        assert first is None or torch.equal(first, layers[1])
        first = layers[1].clone()
    assert (layers[0] == 5).all() and (layers[2] == 5).all()


@pytest.mark.parametrize("new", [1, 9])  # the kernels of few and of many rows
def test_weights_of_tables_for_billions_of_keys(new):
    """Units of work past 2^31 if every request filled its table: 200 requests of a few tokens, whose rows of the table are
    one row of 2^27 pages."""
    import torch
    import flashgann_b200 as fg
    rng = np.random.default_rng(6)
    R, page = 200, 16
    x = make(rng, ctx=[300], new=[0], heads=2, kv_heads=1, dim=64, page=page)
    table = torch.full((1, 2 ** 27), -1, dtype=torch.int32, device="cuda")
    table[0, :x["table"].shape[1]] = _cuda(x["table"][0])
    lens = rng.integers(new, 300, R).astype(np.int32)
    q = (rng.integers(-64, 65, (R * new, 2, 64)) / 32).astype(np.float32)
    lse = (3 + rng.random((R * new, 2))).astype(np.float32)
    w = torch.zeros((x["k"].shape[0], 1, page), device="cuda")
    fg.attention_weights(_cuda(q, torch.bfloat16), _cuda(x["k"], torch.bfloat16), w, table.expand(R, -1),
                         _cuda(np.arange(0, R * new + 1, new, dtype=np.int32)), _cuda(lens), _cuda(lse), held=_cuda(lens))
    j = np.arange(300)
    k = x["k"][x["table"][0, j // page], j % page, 0].astype(np.float64)
    e = np.exp(np.einsum("thd,jd->thj", q.astype(np.float64), k) / 8 - lse[..., None])
    p = (lens[:, None] - new + np.arange(new)).reshape(-1)
    want = np.where(j <= p[:, None, None], e, 0).sum((0, 1))
    got = w[_cuda(x["table"][0, j // page]).long(), 0, _cuda(j % page).long()].double().cpu().numpy()
    # 2 * R * new terms of up to e^10, each off by (10 + 2) 2^-22 of itself, and as many roundings of the sum
    assert (np.abs(got - want) <= want * (12 * 2.0 ** -22 + 2 * R * new * 2.0 ** -24)).all()


def test_weights_of_shared_pages():
    """Requests that share a prompt's pages: the pages get what all of them pay."""
    import torch
    import flashgann_b200 as fg
    rng = np.random.default_rng(5)
    for new in (1, 40):  # both kernels
        x = make(rng, ctx=[96, 96, 96], new=[new] * 3, heads=4, kv_heads=2, dim=64, page=16)
        x["table"][1:, :6] = x["table"][0, :6]
        w = _weights(rng, x)
        lse = _lse(x)
        want = w.astype(np.float64)
        tol = np.zeros_like(want)
        for b in range(3):  # one request after the other
            one = dict(table=x["table"][b:b + 1], start=np.array([0, new]), kv_len=x["kv_len"][b:b + 1])
            rows = slice(b * new, (b + 1) * new)
            got, t = weights_ref(x["q"][rows], x["k"], one["table"], one["start"], one["kv_len"], lse[rows], want.astype(np.float32))
            want, tol = got, tol + t + 2.0 ** -23 * np.abs(got)
        assert (np.abs(_add(x, w, lse, "fp16") - want) <= tol).all()


# ---- eviction ----

def _evict(x, w, budget, recent, sinks, dtype="bf16", order="phd"):
    """(K, V, weights, kv_len, kept) after the call, numpy."""
    import flashgann_b200 as fg
    k, v = _cuda(x["k"], _dt(dtype)), _cuda(x["v"], _dt(dtype))
    if order == "hpd":
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    got = _cuda(w)
    e = fg.kv_evict(k, v, got, _cuda(x["table"]), _cuda(x["kv_len"]), budget, recent=recent, sinks=sinks)
    return [t.float().cpu().numpy() for t in (k, v, got)] + [e.kv_len.cpu().numpy(), e.kept.cpu().numpy()]


def _check_evict(x, w, budget, recent, sinks, **kw):
    want = [x["k"].copy(), x["v"].copy(), w.copy()]
    lens, kept = evict_ref(*want, x["table"], x["kv_len"], budget, recent, sinks)
    got = _evict(x, w, budget, recent, sinks, **kw)
    assert np.array_equal(got[3], lens)
    assert np.array_equal(got[4], kept)
    for g, t in zip(got, want):
        assert np.array_equal(g, t, equal_nan=True)


# (lengths, kv_heads, dim, page, dtype, order, [(budget, recent, sinks)])
EVICTIONS = [
    ([1], 1, 64, 16, "bf16", "phd", [(1, 0, 0), (1, 1, 0)]),
    ([2, 3, 0, 1], 2, 128, 16, "bf16", "phd", [(1, 0, 1), (2, 1, 1), (2, 0, 0)]),
    ([100, 37, 64, 65], 3, 96, 8, "fp16", "hpd", [(64, 16, 4), (64, 0, 0), (64, 60, 4), (36, 5, 31), (1, 0, 0)]),
    ([700], 1, 128, 1, "bf16", "phd", [(512, 100, 3), (699, 0, 0)]),       # 8 CTAs to the row
    ([3000, 10], 2, 64, 64, "fp16", "phd", [(1000, 128, 4), (17, 0, 16)]),
    ([50] * 80, 4, 64, 4, "bf16", "phd", [(20, 4, 1)]),                     # a CTA to each row
]


@pytest.mark.parametrize("case", range(len(EVICTIONS)))
def test_eviction(case):
    lens, kv_heads, dim, page, dtype, order, cuts = EVICTIONS[case]
    rng = np.random.default_rng(case)
    x = make(rng, ctx=lens, new=[0] * len(lens), heads=kv_heads, kv_heads=kv_heads, dim=dim, page=page)
    for budget, recent, sinks in cuts:
        _check_evict(x, np.exp(2 * rng.standard_normal((x["k"].shape[0], kv_heads, page))).astype(np.float32), budget,
                     recent, sinks, dtype=dtype, order=order)
        # few values, many ties; then values of any sign, infinities and NaN
        _check_evict(x, rng.integers(0, 3, (x["k"].shape[0], kv_heads, page)).astype(np.float32), budget, recent, sinks,
                     dtype=dtype, order=order)
        w = rng.standard_normal((x["k"].shape[0], kv_heads, page)).astype(np.float32)
        w[rng.random(w.shape) < 0.2] = np.nan
        w[rng.random(w.shape) < 0.1] = np.inf
        w[rng.random(w.shape) < 0.1] = -np.inf
        w[rng.random(w.shape) < 0.1] = -0.0
        w[rng.random(w.shape) < 0.1] = 0.0
        _check_evict(x, w, budget, recent, sinks, dtype=dtype, order=order)


def test_eviction_with_missing_pages_and_broken_lengths():
    rng = np.random.default_rng(7)
    for change in range(4):
        x = make(rng, ctx=[100, 90, 40], new=[0, 0, 0], heads=2, kv_heads=2, dim=64, page=8)
        if change == 0:
            x["kv_len"] = np.array([-4, 100000, 2 ** 31 - 1], np.int32)
        elif change == 1:
            x["table"][0, 3], x["table"][0, 11], x["table"][1, 1] = -1, x["k"].shape[0], 2 ** 31 - 1
        elif change == 2:
            x["table"][1] = -1
        else:
            x["table"][:, 0] = -5
        w = rng.random((x["k"].shape[0], 2, 8)).astype(np.float32)
        for budget, recent, sinks in [(30, 8, 2), (88, 0, 0)]:
            _check_evict(x, w, budget, recent, sinks)


@pytest.mark.parametrize("R,length", [(20, 26000), (1, 210000)])
def test_eviction_of_more_weights_than_shared_memory_holds(R, length):
    """Keys past a CTA's room are read again in each pass: 1 and 8 CTAs to a row."""
    import torch
    import flashgann_b200 as fg
    H, D, page, budget, recent, sinks = 8, 64, 64, 9000, 1000, 4
    if R == 1:
        H = 1
    g = torch.Generator(device="cuda").manual_seed(R)
    width = -(-length // page)
    pages = R * width
    k, v = (torch.randint(-100, 100, (pages, page, H, D), generator=g, device="cuda").half() for _ in range(2))
    w = torch.randint(0, 5000, (pages, H, page), generator=g, device="cuda").float()  # with ties
    table = torch.randperm(pages, generator=g, device="cuda").int().view(R, width)
    lens = torch.full((R,), length, dtype=torch.int32, device="cuda")
    pos = torch.arange(length, device="cuda")
    rows = table.long()[:, pos // page]
    flat = w[rows[:, None], torch.arange(H, device="cuda")[:, None], pos % page].clone()  # [R, H, length]
    flat[:, :, :sinks], flat[:, :, length - recent:] = np.inf, np.inf
    want = torch.sort(torch.sort(flat, dim=2, descending=True, stable=True).indices[:, :, :budget], dim=2).values
    r, h = torch.arange(R, device="cuda")[:, None, None], torch.arange(H, device="cuda")[:, None]
    src = table.long()[r, want // page]
    wk, wv, ww = k[src, want % page, h], v[src, want % page, h], w[src, h, want % page]
    e = fg.kv_evict(k, v, w, table, lens, budget, recent=recent, sinks=sinks)
    assert torch.equal(e.kept.long(), want) and (e.kv_len == budget).all()
    to = torch.arange(budget, device="cuda")
    dst = table.long()[r, (to // page)[None, None]]
    assert torch.equal(k[dst, to % page, h], wk) and torch.equal(v[dst, to % page, h], wv) and torch.equal(w[dst, h, to % page], ww)
