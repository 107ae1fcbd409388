"""Page summaries and block selection on the GPU against their definitions: whole numbers and single 32-bit roundings,
so that everything has to be equal."""

from __future__ import annotations

import numpy as np
import pytest

from tests.attention_ref import make
from tests.block_ref import select_ref, summary_ref
from tests.test_gpu_attention import _cuda, _dt

pytestmark = pytest.mark.gpu


def _keys(x, dtype, order="phd"):
    k = _cuda(x["k"], _dt(dtype))
    if order == "hpd":
        k = k.transpose(1, 2).contiguous().transpose(1, 2)
    return k


def _summaries(x, dtype="bf16", order="phd", all_pages=True):
    """(bounds, scale) on the GPU and as the definition has them, of all pages or of the step's."""
    import torch
    import flashgann_b200 as fg
    k = _keys(x, dtype, order)
    pages, page, heads, dim = x["k"].shape
    start = np.concatenate([[0], np.cumsum(x["kv_len"])]).astype(np.int32) if all_pages else x["start"]
    bounds = torch.full((pages, heads, 2, dim), 5, dtype=torch.int8, device="cuda")
    scale = torch.full((pages, heads), 9.0, device="cuda")
    want = np.full((pages, heads, 2, dim), 5, np.int8), np.full((pages, heads), 9.0, np.float32)
    summary_ref(k.float().cpu().numpy(), x["table"], start, x["kv_len"], *want)
    fg.kv_summarize(k, bounds, scale, _cuda(x["table"]), _cuda(start), _cuda(x["kv_len"]), tokens=int(start[-1]))
    return (bounds, scale), want


def _same(got, want):
    assert np.array_equal(got[1].cpu().numpy(), want[1])
    assert np.array_equal(got[0].cpu().numpy(), want[0])


# (ctx, new, kv_heads, dim, page, dtype, order)
SUMMARIES = [
    ([0], [1], 1, 64, 16, "bf16", "phd"),
    ([15, 16, 17, 0, 31], [1, 1, 1, 1, 1], 2, 128, 16, "bf16", "phd"),
    ([3, 100, 0, 64], [70, 0, 17, 1], 3, 96, 8, "fp16", "hpd"),
    ([0, 5], [9, 2], 4, 64, 1, "fp16", "phd"),        # pages of one row
    ([10], [300], 1, 96, 128, "bf16", "hpd"),
    ([0, 900], [1000, 3], 2, 128, 64, "fp16", "phd"),
    ([1] * 70, [1] * 70, 8, 64, 2, "bf16", "phd"),
    ([0, 511], [513, 1], 1, 128, 512, "bf16", "phd"),
]


@pytest.mark.parametrize("all_pages", [False, True])
@pytest.mark.parametrize("case", range(len(SUMMARIES)))
def test_summaries(case, all_pages):
    ctx, new, kv_heads, dim, page, dtype, order = SUMMARIES[case]
    x = make(np.random.default_rng(case), ctx=ctx, new=new, heads=kv_heads, kv_heads=kv_heads, dim=dim, page=page)
    if case % 2:  # places behind the last key hold what they like
        for b, n in enumerate(x["kv_len"]):
            for j in range(int(n), -(-int(n) // page) * page):
                x["k"][x["table"][b, j // page], j % page] = np.nan if j % 2 else np.inf
    _same(*_summaries(x, dtype, order, all_pages))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_summaries_of_extreme_keys(dtype):
    """All zero, the least and the largest numbers of the type, one value, infinities and NaN."""
    import torch
    info = torch.finfo(_dt(dtype))
    tiny = info.smallest_normal * info.eps  # the least number
    rng = np.random.default_rng(0)
    x = make(rng, ctx=[0], new=[16 * 12], heads=2, kv_heads=2, dim=64, page=16)
    at = x["table"][0]
    x["k"][at[0]] = 0
    x["k"][at[1]] = tiny * rng.integers(-3, 4, (16, 2, 64))
    x["k"][at[2]] = info.max * rng.choice([-1, 1], (16, 2, 64))
    x["k"][at[3]] = -0.75
    x["k"][at[4], 3, 1, 5] = np.inf
    x["k"][at[5], 15, 0, 63] = -np.inf
    x["k"][at[6], 0, 0, 0] = np.nan
    x["k"][at[7]] = info.max
    x["k"][at[7], 2] = -tiny
    x["k"][at[8]] = -0.0
    x["k"][at[9], :, :, ::2] = 0
    # 127 times as large and as small as one another: quotients that are whole
    x["k"][at[10]] = rng.integers(-127, 128, (16, 2, 64)) / 32
    x["k"][at[10], 0, :, 0] = 127 / 32
    _same(*_summaries(x, dtype))


def test_summaries_of_broken_lengths_and_tables():
    rng = np.random.default_rng(1)
    for change in range(4):
        x = make(rng, ctx=[50, 60, 10], new=[3, 20, 5], heads=2, kv_heads=2, dim=64, page=16)
        if change == 0:
            x["kv_len"] = np.array([2, 0, -5], np.int32)
        elif change == 1:
            x["kv_len"] = x["kv_len"] + np.array([5, 400, 2 ** 31 - 16], np.int32)
        elif change == 2:
            x["table"][0, 3], x["table"][1, 4], x["table"][2, 0] = -1, x["k"].shape[0], 2 ** 31 - 1
        else:
            x["table"][:] = -7
        _same(*_summaries(x, "fp16", all_pages=False))


def _select(x, s, count, window, sinks, dtype="bf16", **kw):
    import flashgann_b200 as fg
    return fg.select_blocks(_cuda(x["q"], _dt(dtype)), *s, _cuda(x["table"]), _cuda(x["start"]), _cuda(x["kv_len"]),
                            count, page_size=x["k"].shape[1], window=window, sinks=sinks, **kw)


def _select_ref(x, want, count, window, sinks):
    return select_ref(x["q"], *want, x["table"], x["start"], x["kv_len"], count, x["k"].shape[1], window, sinks)


# (ctx, new, heads, kv_heads, dim, page, dtype)
SELECTIONS = [
    ([0], [1], 1, 1, 64, 16, "bf16"),
    ([100, 0, 555, 17], [1, 1, 1, 1], 8, 2, 128, 16, "bf16"),
    ([700, 30], [3, 5], 6, 2, 96, 8, "fp16"),
    ([900], [1], 40, 1, 64, 4, "bf16"),                 # 40 heads on one kv head
    ([9000], [1], 9, 3, 128, 2, "fp16"),                # several CTAs to a row
    ([300], [40], 4, 4, 64, 16, "bf16"),                # a chunk, one head each
    ([3, 2000, 0, 60], [0, 2, 4, 1], 5, 1, 96, 1, "bf16"),
    ([40000], [1], 2, 1, 64, 8, "fp16"),
    ([200] * 90, [1] * 90, 16, 8, 64, 4, "bf16"),       # many rows: a CTA to each
    ([290] * 40, [1] * 40, 12, 4, 96, 1, "fp16"),       # the same, more than 256 pages
    ([2300, 100] * 10, [1] * 20, 128, 8, 128, 8, "bf16"),
    ([280] * 80, [1] * 80, 40, 2, 64, 1, "bf16"),       # many rows of many heads
    ([4000] + [50] * 18, [1] * 19, 8, 8, 96, 1, "bf16"),  # many rows of as many pages as one CTA takes
    ([4200] + [10] * 18, [1] * 19, 8, 8, 64, 1, "fp16"),   # and of more
]


@pytest.mark.parametrize("mask", [(0, 0), (1, 0), (17, 4), (64, 100), (100000, 3)])
@pytest.mark.parametrize("case", range(len(SELECTIONS)))
def test_selection(case, mask):
    ctx, new, heads, kv_heads, dim, page, dtype = SELECTIONS[case]
    x = make(np.random.default_rng(case), ctx=ctx, new=new, heads=heads, kv_heads=kv_heads, dim=dim, page=page)
    s, want = _summaries(x, dtype)
    for count in (1, 7, 32, 2000):
        got = _select(x, s, count, *mask, dtype)
        assert np.array_equal(got.cpu().numpy(), _select_ref(x, want, count, *mask)), count
    assert _select(x, s, 0, *mask, dtype).shape == (sum(new), kv_heads, 0)


def test_selection_of_more_pages_than_shared_memory_holds():
    x = make(np.random.default_rng(9), ctx=[61000], new=[1], heads=2, kv_heads=1, dim=64, page=1)
    s, want = _summaries(x)
    for count, mask in [(5, (10, 3)), (1000, (0, 0)), (60000, (100, 0)), (61001, (0, 0))]:
        got = _select(x, s, count, *mask)
        assert np.array_equal(got.cpu().numpy(), _select_ref(x, want, count, *mask)), count


def test_selection_of_many_tokens():
    """Tokens of many requests, some without: the rows of each are found."""
    rng = np.random.default_rng(10)
    new = rng.integers(0, 4, 300).tolist()
    for page in (1, 16):  # one kernel and two
        x = make(rng, ctx=rng.integers(0, 300, 300).tolist(), new=new, heads=4, kv_heads=2, dim=64, page=page)
        s, want = _summaries(x)
        got = _select(x, s, 5, 8, 2)
        assert np.array_equal(got.cpu().numpy(), _select_ref(x, want, 5, 8, 2))


@pytest.mark.parametrize("kv_heads,heads", [(16, 16), (48, 96), (2, 512), (3, 120)])
def test_selection_of_many_heads(kv_heads, heads):
    """More query heads than one CTA keeps."""
    x = make(np.random.default_rng(kv_heads), ctx=[700], new=[2], heads=heads, kv_heads=kv_heads, dim=128, page=2)
    s, want = _summaries(x)
    got = _select(x, s, 9, 20, 2)
    assert np.array_equal(got.cpu().numpy(), _select_ref(x, want, 9, 20, 2))


def test_selection_of_equal_scores():
    """Ties go to the lowest block: all equal, and a few values that repeat."""
    rng = np.random.default_rng(2)
    for kinds in (1, 3):
        x = make(rng, ctx=[5000], new=[1], heads=4, kv_heads=2, dim=64, page=4)
        few = x["k"][:kinds].copy()
        for pg in range(x["k"].shape[0]):
            x["k"][pg] = few[rng.integers(kinds)]
        s, want = _summaries(x)
        for count in (1, 100, 1000):
            got = _select(x, s, count, 10, 4)
            assert np.array_equal(got.cpu().numpy(), _select_ref(x, want, count, 10, 4))


def test_selection_with_extreme_values():
    """Pages and queries of zeros, of infinities and NaN, of numbers near the type's ends; pages that are not there."""
    rng = np.random.default_rng(3)
    x = make(rng, ctx=[800, 800, 800], new=[1, 1, 2], heads=6, kv_heads=2, dim=64, page=8)
    for b in range(3):
        at = x["table"][b]
        x["k"][at[5]] = 0
        x["k"][at[9], 1, 0, 3] = np.nan
        x["k"][at[30], 7, 1, 0] = np.inf
        x["k"][at[31]] = 3e38
        x["k"][at[32]] = -3e38
        x["k"][at[33]] = 1e-38
        x["table"][b, 40], x["table"][b, 41], x["table"][b, 42] = -1, x["k"].shape[0], 2 ** 31 - 1
    x["q"][0, 0], x["q"][0, 1] = 0, np.nan
    x["q"][1, 2, 5] = -np.inf
    x["q"][2, :] = 3e38
    x["q"][3, 3:] = 1e-38
    import torch
    for name in "qk":  # what bfloat16 holds
        x[name] = torch.from_numpy(x[name]).bfloat16().float().numpy()
    s, want = _summaries(x)
    for count in (1, 3, 30, 90, 99):
        got = _select(x, s, count, 5, 2)
        assert np.array_equal(got.cpu().numpy(), _select_ref(x, want, count, 5, 2)), count
    x["table"][:] = -1
    assert (_select(x, s, 4, 5, 2) == -1).all()


def test_selection_of_broken_lengths():
    rng = np.random.default_rng(4)
    for lens in ([1, 0], [5, 5000], [-3, 2 ** 31 - 1]):
        x = make(rng, ctx=[200, 300], new=[2, 3], heads=4, kv_heads=2, dim=64, page=8)
        s, want = _summaries(x)
        x["kv_len"] = np.array(lens, np.int32)
        got = _select(x, s, 9, 16, 2)
        assert np.array_equal(got.cpu().numpy(), _select_ref(x, want, 9, 16, 2))


def test_selection_output_and_strides():
    """Rows past the last request stay; out, q, bounds and scale as slices of larger buffers."""
    import torch
    import flashgann_b200 as fg
    rng = np.random.default_rng(5)
    x = make(rng, ctx=[400, 90], new=[2, 1], heads=4, kv_heads=2, dim=96, page=8)
    (bounds, scale), want = _summaries(x)
    wide = torch.full((5, 3, 20), 77, dtype=torch.int32, device="cuda")
    q = torch.zeros((5, 6, 96), dtype=torch.bfloat16, device="cuda")
    q[:3, :4] = _cuda(x["q"], torch.bfloat16)
    big, bigs = torch.zeros((bounds.shape[0], 5, 2, 96), dtype=torch.int8, device="cuda"), torch.zeros((2, bounds.shape[0]), device="cuda")
    big[:, 1:3], bigs[:] = bounds, scale.T
    out = wide[:, :2, :6]
    got = fg.select_blocks(q[:, :4], big[:, 1:3], bigs.T, _cuda(x["table"]), _cuda(x["start"]), _cuda(x["kv_len"]), 6,
                           page_size=8, window=10, sinks=1, out=out)
    assert got is out
    assert np.array_equal(out[:3].cpu().numpy(), _select_ref(x, want, 6, 10, 1))
    assert (wide[3:] == 77).all() and (wide[:, 2] == 77).all() and (wide[:, :, 6:] == 77).all()
