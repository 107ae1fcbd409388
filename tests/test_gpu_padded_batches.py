"""Batches in larger buffers, as a serving loop keeps them: query_start, kv_len and block_table are leading slices, what lies
behind them looks like one more request, and q has rows that belong to none.  Nothing behind the slices is looked at."""

from __future__ import annotations

import numpy as np
import pytest

from tests.attention_ref import make
from tests.block_ref import select_ref, summary_ref
from tests.test_gpu_attention import _cuda

pytestmark = pytest.mark.gpu

REQUESTS = [1, 2, 31, 33, 34, 64, 70]


def _batch(rng, requests, new, *, kv_heads, group=2, page=4, width=0, rows_behind=9):
    """A batch of `requests`, the last third of them without new tokens, and the same with one request more behind it,
    whose pages are no other's.  (x, leading slices on the GPU, queries with rows behind the last request)"""
    lens = rng.integers(1, 60, requests)
    count = np.where(np.arange(requests) < max(1, requests - requests // 3), new, 0)
    x = make(rng, ctx=lens.tolist(), new=count.tolist(), heads=kv_heads * group, kv_heads=kv_heads, dim=64, page=page, spare=40)
    if width > x["table"].shape[1]:
        x["table"] = np.pad(x["table"], ((0, 0), (0, width - x["table"].shape[1])), constant_values=-1)
    unused = np.setdiff1d(np.arange(x["k"].shape[0]), x["table"]).astype(np.int32)
    assert len(unused) == 40
    W, T = x["table"].shape[1], int(x["start"][-1])
    behind = np.full((1, W), -1, np.int32)
    behind[0, :min(W, 40)] = unused[:min(W, 40)]
    start = _cuda(np.concatenate([x["start"], [T + rows_behind] * 2]).astype(np.int32))
    kv_len = _cuda(np.concatenate([x["kv_len"], [40 * page] * 2]).astype(np.int32))
    table = _cuda(np.concatenate([x["table"], behind, behind]))
    q = np.concatenate([x["q"], np.ones((rows_behind,) + x["q"].shape[1:], np.float32)])
    R = requests
    return x, (table[:R], start[:R + 1], kv_len[:R]), q


@pytest.mark.parametrize("requests", REQUESTS)
@pytest.mark.parametrize("page", [1, 4, 16])
def test_summaries_of_an_upper_bound_of_tokens(requests, page):
    """tokens may be more than there are: the pages of the listed requests are written, and no other."""
    import torch
    import flashgann_b200 as fg
    x, where, q = _batch(np.random.default_rng(requests), requests, 3, kv_heads=2, page=page)
    pages, _, heads, dim = x["k"].shape
    want = np.full((pages, heads, 2, dim), 5, np.int8), np.full((pages, heads), 9.0, np.float32)
    summary_ref(x["k"], x["table"], x["start"], x["kv_len"], *want)
    for tokens in (int(x["start"][-1]), len(q), len(q) + 1000):
        bounds = torch.full(want[0].shape, 5, dtype=torch.int8, device="cuda")
        scale = torch.full(want[1].shape, 9.0, device="cuda")
        fg.kv_summarize(_cuda(x["k"], torch.bfloat16), bounds, scale, *where, tokens=tokens)
        assert np.array_equal(bounds.cpu().numpy(), want[0]) and np.array_equal(scale.cpu().numpy(), want[1])


# (kv heads, width of the table): few rows and short tables, few and long, many and short, many and long, many and longer
# than one kernel takes
KINDS = [(1, 0), (1, 300), (40, 0), (40, 300), (40, 4100)]


@pytest.mark.parametrize("requests", REQUESTS)
@pytest.mark.parametrize("kind", range(len(KINDS)))
def test_selection_leaves_rows_behind_the_last_request(requests, kind):
    import torch
    import flashgann_b200 as fg
    kv_heads, width = KINDS[kind]
    x, where, q = _batch(np.random.default_rng(requests), requests, 1, kv_heads=kv_heads, width=width)
    pages, page, _, dim = x["k"].shape
    T, count = int(x["start"][-1]), 5
    start = np.concatenate([[0], np.cumsum(x["kv_len"])]).astype(np.int32)
    ref = np.zeros((pages, kv_heads, 2, dim), np.int8), np.zeros((pages, kv_heads), np.float32)
    summary_ref(x["k"], x["table"], start, x["kv_len"], *ref)
    out = torch.full((len(q), kv_heads, count), 77, dtype=torch.int32, device="cuda")
    fg.select_blocks(_cuda(q, torch.bfloat16), _cuda(ref[0]), _cuda(ref[1]), *where, count, page_size=page, window=8, sinks=2, out=out)
    want = select_ref(x["q"], *ref, x["table"], x["start"], x["kv_len"], count, page, 8, 2)
    assert np.array_equal(out[:T].cpu().numpy(), want)
    assert (out[T:] == 77).all()


@pytest.mark.parametrize("requests", REQUESTS)
def test_attention_and_weights_leave_what_is_behind(requests):
    """The attention over blocks and the key weights of the same batches: output rows past the last request and weights of
    pages that no listed request has stay as they were."""
    import torch
    import flashgann_b200 as fg
    for new in (1, 20):
        x, where, q = _batch(np.random.default_rng(requests), requests, new, kv_heads=2)
        T = int(x["start"][-1])
        k, v = (_cuda(x[n], torch.bfloat16) for n in "kv")
        queries = _cuda(q, torch.bfloat16)
        out = torch.full(q.shape, 77.0, dtype=torch.bfloat16, device="cuda")
        blocks = torch.arange(5, dtype=torch.int32, device="cuda").expand(len(q), 2, 5)
        _, lse = fg.block_attention(queries, k, v, *where, blocks, window=8, out=out, return_lse=True)
        assert (out[T:] == 77).all() and not (out[:T] == 77).all(-1).any()
        w = torch.full((x["k"].shape[0], 2, 4), 3.0, device="cuda")
        fg.attention_weights(queries, k, w, *where, torch.zeros((len(q), 4), device="cuda"))
        others = torch.ones(x["k"].shape[0], dtype=torch.bool, device="cuda")
        others[where[0][where[0] >= 0].long()] = False
        assert int(others.sum()) == 40 and (w[others] == 3).all() and not (w[~others] == 3).all()
