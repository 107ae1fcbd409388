"""Waits of the block selection that run out: products that are never issued.  The rows that would have needed them are -2
throughout, so that nobody takes them for a choice, all others are right, and the next call is as ever."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from tests.attention_ref import make
from tests.block_ref import select_ref, summary_ref
from tests.test_gpu_attention import _cuda

pytestmark = pytest.mark.gpu


def _lose(first, tries):
    import flashgann_b200 as fg
    hook = fg.lib().fg_test_selection_lose_items
    hook.argtypes = [ctypes.c_int32, ctypes.c_int32]
    hook.restype = None
    hook(first, tries)


def _setup(ctx, heads, kv_heads, page):
    """(call(out=None) -> lists, candidates of each token, the lists from the definition)"""
    import torch
    import flashgann_b200 as fg
    x = make(np.random.default_rng(7), ctx=ctx, new=[1] * len(ctx), heads=heads, kv_heads=kv_heads, dim=64, page=page)
    pages = x["k"].shape[0]
    x["table"][0, 2] = -1  # a page that is missing is no reason to give up
    start = np.concatenate([[0], np.cumsum(x["kv_len"])]).astype(np.int32)
    ref = np.zeros((pages, kv_heads, 2, 64), np.int8), np.zeros((pages, kv_heads), np.float32)
    summary_ref(x["k"], x["table"], start, x["kv_len"], *ref)
    args = (_cuda(x["q"], torch.bfloat16), _cuda(ref[0]), _cuda(ref[1]), _cuda(x["table"]), _cuda(x["start"]), _cuda(x["kv_len"]))
    blocks = (x["kv_len"] - 1) // page + 1
    return (lambda: fg.select_blocks(*args, 9, page_size=page, window=0).cpu().numpy(), blocks,
            select_ref(x["q"], *ref, x["table"], x["start"], x["kv_len"], 9, page, 0, 0))


# a CTA to each row; two kernels whose second keeps keys in registers (one CTA size and another) or reads them again
CASES = [([1000, 3, 60, 100, 500] * 8, 8, 4, 2), ([700, 5], 4, 2, 1), ([6000, 3], 2, 2, 1), ([9000], 2, 1, 1)]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_rows_whose_products_are_lost(case):
    import torch
    ctx, heads, kv_heads, page = CASES[case]
    call, blocks, want = _setup(ctx, heads, kv_heads, page)
    assert np.array_equal(call(), want)
    try:
        _lose(0, 3)
        got = call()
        torch.cuda.synchronize()
    finally:
        _lose(-1, -1)
    chooses = blocks > 9  # others have all their pages, and no products
    assert chooses.any()
    assert (got[chooses] == -2).all() and np.array_equal(got[~chooses], want[~chooses])
    assert np.array_equal(call(), want)


def test_rows_before_the_loss_are_right():
    """Many rows: 128 pages are an item, so that rows of up to 128 pages have what they need."""
    ctx, heads, kv_heads, page = CASES[0]
    call, blocks, want = _setup(ctx, heads, kv_heads, page)
    try:
        _lose(1, 3)
        got = call()
    finally:
        _lose(-1, -1)
    longer = blocks > 128
    assert longer.any() and (~longer & (blocks > 9)).any()
    assert (got[longer] == -2).all() and np.array_equal(got[~longer], want[~longer])


def test_the_attention_takes_nothing_from_lists_that_are_lost():
    import torch
    import flashgann_b200 as fg
    x = make(np.random.default_rng(8), ctx=[300], new=[1], heads=4, kv_heads=2, dim=64, page=16)
    args = [_cuda(x[n], torch.bfloat16) for n in "qkv"] + [_cuda(x[n]) for n in ("table", "start", "kv_len")]
    lost = torch.full((1, 2, 5), -2, dtype=torch.int32, device="cuda")
    assert torch.equal(fg.block_attention(*args, lost, window=20, sinks=2), fg.block_attention(*args, lost[..., :0], window=20, sinks=2))
