"""Key weights of requests that bring no rows to a call: weights from held[b] to kv_len[b] start at 0 there too, whatever was
there, and all others stay as they are."""

from __future__ import annotations

import numpy as np
import pytest

from tests.attention_ref import attention_ref, make
from tests.block_ref import weights_ref
from tests.test_gpu_attention import _cuda

pytestmark = pytest.mark.gpu


def _want(x, lse, w, held, **kw):
    """weights_ref, which looks at requests with rows alone, and the others' beginnings."""
    want, tol = weights_ref(x["q"], x["k"], x["table"], x["start"], x["kv_len"], lse, w, held=held, **kw)
    pages, page = x["k"].shape[:2]
    for b in np.flatnonzero(np.diff(x["start"]) == 0):
        for j in range(max(0, int(held[b])), min(int(x["kv_len"][b]), x["table"].shape[1] * page)):
            pg = x["table"][b, j // page]
            if 0 <= pg < pages:
                want[pg, :, j % page] = 0
    return want, tol


def _add(x, w, lse, held, **kw):
    import torch
    import flashgann_b200 as fg
    got = _cuda(w)
    fg.attention_weights(_cuda(x["q"], torch.bfloat16), _cuda(x["k"], torch.bfloat16), got, _cuda(x["table"]), _cuda(x["start"]),
                         _cuda(x["kv_len"]), _cuda(lse), held=None if held is None else _cuda(held), **kw)
    return got.cpu().numpy()


# (tokens in the cache, new ones, held): the kernels of few and of many rows; nobody has rows; more requests than a warp has lanes
BATCHES = [
    ([300, 50, 700], [0, 1, 0], [0, 50, 129]),
    ([300, 50, 700, 90], [0, 70, 0, 3], [128, 50, 600, 0]),
    ([40, 500, 260], [0, 0, 0], [40, 77, -5]),
    ([200] * 20 + [31] * 21, [0, 2, 0] * 13 + [0, 9], [199, 3, 0] * 13 + [50, 31]),
    ([100, 100], [0, 1], [100, 100]),
    ([6000], [0], [1]),
]


@pytest.mark.parametrize("mask", [(-1, 0), (9, 4), (0, 300)])
@pytest.mark.parametrize("batch", range(len(BATCHES)))
def test_weights_of_requests_without_rows(batch, mask):
    ctx, new, held = BATCHES[batch]
    rng = np.random.default_rng(batch)
    for dim, page in ((64, 16), (96, 1), (128, 64)):
        x = make(rng, ctx=ctx, new=new, heads=6, kv_heads=2, dim=dim, page=page)
        kw = dict(window=mask[0], sinks=mask[1])
        lse = attention_ref(x["q"], x["k"], x["v"], x["table"], x["start"], x["kv_len"], **kw)[1].astype(np.float32)
        lse = lse.reshape(-1, 6)
        w = rng.random((x["k"].shape[0], 2, page)).astype(np.float32)
        h = np.array(held, np.int32)
        for change in range(2):
            if change:  # what lay there before, and pages that are missing
                for b in range(len(ctx)):
                    j = np.arange(max(0, held[b]), ctx[b] + new[b])
                    w[x["table"][b, j // page], :, j % page] = np.nan
                x["table"][0, x["table"].shape[1] // 2] = -1
                lse = np.where(np.isfinite(lse), lse, 0)
            want, tol = _want(x, lse, w, h, **kw)
            got = _add(x, w, lse, h, **kw)
            assert np.array_equal(np.isnan(got), np.isnan(want))
            assert (np.abs(np.where(np.isnan(want), 0, got - want)) <= tol).all()
            still = tol == 0  # moved to 0 or not at all
            assert np.array_equal(got[still], want[still].astype(np.float32), equal_nan=True)


def test_nobody_has_new_tokens():
    """The default is to hold all: nothing is written."""
    rng = np.random.default_rng(0)
    x = make(rng, ctx=[40, 500], new=[0, 0], heads=6, kv_heads=2, dim=64, page=16)
    w = rng.random((x["k"].shape[0], 2, 16)).astype(np.float32)
    assert np.array_equal(_add(x, w, np.zeros((0, 6), np.float32), None), w)


def test_lengths_past_the_table_and_negative_ones():
    rng = np.random.default_rng(1)
    x = make(rng, ctx=[100, 100, 100], new=[0, 0, 1], heads=4, kv_heads=2, dim=64, page=16)
    w = rng.random((x["k"].shape[0], 2, 16)).astype(np.float32)
    x["kv_len"] = np.array([2 ** 31 - 1, -4, 101], np.int32)
    lse = np.full((1, 4), 3, np.float32)
    for held in ([0, -9, 101], [110, 0, 101], [2 ** 31 - 1, 2 ** 31 - 1, 101]):
        want, tol = _want(x, lse, w, np.array(held, np.int32))
        assert (np.abs(_add(x, w, lse, np.array(held, np.int32)) - want) <= tol).all()
