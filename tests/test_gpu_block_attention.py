"""Attention over chosen blocks on the GPU against its definition in 64 bits (attention over the ids of the blocks'
positions); tolerances as in tests/test_gpu_attention.py."""

from __future__ import annotations

import numpy as np
import pytest

from tests.attention_ref import make
from tests.block_ref import block_ids
from tests.test_gpu_attention import _check, _cuda, _dt, _ref

pytestmark = pytest.mark.gpu


def _run(x, blocks, dtype, window, sinks, order="phd", **kw):
    import torch
    import flashgann_b200 as fg
    dt = _dt(dtype)
    k, v = _cuda(x["k"], dt), _cuda(x["v"], dt)
    if order == "hpd":
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    elif order == "joined":
        kv = torch.stack([k, v], 1)
        k, v = kv[:, 0], kv[:, 1]
    return fg.block_attention(_cuda(x["q"], dt), k, v, _cuda(x["table"]), _cuda(x["start"]), _cuda(x["kv_len"]),
                              _cuda(blocks), window=window, sinks=sinks, return_lse=True, **kw)


def _want(x, blocks, window, sinks, **kw):
    ids = block_ids(blocks, x["k"].shape[1], x["q"].shape[1], x["table"].shape[1])
    return _ref(x, window=window, sinks=sinks, ids=ids, **kw)


def _lists(rng, x, count, kind):
    """Lists of blocks: ascending then -1, as a selection leaves them; in any order with repeats, some of them missing,
    in the future or far out; all the same; none."""
    T, kv_heads = x["q"].shape[0], x["k"].shape[2]
    width = x["table"].shape[1]
    if kind == "none":
        return np.full((T, kv_heads, count), -1, np.int32)
    if kind == "same":
        return np.repeat(rng.integers(0, width, (T, kv_heads, 1)), count, 2).astype(np.int32)
    if kind == "any":
        b = rng.integers(-1, width, (T, kv_heads, count))
        b[rng.random(b.shape) < 0.1] = 2 ** 31 - 1
        b[rng.random(b.shape) < 0.1] = -2 ** 31
        return b.astype(np.int32)
    out = np.full((T, kv_heads, count), -1, np.int32)
    for t in range(T):
        for h in range(kv_heads):
            n = min(width, rng.integers(0, count + 1))
            out[t, h, :n] = np.sort(rng.choice(width, n, replace=False))
    return out


# (ctx, new, heads, kv_heads, dim, page, dtype, order, count)
SHAPES = [
    ([0], [1], 1, 1, 64, 16, "bf16", "phd", 1),
    ([0, 5, 300, 1], [1, 1, 1, 1], 8, 2, 128, 16, "bf16", "phd", 8),
    ([700, 0, 3], [1, 0, 1], 5, 1, 64, 1, "fp16", "joined", 200),        # pages of one row
    ([900], [1], 40, 1, 128, 8, "bf16", "joined", 33),                   # three tiles of heads
    ([10, 200, 33], [4, 3, 5], 12, 4, 96, 32, "fp16", "hpd", 3),         # a few drafted tokens
    ([500], [70], 6, 2, 96, 4, "bf16", "phd", 40),                       # a chunk
    ([3000], [1], 4, 2, 64, 2, "fp16", "phd", 1024),                     # as many as a list may have
    ([2000], [1], 16, 2, 128, 128, "bf16", "hpd", 5),                    # pages of more than a chunk
    ([60] * 100, [1] * 100, 8, 4, 64, 16, "bf16", "phd", 3),
]


@pytest.mark.parametrize("kind", ["ascending", "any", "same", "none"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_block_attention(shape, kind):
    ctx, new, heads, kv_heads, dim, page, dtype, order, count = SHAPES[shape]
    rng = np.random.default_rng(shape)
    x = make(rng, ctx=ctx, new=new, heads=heads, kv_heads=kv_heads, dim=dim, page=page)
    blocks = _lists(rng, x, count, kind)
    for window, sinks in [(0, 0), (1, 0), (17, 5), (100, 3), (33, 200)]:
        out, lse = _run(x, blocks, dtype, window, sinks, order)
        _check(out, lse, _want(x, blocks, window, sinks), dtype)


def test_rows_that_see_nothing():
    """No window, no first tokens, no block: 0 and -inf; lists that hold nothing before the token."""
    import torch
    x = make(np.random.default_rng(1), ctx=[100, 200], new=[1, 2], heads=4, kv_heads=2, dim=64, page=16)
    blocks = np.full((3, 2, 6), -1, np.int32)
    blocks[1] = 15
    out, lse = _run(x, blocks, "bf16", 0, 0)
    assert not out.any() and torch.isneginf(lse).all()
    out, lse = _run(x, blocks[:, :, :0], "bf16", 0, 0)
    assert not out.any() and torch.isneginf(lse).all()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_places_outside_may_hold_anything(value):
    """Keys and values outside of window, first tokens and blocks must not touch a row; those inside do as the formula
    says."""
    rng = np.random.default_rng(2)
    for new in (1, 3):
        x = make(rng, ctx=[400], new=[new], heads=6, kv_heads=2, dim=128, page=16)
        blocks = _lists(rng, x, 6, "ascending")
        blocks[:] = blocks[:1]  # the same for all tokens
        blocks[:, 0], blocks[:, 1] = [2, 3, 9, 11, 20, -1], [1, 4, 5, 12, 13, 21]
        window, sinks = 20, 3
        for h in range(2):
            seen = np.zeros(400 + new, bool)
            seen[:sinks], seen[400 - window + 1:] = True, True
            for b in blocks[0, h]:
                if b >= 0:
                    seen[16 * b:16 * b + 16] = True
            at = np.zeros(x["k"].shape[:2], bool)
            js = np.flatnonzero(seen)
            at[x["table"][0, js // 16], js % 16] = True
            x["k"][~at, h], x["v"][~at, h] = value, value
        out, lse = _run(x, blocks, "bf16", window, sinks)
        _check(out, lse, _want(x, blocks, window, sinks), "bf16")
        assert np.isfinite(out.float().cpu().numpy()).all()
        x["v"][x["table"][0, 2], 5, 0, 7] = value  # a key that kv head 0 sees by its list
        out, lse = _run(x, blocks, "bf16", window, sinks)
        _check(out, lse, _want(x, blocks, window, sinks), "bf16")
        x["k"][x["table"][0, 3], 1, 0, 0] = np.nan
        out, lse = _run(x, blocks, "bf16", window, sinks)
        o = out.float().cpu().numpy()
        assert np.isnan(o[:, :3]).all() and np.isfinite(o[:, 3:]).all()


def test_missing_pages_and_broken_lengths():
    rng = np.random.default_rng(3)
    for change in range(4):
        x = make(rng, ctx=[90, 120], new=[2, 1], heads=4, kv_heads=2, dim=64, page=8)
        blocks = _lists(rng, x, 12, "any")
        if change == 0:
            x["kv_len"] = np.array([1, 0], np.int32)
        elif change == 1:
            x["kv_len"] = x["kv_len"] + np.array([5, 4000], np.int32)
        elif change == 2:
            x["table"][0, 3], x["table"][1, 5] = -1, x["k"].shape[0]
        else:
            x["table"][:] = -7
        out, lse = _run(x, blocks, "fp16", 10, 2)
        _check(out, lse, _want(x, blocks, 10, 2), "fp16")


def test_output_rows_strides_and_streams():
    """Rows past the last request stay; blocks as a slice; another stream; the same bits on every run."""
    import torch
    rng = np.random.default_rng(4)
    x = make(rng, ctx=[300, 20], new=[1, 1], heads=8, kv_heads=2, dim=96, page=16)
    blocks = _lists(rng, x, 9, "any")
    want = _want(x, blocks, 16, 1)
    x["q"] = np.concatenate([x["q"], x["q"]])
    wide = np.concatenate([np.concatenate([blocks, blocks]), np.zeros((4, 3, 9), np.int32)], 1)
    out = torch.full((4, 8, 96), 7.0, dtype=torch.float16, device="cuda")
    import flashgann_b200 as fg
    args = (_cuda(x["q"], torch.float16), _cuda(x["k"], torch.float16), _cuda(x["v"], torch.float16), _cuda(x["table"]),
            _cuda(x["start"]), _cuda(x["kv_len"]), _cuda(wide)[:, :2])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    got, lse = fg.block_attention(*args, window=16, sinks=1, out=out, return_lse=True, stream=stream)
    torch.cuda.current_stream().wait_stream(stream)
    assert got is out and (out[2:] == 7).all()
    _check(out[:2], lse[:2], want, "fp16")
    for _ in range(3):
        assert torch.equal(fg.block_attention(*args, window=16, sinks=1)[:2], out[:2])


def test_all_blocks_are_the_whole_attention():
    """With every block listed the rows see what causal attention sees."""
    import torch
    import flashgann_b200 as fg
    x = make(np.random.default_rng(5), ctx=[700, 33], new=[1, 4], heads=8, kv_heads=2, dim=128, page=16)
    width = x["table"].shape[1]
    blocks = np.broadcast_to(np.arange(width, dtype=np.int32), (5, 2, width)).copy()
    out, lse = _run(x, blocks, "bf16", 8, 0)
    _check(out, lse, _ref(x), "bf16")
