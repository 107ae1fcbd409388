"""Which blocks are chosen from, where window and first tokens come near each other: those with x * page <= p - window and
(x + 1) * page > sinks."""

from __future__ import annotations

import numpy as np
import pytest

from tests.attention_ref import make
from tests.test_gpu_attention import _cuda

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requests", [1, 150])  # a CTA of threads to each row, and one of the tensor cores
@pytest.mark.parametrize("length", [24, 25, 27, 28, 29, 31, 40, 41, 57])
def test_window_and_first_tokens_in_one_block(requests, length):
    import torch
    import flashgann_b200 as fg
    page, window, sinks = 16, 8, 20
    x = make(np.random.default_rng(length), ctx=[length - 1] * requests, new=[1] * requests, heads=2, kv_heads=1, dim=64, page=page)
    q, k, v = (_cuda(x[n], torch.bfloat16) for n in "qkv")
    where = _cuda(x["table"]), _cuda(x["start"]), _cuda(x["kv_len"])
    bounds = torch.zeros((k.shape[0], 1, 2, 64), dtype=torch.int8, device="cuda")
    scale = torch.zeros((k.shape[0], 1), device="cuda")
    starts = _cuda(np.arange(requests + 1, dtype=np.int32) * length)
    fg.kv_summarize(k, bounds, scale, where[0], starts, where[2], tokens=requests * length)
    p = length - 1
    want = [b for b in range(-(-length // page)) if b * page <= p - window and (b + 1) * page > sinks]
    for count in (4, 1):  # all of them, and fewer than there may be
        got = fg.select_blocks(q, bounds, scale, *where, count, page_size=page, window=window, sinks=sinks)
        if len(want) <= count:
            assert (got.cpu().numpy() == want + [-1] * (count - len(want))).all()
        else:
            assert np.isin(got.cpu().numpy(), want).all()
    # one without a position of its own adds nothing
    if not any(sinks <= j <= p - window for j in range(length)):
        none = torch.full_like(got, -1)
        assert torch.equal(fg.block_attention(q, k, v, *where, got, window=window, sinks=sinks),
                           fg.block_attention(q, k, v, *where, none, window=window, sinks=sinks))
