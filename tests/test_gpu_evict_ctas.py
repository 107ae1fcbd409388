"""Eviction on both sides of each limit of the choice of CTAs to a row: by the table's room and by the number of rows."""

from __future__ import annotations

import numpy as np
import pytest

from tests.attention_ref import make
from tests.test_gpu_evict import _check_evict

pytestmark = pytest.mark.gpu


# one row: one CTA, four, eight; 40 rows: one and two; 20 rows: one and four
@pytest.mark.parametrize("requests,kv_heads,room", [(1, 1, 640), (1, 1, 656), (1, 1, 2048), (1, 1, 2064), (10, 4, 656), (10, 4, 2064),
                                                    (10, 2, 640), (10, 2, 656), (10, 2, 2064)])
def test_eviction_on_both_sides_of_the_limits(requests, kv_heads, room):
    rng = np.random.default_rng(room + requests)
    for longest in (room, 130):  # as long as the table allows, and far shorter
        lens = [longest] + rng.integers(1, longest + 1, requests - 1).tolist()
        x = make(rng, ctx=lens, new=[0] * requests, heads=kv_heads, kv_heads=kv_heads, dim=64, page=16)
        x["table"] = np.pad(x["table"], ((0, 0), (0, 200)), constant_values=-1)[:, :room // 16]
        for budget, recent, sinks in ((longest - 1, 0, 0), (longest // 3, 20, 4)):
            w = rng.integers(0, 50, (x["k"].shape[0], kv_heads, 16)).astype(np.float32)
            _check_evict(x, w, budget, recent, sinks)
