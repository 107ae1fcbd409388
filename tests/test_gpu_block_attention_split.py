"""Attention over chosen blocks with more and more tiles: on both sides of where each tile gets as many CTAs as any other and
where the work is shared evenly instead."""

from __future__ import annotations

import numpy as np
import pytest

from tests.attention_ref import make
from tests.test_gpu_attention import _check
from tests.test_gpu_block_attention import _lists, _run, _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [15, 40, 58, 59, 69, 70, 98, 100, 103, 104, 147, 149, 177, 178, 200, 236])
def test_block_attention_of_more_and_more_tiles(tokens):
    import torch
    rng = np.random.default_rng(tokens)
    x = make(rng, ctx=[700], new=[tokens], heads=2, kv_heads=1, dim=64, page=16)
    blocks = _lists(rng, x, 40, "ascending")
    out, lse = _run(x, blocks, "bf16", 20, 3)
    _check(out, lse, _want(x, blocks, 20, 3), "bf16")
    for again in (_run(x, blocks, "bf16", 20, 3) for _ in range(3)):  # the same bits on every run
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
