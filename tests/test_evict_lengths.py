"""Eviction refuses an output of lengths that lies over the lengths it reads, which all kv heads' CTAs read until the end."""

from __future__ import annotations

import pytest

import flashgann_b200 as fg
from tests.test_attention_args import PTR
from tests.test_evict_args import _evict, _refused


@pytest.mark.parametrize("by", [-12, -8, -4, 0, 4, 8, 12])
def test_lengths_that_overlap_are_refused(by):
    _refused(_evict(requests=4, kv_len=PTR + 64, out=PTR + 64 + by), "overlap" if by else "same buffer")


@pytest.mark.parametrize("by", [-16, 16])
def test_lengths_beside_each_other_are_not(by):
    """Taken for good, so that the next thing that is wrong is told."""
    _refused(_evict(requests=4, kv_len=PTR + 64, out=PTR + 64 + by, stride=-1), "table stride")
