"""The search by which block selection and page summaries find a row's or a page's request: the arithmetic that the
kernels run, stepped through on the host."""

from __future__ import annotations

import pytest

import flashgann_b200 as fg


@pytest.mark.parametrize("n", list(range(1, 140)) + [255, 256, 257, 1000, 1023, 1024, 1025, 1057, 4095, 4096, 4097, 100003])
def test_search_ends_at_the_first_past_or_the_last(n):
    """None past (a row behind the last request) is the last place, not the one behind it."""
    search = fg.lib().fg_test_first_past
    firsts = range(n + 1) if n < 1100 else [0, 1, 31, 32, 33, n // 32, n // 32 + 1, n // 2, n - 33, n - 32, n - 2, n - 1, n]
    for first in firsts:
        assert search(n, first) == min(first, n - 1), first
    assert search(n, 2 ** 31 - 1) == n - 1
