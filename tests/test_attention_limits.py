"""What the cache and attention entry points refuse at the ends of their ranges: checked before any device work, so
no GPU is needed."""

from __future__ import annotations

import ctypes

import pytest

import flashgann_b200 as fg
from tests.test_attention_args import ARGS, IDS, _args, _cache

# those that say something about counts, the mask or the scale; the rest are buffers and strides
COUNTS = [(kw, word) for kw, word in ARGS if set(kw) & {"tokens", "requests", "heads", "window", "sinks", "scale"}]


@pytest.mark.parametrize("retrieved,kw,word",
                         [(r, kw, w) for r in (0, 1) for kw, w in COUNTS + [(dict(max_new=-1), "max_new=-1"),
                                                                            (dict(table_width=-1), "table_width=-1")]]
                         + [(1, kw, w) for kw, w in IDS if set(kw) & {"window", "ids_count"}]
                         + [(1, dict(ids_count=n), f"{n} ids") for n in (1025, 2 ** 31 - 1)])
def test_workspace_bytes_refuses_what_the_call_refuses(retrieved, kw, word):
    """The size is computed from the counts: it is refused wherever the call itself is, 1025 ids among them."""
    L = fg.lib()
    need = ctypes.c_uint64(7)
    rc = L.fg_attention_workspace_bytes(_cache(), _args(**kw), retrieved, ctypes.byref(need))
    assert rc in (fg.FG_ERR_ARG, fg.FG_ERR_UNSUPPORTED), rc
    assert word in L.fg_last_error().decode(), L.fg_last_error().decode()
    assert need.value == 7
