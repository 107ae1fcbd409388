"""Refusals of the key weights and of the eviction: checked before any device work, so they need no GPU."""

from __future__ import annotations

import pytest

import flashgann_b200 as fg
from tests.test_attention_args import ARGS, CACHE, PTR, _args, _cache


def _weights(cache=None, args=None, w=PTR, page_stride=32, head_stride=16, held=None):
    return fg.lib().fg_attention_weights_device(cache or _cache(), args or _args(lse=PTR), w, page_stride, head_stride,
                                                held, None)


def _evict(cache=None, **kw):
    d = dict(w=PTR, page_stride=32, head_stride=16, table=PTR, width=4, stride=4, kv_len=PTR, requests=2, budget=8,
             recent=2, sinks=1, out=PTR + 64, kept=PTR)
    d.update(kw)
    return fg.lib().fg_kv_evict_device(cache or _cache(), *d.values(), None)


def _refused(rc, word):
    assert rc in (fg.FG_ERR_ARG, fg.FG_ERR_UNSUPPORTED), rc
    assert word in fg.lib().fg_last_error().decode(), fg.lib().fg_last_error().decode()


@pytest.mark.parametrize("kw,word", CACHE)
def test_caches_are_refused(kw, word):
    if kw != dict(v=PTR + 8):  # the weights read the keys alone
        _refused(_weights(_cache(**kw)), word)
    _refused(_evict(_cache(**kw)), word)


@pytest.mark.parametrize("kw,word", [c for c in ARGS if not any(n.startswith("out") for n in c[0])])
def test_arguments_are_refused_as_by_the_attention(kw, word):
    _refused(_weights(args=_args(lse=PTR, **kw)), word)


@pytest.mark.parametrize("kw,word", [
    (dict(w=None), "null weights"), (dict(w=PTR + 2), "aligned"), (dict(page_stride=-32), "negative"),
    (dict(head_stride=-16), "negative"), (dict(head_stride=15), "overlap"), (dict(page_stride=16), "overlap"),
    (dict(page_stride=0), "overlap")])
def test_weights_are_refused(kw, word):
    _refused(_weights(**kw), word)
    _refused(_evict(**kw), word)


def test_null_lse_is_refused():
    _refused(_weights(args=_args(lse=None)), "null lse")


@pytest.mark.parametrize("kw,word", [
    (dict(requests=-1), "requests=-1"), (dict(width=-1), "table_width=-1"), (dict(budget=0), "budget 0"),
    (dict(recent=-1), "recent=-1"), (dict(sinks=-1), "sinks=-1"), (dict(recent=8), "recent=8"),
    (dict(recent=2 ** 31 - 1, sinks=2 ** 31 - 1), "recent"), (dict(kv_len=None), "null buffer"),
    (dict(out=None), "null buffer"), (dict(kept=None), "null buffer"), (dict(table=None), "null buffer"),
    (dict(out=PTR), "same buffer"), (dict(stride=-1), "table stride"), (dict(requests=2 ** 29), "requests of 2 heads")])
def test_evictions_are_refused(kw, word):
    _refused(_evict(**kw), word)


@pytest.mark.parametrize("kw", [dict(page_stride=0), dict(token_stride=0), dict(head_stride=32)])
def test_eviction_from_overlapping_rows_is_refused(kw):
    _refused(_evict(_cache(**kw)), "rows of the cache overlap")


def test_empty_calls_and_null_structs():
    assert _weights(args=_args(lse=None, tokens=0)) == fg.FG_OK
    assert _weights(args=_args(lse=None, requests=0)) == fg.FG_OK
    assert _weights(_cache(v=None), _args(lse=None, requests=0)) == fg.FG_OK
    assert _evict(requests=0, kv_len=None, out=None, kept=None) == fg.FG_OK
    L = fg.lib()
    assert L.fg_attention_weights_device(None, _args(lse=PTR), PTR, 32, 16, None, None) == fg.FG_ERR_ARG
    assert L.fg_attention_weights_device(_cache(), None, PTR, 32, 16, None, None) == fg.FG_ERR_ARG


def test_python_wrappers_refuse_host_tensors():
    import torch
    z = torch.zeros((2, 4, 1, 64), dtype=torch.float16)
    i, w = torch.zeros(1, dtype=torch.int32), torch.zeros((2, 1, 4))
    with pytest.raises(fg.FlashGANNError):
        fg.attention_weights(z[0], z, w, i.view(1, 1), i, i, torch.zeros((4, 1)))
    with pytest.raises(fg.FlashGANNError):
        fg.kv_evict(z, z, w, i.view(1, 1), i, 4)
    with pytest.raises(fg.FlashGANNError):
        fg.block_attention(z[0], z, z, i.view(1, 1), i, i, i.view(1, 1, 1), window=4)
