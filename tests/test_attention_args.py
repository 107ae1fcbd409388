"""Refusals of the cache and attention entry points: checked before any device
work, so they need no GPU."""

from __future__ import annotations

import ctypes

import pytest

import flashgann_b200 as fg
from flashgann_b200 import _capi

PTR = 1 << 20  # a 16-byte aligned address that is never read: every call here is refused first


def _cache(**kw):
    d = dict(k=PTR, v=PTR, page_stride=2048, token_stride=128, head_stride=64, pages=4, page_size=16, heads=2, dim=64,
             dtype=_capi.FG_DTYPE_BF16)
    d.update(kw)
    return _capi.KVCacheArgs(**d)


def _args(**kw):
    d = dict(q=PTR, q_token_stride=256, q_head_stride=64, out=PTR, out_token_stride=256, out_head_stride=64,
             block_table=PTR, table_stride=4, query_start=PTR, kv_len=PTR, ids=PTR, ids_token_stride=40,
             ids_head_stride=10, workspace=PTR, workspace_bytes=0, tokens=3, heads=4, requests=2, table_width=4,
             max_new=2, window=8, sinks=0, ids_count=10, scale=0.125)
    d.update(kw)
    return _capi.AttentionArgs(**d)


CACHE = [(dict(k=None), "null cache"), (dict(dtype=7), "dtype"), (dict(dim=80), "dim 80"), (dict(pages=0), "pages=0"),
         (dict(heads=0), "heads=0"), (dict(page_size=24), "page size 24"), (dict(page_size=0), "page size 0"),
         (dict(v=PTR + 8), "aligned"), (dict(token_stride=132), "strides"), (dict(head_stride=-64), "negative")]
ARGS = [(dict(tokens=-1), "tokens=-1"), (dict(requests=-2), "requests=-2"), (dict(heads=5), "5 query heads"),
        (dict(heads=0), "0 query heads"), (dict(heads=2 * 257), "257 query heads"), (dict(requests=20000), "at most"),
        (dict(window=-2), "window=-2"), (dict(sinks=-1), "sinks=-1"), (dict(scale=float("nan")), "scale"),
        (dict(scale=float("inf")), "scale"), (dict(q=None), "null q"), (dict(q=PTR + 2), "q is not"),
        (dict(q_head_stride=68), "strides of q"), (dict(out=None), "null out"), (dict(out_token_stride=-8), "negative"),
        (dict(query_start=None), "null buffer"), (dict(kv_len=None), "null buffer"), (dict(block_table=None), "null"),
        (dict(table_stride=-1), "table")]
IDS = [(dict(window=-1), "window"), (dict(ids_count=-1), "count -1"), (dict(ids=None), "null"),
       (dict(ids_head_stride=-10), "negative"), (dict(ids_count=70000), "70000 ids")]


def _refused(call, cache, args, word):
    L = fg.lib()
    rc = getattr(L, call)(cache, args, None)
    assert rc in (fg.FG_ERR_ARG, fg.FG_ERR_UNSUPPORTED), rc
    assert word in L.fg_last_error().decode(), L.fg_last_error().decode()


@pytest.mark.parametrize("kw,word", CACHE)
def test_cache_refusals(kw, word):
    _refused("fg_paged_attention_device", _cache(**kw), _args(), word)
    L = fg.lib()
    assert L.fg_kv_append_device(_cache(**kw), PTR, 128, 64, PTR, 128, 64, PTR, 3, None) in (
        fg.FG_ERR_ARG, fg.FG_ERR_UNSUPPORTED)
    assert word in L.fg_last_error().decode()


@pytest.mark.parametrize("kw,word", ARGS)
def test_attention_refusals(kw, word):
    _refused("fg_paged_attention_device", _cache(), _args(**kw), word)
    _refused("fg_retrieved_attention_device", _cache(), _args(**kw), word)


@pytest.mark.parametrize("kw,word", IDS)
def test_retrieved_refusals(kw, word):
    _refused("fg_retrieved_attention_device", _cache(), _args(**kw), word)


def test_null_structs_and_empty_calls():
    L = fg.lib()
    assert L.fg_paged_attention_device(None, _args(), None) == fg.FG_ERR_ARG
    assert L.fg_paged_attention_device(_cache(), None, None) == fg.FG_ERR_ARG
    assert L.fg_attention_workspace_bytes(None, None, 0, None) == fg.FG_ERR_ARG
    # nothing to do: no device is needed
    assert L.fg_paged_attention_device(_cache(), _args(tokens=0, workspace=None), None) == fg.FG_OK
    assert L.fg_retrieved_attention_device(_cache(), _args(requests=0, workspace=None), None) == fg.FG_OK
    assert L.fg_kv_append_device(_cache(), None, 0, 0, None, 0, 0, None, 0, None) == fg.FG_OK


PLAN = [(dict(requests=0), "requests=0"), (dict(requests=9000), "at most"), (dict(page_size=12), "page size 12"),
        (dict(tokens=-1), "tokens=-1"), (dict(free=None), "null"), (dict(table=None), "null"), (dict(slot=None), "null"),
        (dict(ctx=None), "null"), (dict(head=PTR, head_out=PTR), "same buffer"), (dict(width=-1), "table_width=-1")]


@pytest.mark.parametrize("kw,word", PLAN)
def test_plan_refusals(kw, word):
    d = dict(ctx=PTR, new=PTR, requests=2, free=PTR, count=5, head=None, page_size=16, table=PTR, width=4, stride=4,
             tokens=3, qs=PTR, kl=PTR, pos=PTR, slot=PTR, head_out=PTR, refused=PTR)
    d.update(kw)
    L = fg.lib()
    rc = L.fg_kv_plan_device(*d.values(), None)
    assert rc in (fg.FG_ERR_ARG, fg.FG_ERR_UNSUPPORTED)
    assert word in L.fg_last_error().decode()


def test_append_refusals():
    L = fg.lib()
    for args, word in [((None, 128, 64, PTR, 128, 64, PTR, 3), "null k"), ((PTR, 128, 64, None, 128, 64, PTR, 3), "null v"),
                       ((PTR, 130, 64, PTR, 128, 64, PTR, 3), "strides of k"), ((PTR + 4, 128, 64, PTR, 128, 64, PTR, 3), "k is"),
                       ((PTR, 128, 64, PTR, 128, 64, None, 3), "slots"), ((PTR, 128, 64, PTR, 128, 64, PTR, -1), "token")]:
        assert L.fg_kv_append_device(_cache(), *args, None) == fg.FG_ERR_ARG
        assert word in L.fg_last_error().decode()


def test_python_wrappers_refuse_host_tensors():
    import torch
    z = torch.zeros((2, 4, 1, 64), dtype=torch.float16)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(fg.FlashGANNError):
        fg.kv_plan(i, i, i.view(1, 1), i, tokens=1, page_size=4)
    with pytest.raises(fg.FlashGANNError):
        fg.kv_append(z, z, z[0], z[0], i.long())
    with pytest.raises(fg.FlashGANNError):
        fg.paged_attention(z[0], z, z, i.view(1, 1), i, i, 1)
    with pytest.raises(fg.FlashGANNError):
        fg.retrieved_attention(z[0], z, z, i.view(1, 1), i, i, i.view(1, 1, 1), window=4)


def test_struct_sizes():
    """The ctypes mirrors have the C structs' layout (no padding is assumed)."""
    assert ctypes.sizeof(_capi.KVCacheArgs) == 64 and _capi.KVCacheArgs.pages.offset == 40
    assert ctypes.sizeof(_capi.AttentionArgs) == 168 and _capi.AttentionArgs.tokens.offset == 128


@pytest.mark.parametrize("kw", [dict(out_token_stride=0), dict(out_head_stride=0), dict(out_head_stride=56)])
def test_overlapping_outputs_are_refused(kw):
    _refused("fg_paged_attention_device", _cache(), _args(**kw), "rows of out overlap")
    _refused("fg_retrieved_attention_device", _cache(), _args(**kw), "rows of out overlap")


@pytest.mark.parametrize("kw", [dict(page_stride=0), dict(token_stride=0), dict(head_stride=0), dict(head_stride=32)])
def test_append_to_overlapping_rows_is_refused(kw):
    L = fg.lib()
    assert L.fg_kv_append_device(_cache(**kw), PTR, 128, 64, PTR, 128, 64, PTR, 3, None) == fg.FG_ERR_ARG
    assert "rows of the cache overlap" in L.fg_last_error().decode()
