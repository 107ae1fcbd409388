"""Refusals of the page summaries and of the block selection: checked before any device work, so they need no GPU."""

from __future__ import annotations

import ctypes

import pytest

import flashgann_b200 as fg
from flashgann_b200 import _capi
from tests.test_attention_args import CACHE, PTR, _cache


def _summary(**kw):
    d = dict(bounds=PTR, scale=PTR, bounds_page_stride=256, bounds_head_stride=128, scale_page_stride=2,
             scale_head_stride=1, pages=4, page_size=16, heads=2, dim=64)
    d.update(kw)
    return _capi.KVSummaryArgs(**d)


def _selection(**kw):
    d = dict(q=PTR, q_token_stride=256, q_head_stride=64, block_table=PTR, table_stride=4, query_start=PTR, kv_len=PTR,
             blocks=PTR, blocks_token_stride=20, blocks_head_stride=10, tokens=3, heads=4, requests=2, table_width=4,
             window=8, sinks=0, count=10, dtype=_capi.FG_DTYPE_BF16)
    d.update(kw)
    return _capi.BlockSelectionArgs(**d)


def _summarize(cache=None, summary=None, **kw):
    d = dict(table=PTR, width=4, stride=4, query_start=PTR, kv_len=PTR, requests=2, tokens=3)
    d.update(kw)
    return fg.lib().fg_kv_summarize_device(cache or _cache(), summary or _summary(), *d.values(), None)


def _refused(rc, word):
    assert rc in (fg.FG_ERR_ARG, fg.FG_ERR_UNSUPPORTED), rc
    assert word in fg.lib().fg_last_error().decode(), fg.lib().fg_last_error().decode()


SUMMARY = [(dict(bounds=None), "null summary"), (dict(scale=None), "null summary"), (dict(dim=80), "dim 80"),
           (dict(pages=0), "pages=0"), (dict(heads=0), "heads=0"), (dict(page_size=24), "page size 24"),
           (dict(bounds=PTR + 8), "aligned"), (dict(scale=PTR + 2), "aligned"), (dict(bounds_page_stride=264), "strides"),
           (dict(bounds_head_stride=-128), "negative"), (dict(scale_page_stride=-2), "negative")]
REQUESTS = [(dict(requests=-1), "requests=-1"), (dict(tokens=-1), "tokens=-1"), (dict(query_start=None), "null buffer"),
            (dict(kv_len=None), "null buffer")]


@pytest.mark.parametrize("kw,word", [c for c in CACHE if c[0] != dict(v=PTR + 8)])
def test_summaries_refuse_caches(kw, word):
    _refused(_summarize(cache=_cache(**kw)), word)


@pytest.mark.parametrize("kw,word", SUMMARY)
def test_summary_refusals(kw, word):
    _refused(_summarize(summary=_summary(**kw)), word)
    _refused(fg.lib().fg_select_blocks_device(_summary(**kw), _selection(), None), word)


@pytest.mark.parametrize("kw,word", REQUESTS + [(dict(width=-1), "table_width=-1"), (dict(table=None), "null buffer"),
                                                (dict(stride=-4), "table stride"), (dict(requests=2 ** 30), "2 heads")])
def test_summarize_refuses_requests(kw, word):
    _refused(_summarize(**kw), word)


@pytest.mark.parametrize("kw", [dict(pages=5), dict(page_size=8), dict(heads=1), dict(dim=128)])
def test_summarize_refuses_another_caches_summary(kw):
    _refused(_summarize(summary=_summary(**kw)), "not of this cache")


@pytest.mark.parametrize("kw", [dict(bounds_page_stride=128), dict(bounds_head_stride=0), dict(scale_page_stride=0),
                                dict(scale_page_stride=1), dict(scale_head_stride=2)])
def test_summarize_refuses_overlapping_summaries(kw):
    _refused(_summarize(summary=_summary(**kw)), "rows of the summary overlap")
    # the selection only reads them
    _refused(fg.lib().fg_select_blocks_device(_summary(**kw), _selection(blocks=None), None), "null blocks")


@pytest.mark.parametrize("kw,word", REQUESTS + [
    (dict(table_width=-1), "table_width=-1"), (dict(block_table=None), "null buffer"), (dict(table_stride=-1), "stride"),
    (dict(dtype=5), "dtype"), (dict(heads=5), "5 query heads"), (dict(heads=0), "0 query heads"),
    (dict(heads=2 * 257), "257 query heads"), (dict(window=-1), "window=-1"), (dict(sinks=-1), "sinks=-1"),
    (dict(count=-1), "count -1"), (dict(table_width=257), "workspace is null"),
    (dict(table_width=257, workspace=PTR + 8, workspace_bytes=1 << 20), "16-byte aligned"),
    (dict(table_width=257, workspace=PTR, workspace_bytes=3 * 2 * 257 * 4 - 1), "6168 needed"),
    (dict(table_width=2 ** 31 - 1, tokens=1000), "blocks"), (dict(tokens=2 ** 30), "tokens"),
    (dict(q=None), "null q"), (dict(q=PTR + 8), "q is not"), (dict(q_head_stride=4), "strides of q"),
    (dict(blocks=None), "null blocks"), (dict(blocks_head_stride=9), "overlap"), (dict(blocks_token_stride=0), "overlap")])
def test_selection_refusals(kw, word):
    _refused(fg.lib().fg_select_blocks_device(_summary(), _selection(**kw), None), word)


@pytest.mark.parametrize("kw,word", [(dict(requests=-1), "requests=-1"), (dict(heads=5), "5 query heads"),
                                     (dict(window=-1), "window=-1"), (dict(count=-1), "count -1"), (dict(dtype=5), "dtype"),
                                     (dict(tokens=2 ** 30), "tokens"), (dict(table_width=-1), "table_width=-1")])
def test_workspace_bytes_refuses_what_the_call_refuses(kw, word):
    need = ctypes.c_uint64(7)
    _refused(fg.lib().fg_select_blocks_workspace_bytes(_summary(), _selection(**kw), ctypes.byref(need)), word)
    assert need.value == 7


@pytest.mark.parametrize("width,need", [(4, 0), (256, 0), (257, 3 * 2 * 257 * 4), (10 ** 6, 3 * 2 * 10 ** 6 * 4)])
def test_workspace_bytes(width, need):
    got = ctypes.c_uint64(7)
    assert fg.lib().fg_select_blocks_workspace_bytes(_summary(), _selection(table_width=width), ctypes.byref(got)) == fg.FG_OK
    assert got.value == need


def test_empty_calls_and_null_structs():
    L = fg.lib()
    for kw in (dict(tokens=0), dict(requests=0), dict(count=0)):
        assert L.fg_select_blocks_device(_summary(), _selection(blocks=None, **kw), None) == fg.FG_OK
    assert _summarize(tokens=0) == fg.FG_OK and _summarize(requests=0, query_start=None) == fg.FG_OK
    assert _summarize(cache=_cache(v=None), tokens=0) == fg.FG_OK  # only the keys are read
    assert L.fg_select_blocks_device(None, _selection(), None) == fg.FG_ERR_ARG
    assert L.fg_select_blocks_device(_summary(), None, None) == fg.FG_ERR_ARG
    assert L.fg_kv_summarize_device(None, _summary(), PTR, 4, 4, PTR, PTR, 2, 3, None) == fg.FG_ERR_ARG
    assert L.fg_kv_summarize_device(_cache(), None, PTR, 4, 4, PTR, PTR, 2, 3, None) == fg.FG_ERR_ARG


def test_struct_sizes():
    assert ctypes.sizeof(_capi.KVSummaryArgs) == 64 and _capi.KVSummaryArgs.pages.offset == 48
    assert ctypes.sizeof(_capi.BlockSelectionArgs) == 128 and _capi.BlockSelectionArgs.tokens.offset == 96


def test_python_wrappers_refuse_host_tensors():
    import torch
    k = torch.zeros((2, 4, 1, 64), dtype=torch.float16)
    i = torch.zeros(1, dtype=torch.int32)
    bounds, scale = torch.zeros((2, 1, 2, 64), dtype=torch.int8), torch.zeros((2, 1))
    with pytest.raises(fg.FlashGANNError):
        fg.kv_summarize(k, bounds, scale, i.view(1, 1), i, i, tokens=1)
    with pytest.raises(fg.FlashGANNError):
        fg.select_blocks(k[0], bounds, scale, i.view(1, 1), i, i, 1, page_size=4, window=0)
