"""What the cache and attention entry points refuse at the ends of their ranges: checked before any device work, so
no GPU is needed."""

from __future__ import annotations

import ctypes

import pytest

import flashgann_b200 as fg
from tests.test_attention_args import ARGS, IDS, PTR, _args, _cache

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


# ---- rows that are written must not overlap ----

# tokens 3, heads 4, dim 64: (token stride, head stride)
@pytest.mark.parametrize("strides,fine", [
    ((256, 64), True), ((64, 192), True), ((64, 64), False), ((248, 64), False), ((64, 184), False), ((64, 128), False),
    ((1024, 72), True), ((72, 1024), True), ((128, 256), False), ((0, 64), False), ((1 << 62, 1 << 62), False)])
def test_outputs_whose_axes_do_not_nest_are_refused(strides, fine):
    L = fg.lib()
    for call in ("fg_paged_attention_device", "fg_retrieved_attention_device"):
        # a layout that is fine goes on to the next refusal
        rc = getattr(L, call)(_cache(), _args(out_token_stride=strides[0], out_head_stride=strides[1], kv_len=None), None)
        assert rc == fg.FG_ERR_ARG
        assert ("null buffer" if fine else "rows of out overlap") in L.fg_last_error().decode()


@pytest.mark.parametrize("tokens,heads,strides,fine", [(1, 4, (0, 64), True), (3, 1, (64, 0), True), (1, 4, (64, 64), True)])
def test_axes_of_one_entry_have_any_stride(tokens, heads, strides, fine):
    L = fg.lib()
    cache = _cache(heads=1, token_stride=64, page_stride=1024)
    assert L.fg_paged_attention_device(cache, _args(tokens=tokens, heads=heads, out_token_stride=strides[0],
                                                    out_head_stride=strides[1], kv_len=None), None) == fg.FG_ERR_ARG
    assert "null buffer" in L.fg_last_error().decode()


# pages 4, page size 16, heads 2, dim 64: (page, token, head)
@pytest.mark.parametrize("strides", [(64, 64, 64), (2048, 128, 128), (2048, 64, 512), (1024, 128, 64), (2040, 128, 64),
                                     (64, 128, 2048), (4096, 256, 256), (64, 512, 128)])
def test_append_to_caches_whose_axes_do_not_nest_is_refused(strides):
    L = fg.lib()
    cache = _cache(page_stride=strides[0], token_stride=strides[1], head_stride=strides[2])
    assert L.fg_kv_append_device(cache, PTR, 128, 64, PTR, 128, 64, PTR, 3, None) == fg.FG_ERR_ARG
    assert "rows of the cache overlap" in L.fg_last_error().decode()


@pytest.mark.parametrize("strides", [(2048, 128, 64), (2048, 64, 1024), (64, 512, 256), (8192, 128, 64), (128, 512, 8192)])
def test_append_takes_caches_in_any_order_of_axes(strides):
    L = fg.lib()
    cache = _cache(page_stride=strides[0], token_stride=strides[1], head_stride=strides[2])
    assert L.fg_kv_append_device(cache, PTR, 128, 64, PTR, 128, 64, None, 3, None) == fg.FG_ERR_ARG
    assert "null slots" in L.fg_last_error().decode()


@pytest.mark.parametrize("requests,stride,fine", [(2, 0, False), (2, 3, False), (2, 4, True), (1, 0, True), (5, 1, False)])
def test_plan_refuses_overlapping_table_rows(requests, stride, fine):
    L = fg.lib()
    rc = L.fg_kv_plan_device(PTR, PTR, requests, PTR, 5, PTR, 16, PTR, 4, stride, 3, PTR, PTR, PTR, PTR, PTR, PTR, None)
    assert rc == fg.FG_ERR_ARG  # free_head and free_head_out are the same buffer: the next refusal
    assert ("same buffer" if fine else "rows of the block table overlap") in L.fg_last_error().decode()


@pytest.mark.parametrize("scale,fine", [(2.3e38, True), (-2.3e38, True), (2.4e38, False), (-3.4e38, False)])
def test_scales_that_overflow_with_log2e_are_refused(scale, fine):
    L = fg.lib()
    assert L.fg_paged_attention_device(_cache(), _args(scale=scale, kv_len=None), None) == fg.FG_ERR_ARG
    assert ("null buffer" if fine else "scale") in L.fg_last_error().decode()


@pytest.mark.parametrize("cache,args", [
    (dict(pages=1, page_stride=-3), dict()), (dict(heads=1, head_stride=5, token_stride=64), dict()),
    (dict(page_size=1, token_stride=-9), dict()),
    (dict(), dict(tokens=1, q_token_stride=-1, out_token_stride=3)),
    (dict(heads=1), dict(heads=1, q_head_stride=7, out_head_stride=-7))])
def test_strides_of_axes_of_one_entry_are_not_looked_at(cache, args):
    L = fg.lib()
    for call in ("fg_paged_attention_device", "fg_retrieved_attention_device"):
        assert getattr(L, call)(_cache(**cache), _args(kv_len=None, **args), None) == fg.FG_ERR_ARG
        assert "null buffer" in L.fg_last_error().decode()
    rows = (PTR, 1, 64, PTR, 3, 64, None, 1) if not cache.get("heads") else (PTR, 8, 3, PTR, 8, -1, None, 3)
    assert L.fg_kv_append_device(_cache(**cache), *rows, None) == fg.FG_ERR_ARG
    assert "null slots" in L.fg_last_error().decode()
