"""A paged key/value cache and attention over it, for decoders that find the
keys of a long context with this package's search.

The loop of one step: ``kv_plan`` gives each request pages and each new token
a slot, ``kv_append`` writes the new keys and values there, and then either
``paged_attention`` (all of the context, or a sliding window and the first
tokens) or ``retrieved_attention`` (window, first tokens and the ids that a
search returned for each query head) reads them.  All four take torch CUDA
tensors, run in libflashgann.so (include/flashgann.h has the exact rules) on
``stream`` (default: torch's current stream) and wait for nothing.
"""

from __future__ import annotations

import ctypes
import struct
from typing import NamedTuple, Optional

import torch

from . import _capi
from ._capi import FG_ERR_ARG, FG_OK, FlashGANNError, lib

_DTYPES = {torch.float16: _capi.FG_DTYPE_F16, torch.bfloat16: _capi.FG_DTYPE_BF16}

# A decode step makes these calls once for each layer, so the calls themselves are kept short: the two argument structs
# are packed into bytes (a ctypes.Structure takes several times as long to fill), their layout is _capi's.
_CACHE = struct.Struct("@PPqqqiiiii4x")
_ARGS = struct.Struct("@PqqPqqPPqPPPqqPQiiiiiiiif4x")
assert _CACHE.size == ctypes.sizeof(_capi.KVCacheArgs) and _ARGS.size == ctypes.sizeof(_capi.AttentionArgs)
_calls = {}


def _call(name: str, *argtypes):
    """The library's entry point `name`, taking packed structs as bytes."""
    f = _calls.get(name)
    if f is None:
        f = _calls[name] = ctypes.CFUNCTYPE(ctypes.c_int, *argtypes)((name, lib()))
    return f


class KVPlan(NamedTuple):
    """What kv_plan returns; R requests, T token rows."""
    query_start: torch.Tensor  # int32 [R + 1]: first row of each request in the step's token tensors
    kv_len: torch.Tensor       # int32 [R]: tokens after the step (0: refused)
    position: torch.Tensor     # int32 [T]: position in the request (-1: no token, or refused)
    slot: torch.Tensor         # int64 [T]: page * page_size + row, for kv_append (-1 likewise)
    free_head: torch.Tensor    # int32 [1]: first free page that was not taken
    refused: torch.Tensor      # int32 [R]: 1 where the pages did not suffice


def _fail(message: str):
    raise FlashGANNError(FG_ERR_ARG, message)


def _raise(rc: int, what: str):
    L = lib()
    raise FlashGANNError(rc, f"{what}: {L.fg_status_string(rc).decode()} ({L.fg_last_error().decode()})")


class _On:
    """The device and stream of one call.  Output and scratch tensors made
    inside belong to that stream; inputs that live on another one are marked
    as in use there, so that the caller may drop them right after the call."""

    __slots__ = ("index", "handle", "guard")

    def __init__(self, like: torch.Tensor, stream):
        if not like.is_cuda:
            _fail("expected a CUDA tensor")
        self.index = index = like.get_device()
        self.guard = None
        self.handle = torch._C._cuda_getCurrentRawStream(index)
        if stream is not None and getattr(stream, "cuda_stream", stream) != self.handle:
            self.handle = handle = getattr(stream, "cuda_stream", stream) or 0
            s = stream if isinstance(stream, torch.cuda.Stream) else (
                torch.cuda.ExternalStream(handle, device=index) if handle else torch.cuda.default_stream(index))
            self.guard = torch.cuda.stream(s)
        elif torch.cuda.current_device() != index:
            self.guard = torch.cuda.device(index)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return self

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)

    def uses(self, *tensors):
        index = self.index
        for t in tensors:
            if t is None:
                continue
            if t.get_device() != index:
                _fail(f"a tensor is on {t.device}, not on device {index}")
            if self.guard is not None:
                t.record_stream(torch.cuda.current_stream(index))


def _ints(t: torch.Tensor, dims: int, name: str, dtype=torch.int32) -> torch.Tensor:
    if t.dtype != dtype or t.dim() != dims:
        _fail(f"{name} must be {dtype} with {dims} dimension(s), not {t.dtype} {tuple(t.shape)}")
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _rows(t: torch.Tensor, name: str) -> torch.Tensor:
    """[tokens, heads, dim] with a contiguous last axis and 16-byte aligned rows (a copy where it is not)."""
    if t.dim() != 3:
        _fail(f"{name} must be [tokens, heads, dim], not {tuple(t.shape)}")
    s0, s1, s2 = t.stride()
    if (s2 != 1 and t.shape[2] > 1) or (s0 | s1) % 8 or t.data_ptr() % 16:
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _cache(k_cache: torch.Tensor, v_cache: torch.Tensor):
    """(fg_kv_cache as bytes, kv heads, dim)"""
    shape, s = k_cache.shape, k_cache.stride()
    if len(shape) != 4 or v_cache.shape != shape:
        _fail(f"caches must be [pages, page_size, heads, dim] alike, not {tuple(shape)} and {tuple(v_cache.shape)}")
    dtype = _DTYPES.get(k_cache.dtype)
    if dtype is None or v_cache.dtype != k_cache.dtype:
        _fail(f"caches must both be float16 or bfloat16, not {k_cache.dtype} and {v_cache.dtype}")
    if s != v_cache.stride() or s[3] != 1:
        _fail(f"caches must have the same strides and a contiguous last axis, not {s} and {v_cache.stride()}")
    pages, page_size, heads, dim = shape
    return _CACHE.pack(k_cache.data_ptr(), v_cache.data_ptr(), s[0], s[1], s[2], pages, page_size, heads, dim,
                       dtype), heads, dim


def kv_plan(ctx_len: torch.Tensor, new_len: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor, *,
            tokens: int, page_size: int, free_head: Optional[torch.Tensor] = None, stream=None) -> KVPlan:
    """Pages, slots and row offsets of one step, from lengths on the device
    (fg_kv_plan_device).

    ctx_len, new_len int32 [R]: tokens in the cache and new ones of each
    request; block_table int32 [R, width], updated in place; free_pages int32
    [F], used from ``free_head`` (int32 [1], default 0) on; tokens: rows of the
    step's token tensors (at least the sum of new_len for all to be mapped)."""
    with _On(ctx_len, stream) as on:
        on.uses(ctx_len, new_len, block_table, free_pages, free_head)
        ctx_len, new_len = _ints(ctx_len, 1, "ctx_len"), _ints(new_len, 1, "new_len")
        free_pages = _ints(free_pages, 1, "free_pages")
        if new_len.shape != ctx_len.shape:
            _fail("ctx_len and new_len differ in length")
        R = ctx_len.shape[0]
        if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != R or (
                block_table.shape[1] > 1 and block_table.stride(1) != 1):
            _fail(f"block_table must be int32 [{R}, width] with contiguous rows")
        if free_head is not None and (free_head.dtype != torch.int32 or free_head.numel() != 1):
            _fail("free_head must be int32 [1]")
        T = max(tokens, 0)
        slot = torch.empty(T, dtype=torch.int64, device=ctx_len.device)
        ints = ctx_len.new_empty(3 * R + 2 + T)
        base = ints.data_ptr()
        query_start, kv_len, head, refused, position = ints.split_with_sizes((R + 1, R, 1, R, T))
        rc = lib().fg_kv_plan_device(ctx_len.data_ptr(), new_len.data_ptr(), R, free_pages.data_ptr(),
                                     free_pages.shape[0], None if free_head is None else free_head.data_ptr(),
                                     page_size, block_table.data_ptr(), block_table.shape[1], block_table.stride(0),
                                     tokens, base, base + 4 * (R + 1), base + 4 * (3 * R + 2), slot.data_ptr(),
                                     base + 4 * (2 * R + 1), base + 4 * (2 * R + 2), on.handle)
        if rc != FG_OK:
            _raise(rc, "fg_kv_plan_device")
        return KVPlan(query_start, kv_len, position, slot, head, refused)


def kv_append(k_cache: torch.Tensor, v_cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slot: torch.Tensor, *,
              stream=None) -> None:
    """Writes rows k, v [T, heads, dim] to the slots (int64 [T], from kv_plan)
    of the caches [pages, page_size, heads, dim]; negative slots are skipped
    (fg_kv_append_device)."""
    with _On(k_cache, stream) as on:
        on.uses(k_cache, v_cache, k, v, slot)
        c, heads, dim = _cache(k_cache, v_cache)
        want = (slot.shape[0], heads, dim)
        if k.shape != want or v.shape != want or k.dtype != k_cache.dtype or v.dtype != k_cache.dtype:
            _fail(f"k and v must be {k_cache.dtype} {want}, not {k.dtype} {tuple(k.shape)} and {v.dtype} "
                  f"{tuple(v.shape)}")
        slot, k, v = _ints(slot, 1, "slot", torch.int64), _rows(k, "k"), _rows(v, "v")
        k0, k1, _ = k.stride()
        v0, v1, _ = v.stride()
        i64, ptr = ctypes.c_int64, ctypes.c_void_p
        rc = _call("fg_kv_append_device", ctypes.c_char_p, ptr, i64, i64, ptr, i64, i64, ptr, ctypes.c_int32, ptr)(
            c, k.data_ptr(), k0, k1, v.data_ptr(), v0, v1, slot.data_ptr(), want[0], on.handle)
        if rc != FG_OK:
            _raise(rc, "fg_kv_append_device")


_workspace = {}  # bytes that a call needs, by what they depend on


def _attend(retrieved: bool, q, k_cache, v_cache, block_table, query_start, kv_len, max_new, ids, window, sinks, scale, out,
            return_lse, stream):
    with _On(q, stream) as on:
        on.uses(q, k_cache, v_cache, block_table, query_start, kv_len, out, ids)
        c, kv_heads, cache_dim = _cache(k_cache, v_cache)
        q = _rows(q, "q")
        T, heads, dim = q.shape
        if q.dtype != k_cache.dtype or dim != cache_dim:
            _fail(f"q must be {k_cache.dtype} [tokens, heads, {cache_dim}], not {q.dtype} {tuple(q.shape)}")
        block_table = _ints(block_table, 2, "block_table")
        query_start, kv_len = _ints(query_start, 1, "query_start"), _ints(kv_len, 1, "kv_len")
        R = kv_len.shape[0]
        if query_start.shape[0] != R + 1 or block_table.shape[0] != R:
            _fail(f"{R} lengths need {R + 1} query_start entries and {R} table rows, not {query_start.shape[0]} and "
                  f"{block_table.shape[0]}")
        if out is None:
            out = torch.empty_like(q) if q.is_contiguous() else torch.empty((T, heads, dim), dtype=q.dtype, device=q.device)
        elif out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1:
            _fail(f"out must be {q.dtype} {tuple(q.shape)} with a contiguous last axis")
        lse = torch.empty((T, heads), dtype=torch.float32, device=q.device) if return_lse else None
        id_ptr = id_token = id_head = count = 0
        if ids is not None:
            if ids.dtype != torch.int32 or ids.dim() != 3 or ids.shape[:2] != q.shape[:2]:
                _fail(f"ids must be int32 [{T}, {heads}, count], not {ids.dtype} {tuple(ids.shape)}")
            if ids.stride(2) != 1 and ids.shape[2] > 1:
                ids = ids.contiguous()
            id_ptr, count = ids.data_ptr(), ids.shape[2]
            id_token, id_head, _ = ids.stride()
        q0, q1, _ = q.stride()
        o0, o1, _ = out.stride()
        args = [q.data_ptr(), q0, q1, out.data_ptr(), o0, o1, lse.data_ptr() if return_lse else 0,
                block_table.data_ptr(), block_table.stride(0), query_start.data_ptr(), kv_len.data_ptr(), id_ptr,
                id_token, id_head, 0, 0, T, heads, R, block_table.shape[1], max_new, -1 if window is None else window,
                sinks, count, dim ** -0.5 if scale is None else scale]
        key = (on.index, retrieved, c[16:], q0 == 0, q1 == 0, T, heads, R, max_new, block_table.shape[1], window, sinks, count, args[-1] > 0)
        need = _workspace.get(key)
        if need is None:
            size = ctypes.c_uint64()
            rc = _call("fg_attention_workspace_bytes", ctypes.c_char_p, ctypes.c_char_p, ctypes.c_int32,
                       ctypes.c_void_p)(c, _ARGS.pack(*args), retrieved, ctypes.addressof(size))
            if rc != FG_OK:
                _raise(rc, "fg_attention_workspace_bytes")
            if len(_workspace) > 1000:  # table widths that never come back
                _workspace.clear()
            need = _workspace[key] = size.value
        if need:
            work = torch.empty(need, dtype=torch.uint8, device=q.device)
            args[14], args[15] = work.data_ptr(), need
        call = "fg_retrieved_attention_device" if retrieved else "fg_paged_attention_device"
        rc = _call(call, ctypes.c_char_p, ctypes.c_char_p, ctypes.c_void_p)(c, _ARGS.pack(*args), on.handle)
        if rc != FG_OK:
            _raise(rc, call)
        return (out, lse) if return_lse else out


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    query_start: torch.Tensor, kv_len: torch.Tensor, max_new: int, *, window: Optional[int] = None,
                    sinks: int = 0, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                    return_lse: bool = False, stream=None):
    """Causal attention of each request's new tokens over its cache
    (fg_paged_attention_device).

    q [T, heads, dim] (a request's rows are query_start[b] .. query_start[b+1],
    its last ones the newest positions of kv_len[b]); caches [pages, page_size,
    kv_heads, dim], any strides; heads a multiple of kv_heads.  max_new: most
    new tokens of a request (picks the kernel).  window: how many newest keys
    a token sees, itself included (None or -1: all); sinks: first tokens that
    stay visible.  scale: default dim ** -0.5.  Returns out [T, heads, dim],
    with return_lse also the rows' log-sum-exp float32 [T, heads]; a row that
    sees nothing is 0 and -inf."""
    return _attend(False, q, k_cache, v_cache, block_table, query_start, kv_len, max_new, None, window, sinks, scale,
                   out, return_lse, stream)


def retrieved_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                        query_start: torch.Tensor, kv_len: torch.Tensor, ids: torch.Tensor, *, window: int,
                        sinks: int = 0, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                        return_lse: bool = False, stream=None):
    """paged_attention over the window, the first tokens and retrieved keys
    (fg_retrieved_attention_device): ids int32 [T, heads, count] are positions
    of the request's context, in any order, as a search over its keys returns
    them (uint32 ids as int32 bits; negative, repeated, already visible and
    future ones count nothing)."""
    return _attend(True, q, k_cache, v_cache, block_table, query_start, kv_len, 1, ids, window, sinks, scale, out,
                   return_lse, stream)
