"""A paged key/value cache and attention over it, for decoders that find the
keys of a long context with this package's search.

The loop of one step: ``kv_plan`` gives each request pages and each new token
a slot, ``kv_append`` writes the new keys and values there, and then either
``paged_attention`` (all of the context, or a sliding window and the first
tokens) or ``retrieved_attention`` (window, first tokens and the ids that a
search returned for each query head) reads them.  All four take torch CUDA
tensors, run in libflashgann.so (include/flashgann.h has the exact rules) on
``stream`` (default: torch's current stream) and wait for nothing.  They are
for serving and have no backward pass: where torch records gradients, a tensor
that requires one is refused (call them under ``torch.no_grad()``).
"""

from __future__ import annotations

import os
from typing import NamedTuple, Optional

import torch

from . import _capi

_capi.lib()  # the library that the binding calls; says how to build both where they are missing
try:
    from . import _torch_ops
except ImportError as e:
    raise ImportError(f"{os.path.join(os.path.dirname(_capi.LIB_PATH), '_torch_ops.so')} is missing or does not load: "
                      f"build it with `make lib` (or __graft_entry__.build()): {e}") from e


class KVPlan(NamedTuple):
    """What kv_plan returns; R requests, T token rows."""
    query_start: torch.Tensor  # int32 [R + 1]: first row of each request in the step's token tensors
    kv_len: torch.Tensor       # int32 [R]: tokens after the step (0: refused)
    position: torch.Tensor     # int32 [T]: position in the request (-1: no token, or refused)
    slot: torch.Tensor         # int64 [T]: page * page_size + row, for kv_append (-1 likewise)
    free_head: torch.Tensor    # int32 [1]: first free page that was not taken
    refused: torch.Tensor      # int32 [R]: 1 where the pages did not suffice


def _handle(stream) -> int:
    return -1 if stream is None else getattr(stream, "cuda_stream", stream) or 0


def kv_plan(ctx_len: torch.Tensor, new_len: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor, *,
            tokens: int, page_size: int, free_head: Optional[torch.Tensor] = None, stream=None) -> KVPlan:
    """Pages, slots and row offsets of one step, from lengths on the device
    (fg_kv_plan_device).

    ctx_len, new_len int32 [R]: tokens in the cache and new ones of each
    request; block_table int32 [R, width], updated in place; free_pages int32
    [F], used from ``free_head`` (int32 [1], default 0) on; tokens: rows of the
    step's token tensors (at least the sum of new_len for all to be mapped)."""
    return KVPlan(*_torch_ops.kv_plan(ctx_len, new_len, block_table, free_pages, tokens, page_size, free_head,
                                      _handle(stream)))


def kv_append(k_cache: torch.Tensor, v_cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slot: torch.Tensor, *,
              stream=None) -> None:
    """Writes rows k, v [T, heads, dim] to the slots (int64 [T], from kv_plan)
    of the caches [pages, page_size, heads, dim]; negative slots are skipped
    (fg_kv_append_device)."""
    _torch_ops.kv_append(k_cache, v_cache, k, v, slot, _handle(stream))


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
    sees nothing is 0 and -inf.  Sums are 32 bits, the weights of the product
    with V are rounded to the cache's type."""
    out, lse = _torch_ops.attention(q, k_cache, v_cache, block_table, query_start, kv_len, max_new, None,
                                    -1 if window is None else window, sinks, scale, out, return_lse, _handle(stream))
    return (out, lse) if return_lse else out


def retrieved_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                        query_start: torch.Tensor, kv_len: torch.Tensor, ids: torch.Tensor, *, window: int,
                        sinks: int = 0, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                        return_lse: bool = False, stream=None):
    """paged_attention over the window, the first tokens and retrieved keys
    (fg_retrieved_attention_device): ids int32 [T, heads, count] are positions
    of the request's context, in any order, as a search over its keys returns
    them (uint32 ids as int32 bits; negative, repeated, already visible and
    future ones count nothing)."""
    out, lse = _torch_ops.attention(q, k_cache, v_cache, block_table, query_start, kv_len, 1, ids, window, sinks, scale,
                                    out, return_lse, _handle(stream))
    return (out, lse) if return_lse else out
