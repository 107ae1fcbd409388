"""A paged key/value cache and attention over it, for decoders that find the
keys of a long context with this package's search, or that bound what they read
of it without one.

The loop of one step: ``kv_plan`` gives each request pages and each new token
a slot, ``kv_append`` writes the new keys and values there, and then either
``paged_attention`` (all of the context, or a sliding window and the first
tokens), ``retrieved_attention`` (window, first tokens and the ids that a
search returned for each query head) or ``block_attention`` (window, first
tokens and whole pages) reads them.  For the last, ``kv_summarize`` keeps bounds
of each page's keys and ``select_blocks`` chooses the pages of the highest
bounds.  To keep the cache short instead, ``attention_weights`` sums up what
each key was paid and ``kv_evict`` drops the lightest.  All take torch CUDA
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


class KVEviction(NamedTuple):
    """What kv_evict returns; R requests."""
    kv_len: torch.Tensor  # int32 [R]: tokens that stayed
    kept: torch.Tensor    # int32 [R, kv_heads, budget]: where each was before, ascending (-1 past the length)


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
                                    False, -1 if window is None else window, sinks, scale, out, return_lse, _handle(stream))
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
    out, lse = _torch_ops.attention(q, k_cache, v_cache, block_table, query_start, kv_len, 1, ids, False, window, sinks,
                                    scale, out, return_lse, _handle(stream))
    return (out, lse) if return_lse else out


def kv_summarize(k_cache: torch.Tensor, bounds: torch.Tensor, scale: torch.Tensor, block_table: torch.Tensor,
                 query_start: torch.Tensor, kv_len: torch.Tensor, *, tokens: int, stream=None) -> None:
    """Summaries of the pages that hold the step's new tokens, for
    ``select_blocks`` (fg_kv_summarize_device); after ``kv_append``.

    bounds int8 [pages, kv_heads, 2, dim], scale float32 [pages, kv_heads]:
    least and largest value of each element over a page's keys, in whole
    multiples of scale; made once beside the caches and updated in place.
    query_start, kv_len: as from ``kv_plan`` (new pages only; a query_start of
    the running sums of kv_len gives all pages, as after ``kv_evict``); tokens:
    at least query_start's last entry."""
    _torch_ops.kv_summarize(k_cache, bounds, scale, block_table, query_start, kv_len, tokens, _handle(stream))


def select_blocks(q: torch.Tensor, bounds: torch.Tensor, scale: torch.Tensor, block_table: torch.Tensor,
                  query_start: torch.Tensor, kv_len: torch.Tensor, count: int, *, page_size: int, window: int,
                  sinks: int = 0, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """For each new token and kv head the ``count`` pages (numbers of blocks of
    page_size positions) whose bound on the token's scores is highest, among
    those that end past the first tokens and begin before the window: int32 [T,
    kv_heads, count], ascending, then -1 (fg_select_blocks_device).

    q [T, heads, dim]; bounds and scale from ``kv_summarize``.  The heads of a
    group choose together, by the largest of their bounds.  Queries are rounded
    to 8 bits for it, so that a bound holds but for that rounding.  A row that is
    -2 throughout says that the kernel gave up a wait."""
    return _torch_ops.select_blocks(q, bounds, scale, block_table, query_start, kv_len, count, page_size, window, sinks,
                                    out, _handle(stream))


def block_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    query_start: torch.Tensor, kv_len: torch.Tensor, blocks: torch.Tensor, *, window: int,
                    sinks: int = 0, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                    return_lse: bool = False, stream=None):
    """paged_attention over the window, the first tokens and chosen blocks
    (fg_block_attention_device): blocks int32 [T, kv_heads, count], as
    ``select_blocks`` returns them or any others (block x: positions x *
    page_size to (x + 1) * page_size - 1; negative, repeated and future ones
    and positions that are visible already count nothing).  Sums are 32 bits,
    the weights of the product with V are rounded to the cache's type."""
    out, lse = _torch_ops.attention(q, k_cache, v_cache, block_table, query_start, kv_len, 1, blocks, True, window,
                                    sinks, scale, out, return_lse, _handle(stream))
    return (out, lse) if return_lse else out


def attention_weights(q: torch.Tensor, k_cache: torch.Tensor, weights: torch.Tensor, block_table: torch.Tensor,
                      query_start: torch.Tensor, kv_len: torch.Tensor, lse: torch.Tensor, *,
                      window: Optional[int] = None, sinks: int = 0, scale: Optional[float] = None,
                      held: Optional[torch.Tensor] = None, stream=None) -> None:
    """Adds to weights float32 [pages, kv_heads, page_size] the attention that
    the step's rows paid to each key of their requests
    (fg_attention_weights_device); after ``paged_attention(...,
    return_lse=True)`` with the same arguments, whose lse float32 [T, heads]
    this takes.

    Weights of positions from held[b] on (int32 [R]; default: of the new tokens)
    start at 0.  For a prompt the last tokens may do: their rows of q and lse,
    a query_start that counts them alone, and held of 0."""
    _torch_ops.attention_weights(q, k_cache, weights, block_table, query_start, kv_len, lse, held,
                                 -1 if window is None else window, sinks, scale, _handle(stream))


def kv_evict(k_cache: torch.Tensor, v_cache: torch.Tensor, weights: torch.Tensor, block_table: torch.Tensor,
             kv_len: torch.Tensor, budget: int, *, recent: int = 0, sinks: int = 0, stream=None) -> KVEviction:
    """Cuts requests of more than ``budget`` tokens down to it, in place
    (fg_kv_evict_device): each kv head keeps the first ``sinks`` tokens, the
    last ``recent`` and the heaviest of those between, by weights float32
    [pages, kv_heads, page_size] from ``attention_weights``; keys, values and
    weights of those move to the first positions, in order.  A length past what
    the table holds counts as that.

    Table entries from ceil(budget / page_size) on of such requests are free
    afterwards; kv_len of the result is the next step's ctx_len.  Page
    summaries are made anew with ``kv_summarize`` over all pages."""
    return KVEviction(*_torch_ops.kv_evict(k_cache, v_cache, weights, block_table, kv_len, budget, recent, sinks,
                                           _handle(stream)))
