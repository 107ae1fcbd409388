"""Decoding over a long context whose keys are searched, not scanned.

One request of a decoder with grouped heads has a long prompt in the paged cache.  The keys of each kv head are also
the base of a graph index (inner-product metric; graph, 1-bit codes and layout from ``flashgann_b200.builder``).  Each
step plans slots for the new token, appends its key and value, searches every query head's vector in its head's index,
and attends over the first tokens, a sliding window and the retrieved positions.  The step's exact counterpart,
attention over the whole context, is computed beside it and compared.

    python examples/retrieval_decode.py [--context 20000] [--steps 4]

Keys are drawn from a mixture, and each query from the neighbourhood of one of its components: attention that
concentrates on the 60 keys or so of that component, which is the case that retrieval is for.
"""

from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import flashgann_b200 as fg  # noqa: E402
from flashgann_b200 import builder  # noqa: E402


def key_index(keys: torch.Tensor, degree: int, seed: int) -> fg.QuantizationGraph:
    """A graph index over keys float32 [n, dim] on the GPU, searched by inner product (L2 neighbours make the graph:
    the keys have much the same length)."""
    dim = keys.shape[1]
    x = keys.cpu().numpy()
    nbrs, entry = builder.build_graph(x, degree, seed, device="cuda")
    signs = builder.make_signs(builder.padded_dim(dim), seed)
    rows = builder.encode_rows_device(keys, torch.from_numpy(nbrs).to(keys.device, torch.int32), signs, metric="ip")
    return fg.QuantizationGraph.from_device(rows, torch.from_numpy(signs).to(keys.device), entry, dim, degree,
                                            metric=fg.METRIC_IP)


def run(context: int = 20000, steps: int = 4, heads: int = 8, kv_heads: int = 2, dim: int = 128, top: int = 100,
        beam: int = 256, window: int = 128, sinks: int = 4, page_size: int = 16, seed: int = 0) -> dict:
    """Decodes ``steps`` tokens; returns the share of the exact attention's weight that the retrieved form saw, the
    relative difference of their outputs (means over steps and heads), and the last step's query, ids and output with
    the cache, for who wants to check them."""
    dev, dt = torch.device("cuda"), torch.bfloat16
    group = heads // kv_heads
    gen = torch.Generator(device=dev).manual_seed(seed)
    spots = max(4, context // 60)
    centre = torch.randn(kv_heads, spots, dim, generator=gen, device=dev)
    centre = centre / centre.norm(dim=-1, keepdim=True) * dim ** 0.5

    def draw(n):
        c = torch.randint(spots, (n,), generator=gen, device=dev)
        return (centre[:, c].transpose(0, 1) + 0.35 * torch.randn(n, kv_heads, dim, generator=gen, device=dev)).to(dt)

    pages = -(-(context + steps) // page_size) + 8
    k_cache = torch.zeros(pages, page_size, kv_heads, dim, dtype=dt, device=dev)
    v_cache = torch.zeros_like(k_cache)
    table = torch.full((1, pages), -1, dtype=torch.int32, device=dev)
    free = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    length, free_head = torch.zeros(1, dtype=torch.int32, device=dev), None

    def append(k, v):
        """The new tokens' pages and slots, and their rows in the cache."""
        nonlocal length, free_head
        new = torch.full((1,), k.shape[0], dtype=torch.int32, device=dev)
        plan = fg.kv_plan(length, new, table, free, tokens=k.shape[0], page_size=page_size, free_head=free_head)
        fg.kv_append(k_cache, v_cache, k, v, plan.slot)
        length, free_head = plan.kv_len, plan.free_head
        return plan

    prompt = draw(context)
    append(prompt, torch.randn(context, kv_heads, dim, generator=gen, device=dev).to(dt))
    index = [key_index(prompt[:, h].float().contiguous(), 32, seed + h) for h in range(kv_heads)]

    seen, error = [], []
    for _ in range(steps):
        plan = append(draw(1), torch.randn(1, kv_heads, dim, generator=gen, device=dev).to(dt))
        at = torch.randint(spots, (group,), generator=gen, device=dev)
        q = centre[:, at] + 0.35 * torch.randn(kv_heads, group, dim, generator=gen, device=dev)
        q = q.reshape(1, heads, dim).to(dt)
        # one search for each kv head: its group's queries, ids [group, top] as the search leaves them
        ids = torch.empty(1, heads, top, dtype=torch.int32, device=dev)
        wanted = q.float().reshape(kv_heads, group, dim)
        stream = torch.cuda.current_stream()
        for h in range(kv_heads):
            index[h].search_device(wanted[h], top, beam, d_out=ids[0, h * group:(h + 1) * group], stream=stream)
        args = (q, k_cache, v_cache, table, plan.query_start, plan.kv_len)
        out, lse = fg.retrieved_attention(*args, ids, window=window, sinks=sinks, return_lse=True)
        exact, full = fg.paged_attention(*args, 1, return_lse=True)
        seen.append(torch.exp(lse - full).mean())
        error.append((out.float() - exact.float()).norm() / exact.float().norm())
    result = {"weight_seen": float(torch.stack(seen).mean()), "error": float(torch.stack(error).mean()),
              "refused": int(plan.refused.sum()), "tokens": int(plan.kv_len[0]),
              "last": dict(q=q, ids=ids, out=out, lse=lse, k_cache=k_cache, v_cache=v_cache, table=table,
                           window=window, sinks=sinks)}
    for i in index:
        i.close()
    return result


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--context", type=int, default=20000)
    ap.add_argument("--steps", type=int, default=4)
    a = ap.parse_args()
    r = run(a.context, a.steps)
    print("%d tokens: the retrieved keys, window and first tokens hold %.2f %% of the attention's weight; outputs differ "
          "by %.2f %%" % (r["tokens"], 100 * r["weight_seen"], 100 * r["error"]))


if __name__ == "__main__":
    main()
