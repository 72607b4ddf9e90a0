"""Serving many requests at once from a paged key/value cache.

A cache is two tensors (n_pages, n_kv_heads, page_size, head_dim), fp16 or bf16; a request's row of the page table names
the pages that hold its tokens in order.  One step of a server, for any mix of requests that get one token and requests
that get a chunk of their prompt:

    plan = plan_pages(cached, new, tables, free_pages, n_free, page_size, rows)    # pages and slots for the new tokens
    q, k, v = ...                                                                  # packed rows: (rows, heads * head_dim)
    q = rope_append_paged(q, k, v, k_cache, v_cache, plan.positions, plan.slots, inv_freq)
    att = paged_attention(q, k_cache, v_cache, tables, plan.kv_lens, plan.cu_rows, max_rows)

and `prompt_attention` where all keys are in the call itself.  Lengths and tables stay on the device: nothing here waits
for the GPU, and a captured step can be replayed for other lengths.  As everywhere in this package there is no fallback
(a CPU tensor raises), launches go to the current stream, and no gradient is formed (a tensor that wants one raises).

Every wait inside the attention kernels is bounded (2 s).  One that runs out cannot raise, because no call waits for the GPU: it
leaves a code in the status word of the stream's scratch, and the outputs are not valid.  `kernels.workspace_status_all(device)`
reads and clears the words of all streams; a server asks for it where it waits for a step's tokens anyway.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .. import _lib

__all__ = ["PagePlan", "plan_pages", "rope_append_paged", "paged_attention", "prompt_attention"]


class PagePlan(NamedTuple):
    """What `plan_pages` returns, all on the device: for B requests and `rows` rows of packed new tokens.  The five are parts of
    one allocation, which lives as long as any of them."""
    cu_rows: torch.Tensor       # int32 (B + 1): rows cu_rows[b] .. cu_rows[b+1]-1 belong to request b
    kv_lens: torch.Tensor       # int32 (B): keys of the request with its new tokens, 0 where it was not served
    positions: torch.Tensor     # int64 (rows): a row's place in its request
    slots: torch.Tensor         # int64 (rows): page * page_size + place in the page, -1 where there is none
    n_free: torch.Tensor        # int32 (1): free pages left


def plan_pages(cached: torch.Tensor, new: torch.Tensor, tables: torch.Tensor, free_pages: torch.Tensor,
               n_free: torch.Tensor, page_size: int, rows: int) -> PagePlan:
    """Pages, slots and row ranges for the new tokens of B requests, from their lengths, in one launch.

    `cached`, `new` int32 (B): tokens in the cache and tokens of this step (0 is fine).  `tables` int32 (B, width): page
    ids; those for the `cached` tokens are there, those for the new ones are written.  `free_pages` int32: ids of free
    pages, of which the first `n_free` (int32, one value) count; pages are taken from their end, in the order of the
    requests.  `n_free` itself stays: the count that is left is in the result, and a server that keeps its state in one
    place copies it there.  Pages go back by writing them behind what is left.  `rows`: rows of the packed step, at
    least the sum of `new`; rows behind the last request get position 0 and slot -1.

    A request is not served (kv_lens 0, slots -1, no pages) if its tokens need more than `width` pages, if its rows end
    behind `rows`, or if the free pages do not last up to it; one that needs no page is served all the same."""
    return PagePlan(*_lib.host().plan_pages(cached, new, tables, free_pages, n_free, page_size, rows))


def rope_append_paged(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      positions: torch.Tensor, slots: torch.Tensor, inv_freq: torch.Tensor, scaling: float = 1.0,
                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary embedding of packed q and k (rows, heads * head_dim) and the store of k and v at `slots` of the caches;
    returns the rotated q (`out`, which may be q itself but overlaps nothing else, or a new tensor).  Pairs
    (i, i + head_dim / 2), angle positions[r] * inv_freq[i] formed in 64 bits, cos and sin kept in 32.  q, k and v may be
    column ranges of one projection's output.  A slot outside the cache (-1: a row without one) is not written; slots
    differ otherwise, or the slot holds a mixture."""
    return _lib.host().rope_append_paged(q, k, v, k_cache, v_cache, positions, slots, inv_freq, scaling, out)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, tables: torch.Tensor,
                    kv_lens: torch.Tensor, cu_rows: torch.Tensor, max_rows: int, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of every request's new rows over its pages: request b owns the rows cu_rows[b] .. cu_rows[b+1]-1
    of q (rows, n_heads * head_dim), they are the last of its kv_lens[b] keys, and row t of n sees the keys
    0 .. kv_lens[b] - n + t.  One row per request while tokens are generated, many for a chunk of a prompt, both in one
    call.  `max_rows`: the most rows that one request has; it chooses the kernel and changes no result but its rounding.
    Scores, maxima and sums are held in 32 bits.  Weights meet the values as two 16-bit numbers in the kernel for few rows
    (`max_rows` tokens of one key/value head in 16 rows, or twice that with heads of 64), rounded to the inputs' type in
    the one for many.  Rows that see no key come out as zeros, rows of no request as they were in `out` (q itself, or
    memory of its own), and as zeros without one.  A page id outside the cache stands for keys that are not there;
    kv_lens[b] counts as what the table's width holds at most."""
    return _lib.host().paged_attention(q, k_cache, v_cache, tables, kv_lens, cu_rows, max_rows, scale, out)


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_rows: torch.Tensor, head_dim: int,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention inside each of many prompts packed into one call: q (rows, n_heads * head_dim), k and v
    (rows, n_kv_heads * head_dim), prompt b in the rows cu_rows[b] .. cu_rows[b+1]-1.  q, k and v may be column ranges of
    one projection's output.  Rows of no prompt stay as they were in `out` (q itself, or memory of its own), and are
    zeros without one.  Weights are rounded to the inputs' type before they meet the values; all else is held in 32 bits."""
    return _lib.host().prompt_attention(q, k, v, cu_rows, head_dim, scale, out)
