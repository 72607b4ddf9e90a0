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
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from .. import _lib
from . import workspace_for

__all__ = ["PagePlan", "plan_pages", "rope_append_paged", "paged_attention", "prompt_attention"]

_STATUS_WORD = 4092          # byte of the scratch buffers' status word: the last counter
_DTYPES = {torch.float16: _lib.EPTQ_FP16, torch.bfloat16: _lib.EPTQ_BF16}


class PagePlan(NamedTuple):
    """What `plan_pages` returns, all on the device: for B requests and `rows` rows of packed new tokens."""
    cu_rows: torch.Tensor       # int32 (B + 1): rows cu_rows[b] .. cu_rows[b+1]-1 belong to request b
    kv_lens: torch.Tensor       # int32 (B): keys of the request with its new tokens, 0 where it was not served
    positions: torch.Tensor     # int64 (rows): a row's place in its request
    slots: torch.Tensor         # int64 (rows): page * page_size + place in the page, -1 where there is none
    n_free: torch.Tensor        # int32 (1): free pages left


def _fail(what: str):
    raise RuntimeError(f"eptq_b200: {what}")


def _on_gpu(device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if not t.is_cuda:
            _fail(f"`{name}` must be a CUDA tensor (there is no CPU path)")
        if t.device != device:
            _fail(f"`{name}` is on {t.device}, not on {device}")
        if t.requires_grad and torch.is_grad_enabled():
            _fail(f"`{name}` wants a gradient, and the paged operators form none")


def _whole(dtype: torch.dtype, numel: Optional[int] = None, **tensors) -> None:
    for name, t in tensors.items():
        if t.dtype != dtype or not t.is_contiguous() or (numel is not None and t.numel() != numel):
            _fail(f"`{name}` must be a contiguous {dtype} tensor" + ("" if numel is None else f" of {numel} values"))


def _packed(dtype: torch.dtype, rows: int, **tensors) -> None:
    for name, t in tensors.items():
        if t.dim() != 2 or t.dtype != dtype or t.shape[0] != rows:
            _fail(f"`{name}` must be a ({rows}, heads * head_dim) {dtype} tensor")
        if t.numel() and (t.stride(1) != 1 or t.stride(0) % 8 or t.stride(0) < t.shape[1] and rows > 1 or t.data_ptr() % 16):
            _fail(f"`{name}` needs unit stride in a row, a row stride that is a multiple of 8 and 16-byte alignment")


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _cache(dtype: torch.dtype, k_cache: torch.Tensor, v_cache: torch.Tensor) -> int:
    """Checks a pair of caches; returns the elements from page to page."""
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if t.dim() != 4 or t.dtype != dtype or t.shape != k_cache.shape:
            _fail(f"`{name}` must be a (n_pages, n_kv_heads, page_size, head_dim) {dtype} tensor, k_cache and v_cache alike")
        if t.shape[2] not in (16, 32, 64, 128):
            _fail("page_size must be 16, 32, 64 or 128")
        n, g, ps, hd = t.shape
        if t.numel() and (t.stride()[1:] != (ps * hd, hd, 1) or n > 1 and t.stride(0) < g * ps * hd or t.stride(0) % 8 or t.data_ptr() % 16):
            _fail(f"`{name}`: a page must be contiguous and 16-byte aligned, pages a multiple of 8 values apart")
        if n > 1 and t.stride(0) != k_cache.stride(0):
            _fail("k_cache and v_cache must have their pages equally far apart")
    n, g, ps, hd = k_cache.shape
    return k_cache.stride(0) if n > 1 else g * ps * hd


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


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
    _on_gpu(cached.device, cached=cached, new=new, tables=tables, free_pages=free_pages, n_free=n_free)
    B = cached.numel()
    _whole(torch.int32, B, cached=cached, new=new)
    _whole(torch.int32, None, free_pages=free_pages)
    _whole(torch.int32, 1, n_free=n_free)
    if tables.dim() != 2 or tables.dtype != torch.int32 or tables.shape[0] != B or tables.numel() and (tables.stride(1) != 1 or B > 1 and tables.stride(0) < tables.shape[1]):
        _fail(f"`tables` must be an int32 ({B}, width) tensor with unit stride in a row")
    dev = cached.device
    width = tables.shape[1]
    plan = PagePlan(torch.empty(B + 1, dtype=torch.int32, device=dev), torch.empty(B, dtype=torch.int32, device=dev),
                    torch.empty(rows, dtype=torch.int64, device=dev), torch.empty(rows, dtype=torch.int64, device=dev),
                    torch.empty(1, dtype=torch.int32, device=dev))
    with torch.cuda.device(dev):
        st = _lib.load().eptq_plan_pages(cached.data_ptr(), new.data_ptr(), B, tables.data_ptr(), tables.stride(0) if B > 1 else width, width,
                                         free_pages.data_ptr(), free_pages.numel(), n_free.data_ptr(), int(page_size), int(rows),
                                         plan.cu_rows.data_ptr(), plan.kv_lens.data_ptr(), plan.positions.data_ptr(),
                                         plan.slots.data_ptr(), plan.n_free.data_ptr(), _stream(dev))
    _lib.check(st, "eptq plan_pages")
    return plan


def rope_append_paged(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      positions: torch.Tensor, slots: torch.Tensor, inv_freq: torch.Tensor, scaling: float = 1.0,
                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary embedding of packed q and k (rows, heads * head_dim) and the store of k and v at `slots` of the caches;
    returns the rotated q (`out`, which may be q itself, or a new tensor).  Pairs (i, i + head_dim / 2), angle
    positions[r] * inv_freq[i] formed in 64 bits, cos and sin kept in 32.  q, k and v may be column ranges of one
    projection's output.  A slot outside the cache (-1: a row without one) is not written; slots differ otherwise, or
    the slot holds a mixture."""
    _on_gpu(q.device, q=q, k=k, v=v, k_cache=k_cache, v_cache=v_cache, positions=positions, slots=slots, inv_freq=inv_freq)
    if q.dtype not in _DTYPES:
        _fail("rope_append_paged takes fp16 or bf16 tensors")
    rows = q.shape[0]
    _packed(q.dtype, rows, q=q, k=k, v=v)
    page_stride = _cache(q.dtype, k_cache, v_cache)
    n_pages, nkv, ps, hd = k_cache.shape
    if hd == 0 or q.shape[1] % hd or q.shape[1] == 0 or k.shape[1] != nkv * hd or v.shape[1] != nkv * hd:
        _fail("q, k and v must hold whole heads of the caches' head_dim, k and v as many as the caches")
    _whole(torch.int64, rows, positions=positions, slots=slots)
    _whole(torch.float32, hd // 2, inv_freq=inv_freq)
    out = torch.empty((rows, q.shape[1]), dtype=q.dtype, device=q.device) if out is None else _check_out(out, q)
    with torch.cuda.device(q.device):
        st = _lib.load().eptq_rope_append_paged(_DTYPES[q.dtype], q.data_ptr(), _row_stride(q), k.data_ptr(), _row_stride(k), v.data_ptr(),
                                                _row_stride(v), out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), page_stride,
                                                positions.data_ptr(), slots.data_ptr(), inv_freq.data_ptr(), rows, q.shape[1] // hd, nkv,
                                                hd, n_pages, ps, float(scaling), _stream(q.device))
    _lib.check(st, "eptq rope_append_paged")
    return out


def _check_out(out: torch.Tensor, q: torch.Tensor) -> torch.Tensor:
    _on_gpu(q.device, out=out)
    if out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous() or out.data_ptr() % 16:
        _fail("`out` must be contiguous, of q's shape and type")
    return out


def _attention(a: "_lib.EptqAttention", q: torch.Tensor, cu_rows: torch.Tensor, scale: Optional[float],
               out: Optional[torch.Tensor]) -> torch.Tensor:
    lib = _lib.load()
    out = torch.empty((q.shape[0], q.shape[1]), dtype=q.dtype, device=q.device) if out is None else _check_out(out, q)
    a.dtype, a.rows, a.batch = _DTYPES[q.dtype], q.shape[0], cu_rows.numel() - 1
    a.scale = float(scale if scale is not None else a.head_dim ** -0.5)
    a.q_stride, a.q, a.cu_rows, a.out = _row_stride(q), q.data_ptr(), cu_rows.data_ptr(), out.data_ptr()
    with torch.cuda.device(q.device):
        # Scratch of its own for every call, from torch's allocator: calls on different streams, and graphs captured on one
        # stream and replayed on others, share none.  The status word is the framework's (see workspace_status_all).
        a.status = workspace_for(q.device, 1 << 20).data_ptr() + _STATUS_WORD
        need = lib.eptq_ragged_attention_workspace_bytes(C.byref(a))
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        st = lib.eptq_ragged_attention(C.byref(a), ws.data_ptr() if need else None, need, _stream(q.device))
    _lib.check(st, "eptq ragged attention")
    return out


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, tables: torch.Tensor,
                    kv_lens: torch.Tensor, cu_rows: torch.Tensor, max_rows: int, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of every request's new rows over its pages: request b owns the rows cu_rows[b] .. cu_rows[b+1]-1
    of q (rows, n_heads * head_dim), they are the last of its kv_lens[b] keys, and row t of n sees the keys
    0 .. kv_lens[b] - n + t.  One row per request while tokens are generated, many for a chunk of a prompt, both in one
    call.  `max_rows`: the most rows that one request has; it chooses the kernel and changes no result but its rounding.
    Rows that see no key come out as zeros, rows behind the last request as they were in `out`.  A page id outside the
    cache stands for keys that are not there."""
    _on_gpu(q.device, q=q, k_cache=k_cache, v_cache=v_cache, tables=tables, kv_lens=kv_lens, cu_rows=cu_rows)
    if q.dtype not in _DTYPES:
        _fail("paged_attention takes fp16 or bf16 tensors")
    _packed(q.dtype, q.shape[0], q=q)
    page_stride = _cache(q.dtype, k_cache, v_cache)
    n_pages, nkv, ps, hd = k_cache.shape
    if hd == 0 or q.shape[1] == 0 or q.shape[1] % hd:
        _fail("q must hold whole heads of the caches' head_dim")
    _whole(torch.int32, None, cu_rows=cu_rows)
    B = cu_rows.numel() - 1
    _whole(torch.int32, B, kv_lens=kv_lens)
    if tables.dim() != 2 or tables.dtype != torch.int32 or tables.shape[0] != B or tables.numel() and (tables.stride(1) != 1 or B > 1 and tables.stride(0) < tables.shape[1]):
        _fail(f"`tables` must be an int32 ({B}, width) tensor with unit stride in a row")
    a = _lib.EptqAttention()
    a.n_heads, a.n_kv_heads, a.head_dim, a.max_rows = q.shape[1] // hd, nkv, hd, int(max_rows)
    a.page_size, a.n_pages, a.table_width = ps, n_pages, tables.shape[1]
    a.table_stride = tables.stride(0) if B > 1 else tables.shape[1]
    a.k_stride = a.v_stride = page_stride
    a.k, a.v, a.tables, a.kv_lens = k_cache.data_ptr(), v_cache.data_ptr(), tables.data_ptr(), kv_lens.data_ptr()
    return _attention(a, q, cu_rows, scale, out)


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_rows: torch.Tensor, head_dim: int,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention inside each of many prompts packed into one call: q (rows, n_heads * head_dim), k and v
    (rows, n_kv_heads * head_dim), prompt b in the rows cu_rows[b] .. cu_rows[b+1]-1.  q, k and v may be column ranges of
    one projection's output.  Rows behind the last prompt stay as they were in `out`."""
    _on_gpu(q.device, q=q, k=k, v=v, cu_rows=cu_rows)
    if q.dtype not in _DTYPES:
        _fail("prompt_attention takes fp16 or bf16 tensors")
    _packed(q.dtype, q.shape[0], q=q, k=k, v=v)
    if q.shape[1] == 0 or k.shape[1] == 0 or q.shape[1] % head_dim or k.shape[1] % head_dim or k.shape != v.shape:
        _fail("q, k and v must hold whole heads of head_dim, k and v as many")
    _whole(torch.int32, None, cu_rows=cu_rows)
    a = _lib.EptqAttention()
    a.n_heads, a.n_kv_heads, a.head_dim, a.max_rows = q.shape[1] // head_dim, k.shape[1] // head_dim, int(head_dim), q.shape[0]
    a.k_stride, a.v_stride, a.k, a.v = _row_stride(k), _row_stride(v), k.data_ptr(), v.data_ptr()
    return _attention(a, q, cu_rows, scale, out)
