"""The paged key/value cache and its attention on MI355X: the full-attention layers that stand between the
GDN layers of a served hybrid decoder, beside ``gdn_prefill`` and ``gdn_decode_step`` (serve.py). Inference
only (no autograd), through the HIP library; nothing here waits for the GPU or reads a length on the host.

A step of a batch, with what every layer shares first:

    t = paged_tables(cached, new, block_table, free_pages, taken, page_size=P, tokens=N)
    q, k = rotary_axes(q, k, positions, inv_freq, sections=...)            (rotary.py)
    paged_append(k, v, k_cache, v_cache, t.slots)
    out = paged_attention(q, k_cache, v_cache, t.block_table, t.starts, t.lengths, gate=gate)

Caches are [pages, page_size, kv_heads, dim] with any strides whose last dim is contiguous (another order
of the dims, or keys and values in one tensor, are views of this). Token t of a request lies in page
block_table[request, t // page_size] at place t % page_size; its slot is page * page_size + place. A
table entry that is no page of the cache (-1) holds no keys. Every call runs on torch's current stream of the tensors'
device; workspaces come from torch's allocator, so calls on several streams, and captured graphs,
have their own.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}


class PagedTables(NamedTuple):
    """What a step's layers share: the block table [B, M] int32, the new tokens' slots [tokens] int64, the
    requests' first tokens [B + 1] int32, their lengths (cached + new) [B] int32, and the pages taken so
    far [1] int32 (more than there are free ones: a shortage)."""

    block_table: torch.Tensor
    slots: torch.Tensor
    starts: torch.Tensor
    lengths: torch.Tensor
    taken: torch.Tensor


def _on_gpu(what: str, first: torch.Tensor, *rest) -> None:
    for t in (first, *rest):
        if t is not None and not t.is_cuda:
            raise RuntimeError(f"{what} runs on the GPU (HIP); got a CPU tensor")
        if t is not None and t.device != first.device:
            raise ValueError(f"{what}: tensors on {first.device} and {t.device}")


def _int32(x: torch.Tensor) -> torch.Tensor:
    return x if x.dtype == torch.int32 and x.is_contiguous() else x.to(torch.int32).contiguous()


def _caches(k_cache: torch.Tensor, v_cache: torch.Tensor, heads: int, dim: int) -> None:
    for c in (k_cache, v_cache):
        if c.dim() != 4 or c.shape[2:] != (heads, dim) or c.shape != k_cache.shape or c.dtype != k_cache.dtype:
            raise ValueError(f"caches [pages, page_size, {heads}, {dim}] of one type, not {tuple(k_cache.shape)} {k_cache.dtype} "
                             f"and {tuple(v_cache.shape)} {v_cache.dtype}")
        if c.shape[-1] > 1 and c.stride(-1) != 1:
            raise ValueError("the caches' last dim must be contiguous (a copy would leave the caller's cache unchanged)")


def paged_tables(cached: torch.Tensor, new: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                 taken: torch.Tensor | None = None, *, page_size: int, tokens: int, inplace: bool = False) -> PagedTables:
    """Block tables and slot maps of a step, built on the GPU in one launch: request b holds ``cached[b]``
    tokens and brings ``new[b]``. It keeps the pages of its cached tokens (the first entries of its row of
    ``block_table`` [B, M] int32) and takes the further ones it needs from ``free_pages`` [F], in order of the
    requests from index ``taken`` [1] (None: 0). Entries behind a request's pages come back -1; with
    ``inplace`` the taken ones are written into ``block_table`` and all others left. ``tokens``: the size of the
    slot map; slots behind the last request's tokens, and of tokens without a page (past the free list or the
    table's width), are -1. Unused requests have both lengths 0; up to 8192 requests."""
    if block_table.dim() != 2 or block_table.dtype != torch.int32:
        raise ValueError(f"block_table is [requests, pages] int32, not {tuple(block_table.shape)} {block_table.dtype}")
    requests, width = block_table.shape
    if not 1 <= requests <= _lib.MAX_REQUESTS or width < 1 or page_size < 1 or tokens < 0:
        raise ValueError(f"1 to {_lib.MAX_REQUESTS} requests of pages of at least one token, not {requests} of {width} pages of "
                         f"{page_size}, and {tokens} tokens")
    if cached.shape != (requests,) or new.shape != (requests,):
        raise ValueError(f"lengths {tuple(cached.shape)} and {tuple(new.shape)} of {requests} requests")
    if free_pages.dim() != 1 or (taken is not None and taken.numel() != 1):
        raise ValueError("free_pages is a list of pages and taken one number")
    for t in (cached, new, free_pages, taken):
        if t is not None and t.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"lengths, pages and taken are int32 or int64, not {t.dtype}")
    _on_gpu("paged_tables", block_table, cached, new, free_pages, taken)
    if inplace and not block_table.is_contiguous():
        raise ValueError("inplace: the block table must be contiguous (a copy would leave the caller's unchanged)")
    dev = block_table.device
    cached, new, free_pages, table = _int32(cached), _int32(new), _int32(free_pages), block_table.contiguous()
    taken = None if taken is None else _int32(taken)
    p = _lib.PagedParams(tokens=int(tokens), requests=requests, table_width=width, page_size=int(page_size))
    table_out = table if inplace else torch.empty_like(table)
    slots = torch.empty(max(0, int(tokens)), dtype=torch.int64, device=dev)
    small = torch.empty(2 * requests + 2, dtype=torch.int32, device=dev)
    starts, lengths, taken_out = small[:requests + 1], small[requests + 1:-1], small[-1:]
    with _lib.on_device(dev):
        _lib.check_status(_lib.load().tjev_gdn_paged_tables(
            ctypes.byref(p), _lib.current_stream(dev), cached.data_ptr(), new.data_ptr(), table.data_ptr(), free_pages.data_ptr(),
            free_pages.numel(), None if taken is None else taken.data_ptr(), table_out.data_ptr(), slots.data_ptr(),
            starts.data_ptr(), lengths.data_ptr(), taken_out.data_ptr()))
    return PagedTables(table_out, slots, starts, lengths, taken_out)


def paged_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor) -> None:
    """Writes the new tokens' k and v [N, kv_heads, dim] (any strides with a contiguous last dim) into the
    slots [N] of the caches, in place. Slots outside the cache (-1) are skipped. The slots of one call are
    distinct: of two tokens with one slot, either's values or parts of both remain."""
    if k.dim() != 3 or k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError(f"k and v are [tokens, heads, dim] alike, not {tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
    if k.dtype not in _DTYPES or k_cache.dtype != k.dtype:
        raise ValueError(f"paged_append takes float32 or bfloat16 tensors of the cache's type, not {k.dtype} for {k_cache.dtype}")
    tokens, heads, dim = k.shape
    _caches(k_cache, v_cache, heads, dim)
    if slots.shape != (tokens,) or slots.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"slots are [{tokens}] int32 or int64, not {tuple(slots.shape)} {slots.dtype}")
    if any(s == 0 and n > 1 for c in (k_cache, v_cache) for s, n in zip(c.stride(), c.shape)):
        raise ValueError("an expanded cache cannot be written")
    _on_gpu("paged_append", k, v, k_cache, v_cache, slots)
    k, v = (x if x.stride(-1) == 1 else x.contiguous() for x in (k, v))
    slots = slots.to(torch.int64).contiguous()
    p = _lib.PagedParams(tokens=tokens, pages=k_cache.shape[0], page_size=k_cache.shape[1], kv_heads=heads, dim=dim,
                         dtype=_DTYPES[k.dtype], k_stride=k_cache.stride()[:3], v_stride=v_cache.stride()[:3],
                         k_new_stride=k.stride()[:2], v_new_stride=v.stride()[:2])
    with _lib.on_device(k.device):
        _lib.check_status(_lib.load().tjev_gdn_paged_append(
            ctypes.byref(p), _lib.current_stream(k.device), k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
            slots.data_ptr()))


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    starts: torch.Tensor, lengths: torch.Tensor, *, scale: float | None = None,
                    gate: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of the batch's new tokens over the paged cache, which holds their own keys and
    values already: one token per request, chunks of prompts, or both in one call.

    q [N, heads, dim] (heads: groups of kv_heads; dim in multiples of 8 up to 256): rows starts[b] ..
    starts[b + 1] - 1 are the last tokens of request b, whose keys are ``lengths[b]`` in all, in the pages of row b of
    ``block_table`` [B, M] int32. Each attends to the keys up to its own, softmax(scale q k^T) v with scale
    dim^-1/2 by default, in 32 bits; a row without keys is 0. ``gate`` [N, heads, dim] multiplies the result by its
    sigmoid. Rows of no request (a padded batch) come back 0, or, with ``out`` given, are left as they were.
    q, gate and out may be views whose rows start on 16 bytes. What the cache holds elsewhere (NaN too) does
    not matter."""
    if q.dim() != 3 or q.dtype not in _DTYPES or k_cache.dtype != q.dtype:
        raise ValueError(f"q is [tokens, heads, dim], float32 or bfloat16 as the cache is, not {tuple(q.shape)} {q.dtype} "
                         f"for {k_cache.dtype}")
    tokens, heads, dim = q.shape
    kv_heads = k_cache.shape[2] if k_cache.dim() == 4 else 0
    _caches(k_cache, v_cache, kv_heads, dim)
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} query heads are not groups of {kv_heads} key heads")
    if block_table.dim() != 2 or block_table.dtype != torch.int32:
        raise ValueError(f"block_table is [requests, pages] int32, not {tuple(block_table.shape)} {block_table.dtype}")
    if dim % 8 or not 8 <= dim <= 256:
        raise ValueError(f"head dims in multiples of 8 up to 256, not {dim}")
    requests = block_table.shape[0]
    if requests < 1 or block_table.shape[1] < 1 or k_cache.shape[0] < 1 or k_cache.shape[1] < 1:
        raise ValueError(f"a block table {tuple(block_table.shape)} or a cache {tuple(k_cache.shape)} without pages")
    if starts.shape != (requests + 1,) or lengths.shape != (requests,):
        raise ValueError(f"starts {tuple(starts.shape)} and lengths {tuple(lengths.shape)} of {requests} requests")
    for t in (starts, lengths):
        if t.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"starts and lengths are int32 or int64, not {t.dtype}")
    for name, t in (("gate", gate), ("out", out)):
        if t is not None and (t.shape != q.shape or t.dtype != q.dtype):
            raise ValueError(f"{name} {tuple(t.shape)} {t.dtype} is not like q {tuple(q.shape)} {q.dtype}")
    if out is not None and (out.stride(-1) != 1 or any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape))):
        raise ValueError("out's last dim must be contiguous, and none expanded")
    _on_gpu("paged_attention", q, k_cache, v_cache, block_table, starts, lengths, gate, out)
    q, gate = (x if x is None or _aligned(x) else x.contiguous() for x in (q, gate))
    starts, lengths, block_table = _int32(starts), _int32(lengths), block_table.contiguous()
    dev = q.device
    y = torch.empty((tokens, heads, dim), dtype=q.dtype, device=dev) if out is None else out
    p = _lib.PagedParams(tokens, requests, block_table.shape[1], k_cache.shape[0], k_cache.shape[1], heads, kv_heads, dim,
                         _DTYPES[q.dtype], int(out is None), dim ** -0.5 if scale is None else float(scale), q.stride()[:2],
                         (0, 0) if gate is None else gate.stride()[:2], y.stride()[:2], k_cache.stride()[:3], v_cache.stride()[:3])
    lib = _lib.load()
    ws = torch.empty(lib.tjev_gdn_paged_workspace_bytes(ctypes.byref(p)), dtype=torch.uint8, device=dev)
    with _lib.on_device(dev):
        _lib.check_status(lib.tjev_gdn_paged_attention(
            ctypes.byref(p), _lib.current_stream(dev), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(),
            starts.data_ptr(), lengths.data_ptr(), None if gate is None else gate.data_ptr(), y.data_ptr(), ws.data_ptr(), ws.numel()))
    return y


def _aligned(x: torch.Tensor) -> bool:
    """Whether the rows of x [N, heads, dim] start on 16 bytes."""
    e = 16 // x.element_size()
    return x.stride(2) == 1 and x.stride(0) % e == 0 and x.stride(1) % e == 0 and x.data_ptr() % 16 == 0
