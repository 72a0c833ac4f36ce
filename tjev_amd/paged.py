"""The paged key/value cache and its attention on MI355X: the full-attention layers that stand between the
GDN layers of a served hybrid decoder, beside ``gdn_prefill`` and ``gdn_decode_step`` (serve.py). Inference
only, through the HIP library: there is no gradient, and tensors that carry one raise outside
torch.no_grad(). Nothing here waits for the GPU or reads a length on the host.

A step of a batch, with what every layer shares first:

    t = paged_tables(cached, new, block_table, free_pages, taken, page_size=P, tokens=N)
    q, k = rotary_axes(q, k, positions, inv_freq, sections=...)            (rotary.py)
    paged_append(k, v, k_cache, v_cache, t.slots)
    out = paged_attention(q, k_cache, v_cache, t.block_table, t.starts, t.lengths, gate=gate)

Caches are [pages, page_size, kv_heads, dim] with any strides whose last dim is contiguous (another order
of the dims, or keys and values in one tensor, are views of this). Token t of a request lies in page
block_table[request, t // page_size] at place t % page_size; its slot is page * page_size + place. A
table entry that is no page of the cache (-1) holds no keys. Every call runs on torch's current stream of the
tensors' device; workspaces come from torch's allocator, so calls on several streams, and captured
graphs, have their own. Calls recorded by jit tracing or make_fx raise.
"""

from __future__ import annotations

import ctypes
import functools
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


def _int32(x: torch.Tensor) -> torch.Tensor:
    return x if x.dtype == torch.int32 and x.is_contiguous() else x.to(torch.int32).contiguous()


def _device(x: torch.Tensor | None, like: torch.Tensor) -> int:
    return like.get_device() if x is None else x.get_device()


def _check_sizes(*sizes: int) -> None:
    """The library's sizes are 32-bit numbers: a larger one would arrive as its low half."""
    if max(sizes) >= 1 << 31:
        raise ValueError(f"tables, pages and page sizes of less than 2^31, not {max(sizes)}")


def _check_caches(k_shape, k_stride, k_dtype, v_shape, v_stride, v_dtype, heads: int, dim: int) -> None:
    if len(k_shape) != 4 or k_shape[2:] != (heads, dim) or v_shape != k_shape or v_dtype != k_dtype:
        raise ValueError(f"caches [pages, page_size, {heads}, {dim}] of one type, not {tuple(k_shape)} {k_dtype} and {tuple(v_shape)} "
                         f"{v_dtype}")
    if dim > 1 and (k_stride[-1] != 1 or v_stride[-1] != 1):
        raise ValueError("the caches' last dim must be contiguous (a copy would leave the caller's cache unchanged)")
    _check_sizes(*k_shape[:2])


# The checks and parameters of a call depend on its shapes, strides, types and options alone, and are kept by
# them (the latest 256; a decode loop's calls are alike).
@functools.lru_cache(maxsize=256)
def _tables_params(t_shape, t_stride, t_dtype, lengths, list_shapes, int_dtypes, page_size: int, tokens: int, inplace: bool, devices):
    if len(t_shape) != 2 or t_dtype != torch.int32:
        raise ValueError(f"block_table is [requests, pages] int32, not {tuple(t_shape)} {t_dtype}")
    requests, width = t_shape
    if not 1 <= requests <= _lib.MAX_REQUESTS or width < 1 or page_size < 1 or tokens < 0:
        raise ValueError(f"1 to {_lib.MAX_REQUESTS} requests of pages of at least one token, not {requests} of {width} pages of "
                         f"{page_size}, and {tokens} tokens")
    _check_sizes(width, page_size)
    if lengths != ((requests,), (requests,)):
        raise ValueError(f"lengths {tuple(map(tuple, lengths))} of {requests} requests")
    free_shape, taken_size = list_shapes
    if len(free_shape) != 1 or taken_size != 1:
        raise ValueError("free_pages is a list of pages and taken one number")
    for dt in int_dtypes:
        if dt not in (torch.int32, torch.int64):
            raise ValueError(f"lengths, pages and taken are int32 or int64, not {dt}")
    _lib.one_gpu("paged_tables", devices)
    if inplace and ((width > 1 and t_stride[1] != 1) or (requests > 1 and t_stride[0] != width)):
        raise ValueError("inplace: the block table must be contiguous (a copy would leave the caller's unchanged)")
    return ctypes.byref(_lib.PagedParams(tokens=tokens, requests=requests, table_width=width, page_size=page_size))


def paged_tables(cached: torch.Tensor, new: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                 taken: torch.Tensor | None = None, *, page_size: int, tokens: int, inplace: bool = False) -> PagedTables:
    """Block tables and slot maps of a step, built on the GPU in one launch: request b holds ``cached[b]``
    tokens and brings ``new[b]``. It keeps the pages of its cached tokens (the first entries of its row of
    ``block_table`` [B, M] int32) and takes the further ones it needs from ``free_pages`` [F], in order of the
    requests from index ``taken`` [1] (None: 0). Entries behind a request's pages come back -1; with
    ``inplace`` the taken ones are written into ``block_table`` and all others left. ``tokens``: the size of the
    slot map; slots behind the last request's tokens, and of tokens without a page (past the free list or the
    table's width), are -1. Unused requests have both lengths 0; up to 8192 requests."""
    _lib.not_recorded("paged_tables")
    p = _tables_params(
        block_table.shape, block_table.stride(), block_table.dtype, (cached.shape, new.shape),
        (free_pages.shape, 1 if taken is None else taken.numel()),
        (cached.dtype, new.dtype, free_pages.dtype, torch.int32 if taken is None else taken.dtype), int(page_size), int(tokens),
        bool(inplace), (block_table.get_device(), cached.get_device(), new.get_device(), free_pages.get_device(),
                        _device(taken, block_table)))
    dev, requests = block_table.device, block_table.shape[0]
    cached, new, free_pages, table = _int32(cached), _int32(new), _int32(free_pages), block_table.contiguous()
    taken = None if taken is None else _int32(taken)
    table_out = table if inplace else torch.empty_like(table)
    slots = torch.empty(int(tokens), dtype=torch.int64, device=dev)
    starts, lengths, taken_out = torch.empty(2 * requests + 2, dtype=torch.int32, device=dev).split((requests + 1, requests, 1))
    with _lib.on_device(dev):
        _lib.check_status(_lib.load().tjev_gdn_paged_tables(
            p, _lib.current_stream(dev), cached.data_ptr(), new.data_ptr(), table.data_ptr(), free_pages.data_ptr(), free_pages.shape[0],
            None if taken is None else taken.data_ptr(), table_out.data_ptr(), slots.data_ptr(), starts.data_ptr(), lengths.data_ptr(),
            taken_out.data_ptr()))
    return PagedTables(block_table if inplace else table_out, slots, starts, lengths, taken_out)


@functools.lru_cache(maxsize=256)
def _append_params(k_shape, k_stride, k_dtype, v_shape, v_stride, v_dtype, kc_shape, kc_stride, kc_dtype, vc_shape, vc_stride, vc_dtype,
                   s_shape, s_dtype, devices):
    if len(k_shape) != 3 or k_shape != v_shape or k_dtype != v_dtype:
        raise ValueError(f"k and v are [tokens, heads, dim] alike, not {tuple(k_shape)} {k_dtype} and {tuple(v_shape)} {v_dtype}")
    if k_dtype not in _DTYPES or kc_dtype != k_dtype:
        raise ValueError(f"paged_append takes float32 or bfloat16 tensors of the cache's type, not {k_dtype} for {kc_dtype}")
    tokens, heads, dim = k_shape
    _check_caches(kc_shape, kc_stride, kc_dtype, vc_shape, vc_stride, vc_dtype, heads, dim)
    if s_shape != (tokens,) or s_dtype not in (torch.int32, torch.int64):
        raise ValueError(f"slots are [{tokens}] int32 or int64, not {tuple(s_shape)} {s_dtype}")
    if any(s == 0 and n > 1 for strides in (kc_stride, vc_stride) for s, n in zip(strides, kc_shape)):
        raise ValueError("an expanded cache cannot be written")
    _lib.one_gpu("paged_append", devices)
    return ctypes.byref(_lib.PagedParams(
        tokens=tokens, pages=kc_shape[0], page_size=kc_shape[1], kv_heads=heads, dim=dim, dtype=_DTYPES[k_dtype], k_stride=kc_stride[:3],
        v_stride=vc_stride[:3], k_new_stride=k_stride[:2], v_new_stride=v_stride[:2]))


def paged_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor) -> None:
    """Writes the new tokens' k and v [N, kv_heads, dim] (any strides with a contiguous last dim) into the
    slots [N] of the caches, in place. Slots outside the cache (-1) are skipped. The slots of one call are
    distinct: of two tokens with one slot, either's values or parts of both remain."""
    _lib.not_recorded("paged_append")
    if _lib.dual_level() or (torch.is_grad_enabled() and (k.requires_grad or v.requires_grad or k_cache.requires_grad
                                                          or v_cache.requires_grad)):
        _lib.inference_only("paged_append", k, v, k_cache, v_cache)
    if k.dim() == 3 and k.stride(-1) != 1:
        k = k.contiguous()
    if v.dim() == 3 and v.stride(-1) != 1:
        v = v.contiguous()
    p = _append_params(
        k.shape, k.stride(), k.dtype, v.shape, v.stride(), v.dtype, k_cache.shape, k_cache.stride(), k_cache.dtype, v_cache.shape,
        v_cache.stride(), v_cache.dtype, slots.shape, slots.dtype,
        (k.get_device(), v.get_device(), k_cache.get_device(), v_cache.get_device(), slots.get_device()))
    slots, dev = slots.to(torch.int64).contiguous(), k.device
    with _lib.on_device(dev):
        _lib.check_status(_lib.load().tjev_gdn_paged_append(
            p, _lib.current_stream(dev), k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), slots.data_ptr()))


@functools.lru_cache(maxsize=256)
def _attention_params(lib, q_shape, q_stride, q_dtype, kc_shape, kc_stride, kc_dtype, vc_shape, vc_stride, vc_dtype, t_shape, t_dtype,
                      s_shape, s_dtype, l_shape, l_dtype, gate, out, scale, max_new, devices):
    """The library's view of a call (a reference to the struct; never changed) and its workspace. gate and out: their
    (shape, stride, dtype), or None."""
    if len(q_shape) != 3 or q_dtype not in _DTYPES or kc_dtype != q_dtype:
        raise ValueError(f"q is [tokens, heads, dim], float32 or bfloat16 as the cache is, not {tuple(q_shape)} {q_dtype} for {kc_dtype}")
    tokens, heads, dim = q_shape
    kv_heads = kc_shape[2] if len(kc_shape) == 4 else 0
    _check_caches(kc_shape, kc_stride, kc_dtype, vc_shape, vc_stride, vc_dtype, kv_heads, dim)
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} query heads are not groups of {kv_heads} key heads")
    if len(t_shape) != 2 or t_dtype != torch.int32:
        raise ValueError(f"block_table is [requests, pages] int32, not {tuple(t_shape)} {t_dtype}")
    if dim % 8 or not 8 <= dim <= 256:
        raise ValueError(f"head dims in multiples of 8 up to 256, not {dim}")
    requests = t_shape[0]
    _check_sizes(*t_shape)
    if requests < 1 or t_shape[1] < 1 or kc_shape[0] < 1 or kc_shape[1] < 1:
        raise ValueError(f"a block table {tuple(t_shape)} or a cache {tuple(kc_shape)} without pages")
    if s_shape != (requests + 1,) or l_shape != (requests,):
        raise ValueError(f"starts {tuple(s_shape)} and lengths {tuple(l_shape)} of {requests} requests")
    for dt in (s_dtype, l_dtype):
        if dt not in (torch.int32, torch.int64):
            raise ValueError(f"starts and lengths are int32 or int64, not {dt}")
    for name, t in (("gate", gate), ("out", out)):
        if t is not None and (t[0] != q_shape or t[2] != q_dtype):
            raise ValueError(f"{name} {tuple(t[0])} {t[2]} is not like q {tuple(q_shape)} {q_dtype}")
    if out is not None and (out[1][-1] != 1 or any(s == 0 and n > 1 for s, n in zip(out[1], out[0]))):
        raise ValueError("out's last dim must be contiguous, and none expanded")
    if max_new is not None and not 1 <= max_new < 1 << 31:
        raise ValueError(f"max_new is a number of tokens, not {max_new}")
    _lib.one_gpu("paged_attention", devices)
    p = _lib.PagedParams(tokens, requests, t_shape[1], kc_shape[0], kc_shape[1], heads, kv_heads, dim, _DTYPES[q_dtype], int(out is None),
                         dim ** -0.5 if scale is None else scale, _strides(q_shape, q_stride),
                         (0, 0) if gate is None else _strides(*gate[:2]), (heads * dim, dim) if out is None else _strides(*out[:2]),
                         _strides(kc_shape, kc_stride), _strides(vc_shape, vc_stride), max_new=max_new or 0)
    return ctypes.byref(p), lib.tjev_gdn_paged_workspace_bytes(ctypes.byref(p))


def _strides(shape, stride):
    """The strides of all dims but the last, 0 where a dim has one place: no distance between rows, which may be any number."""
    return tuple(s if n > 1 else 0 for n, s in zip(shape[:-1], stride))


def _like(x: torch.Tensor | None):
    return None if x is None else (x.shape, x.stride(), x.dtype)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    starts: torch.Tensor, lengths: torch.Tensor, *, scale: float | None = None,
                    gate: torch.Tensor | None = None, out: torch.Tensor | None = None, max_new: int | None = None) -> torch.Tensor:
    """Causal attention of the batch's new tokens over the paged cache, which holds their own keys and
    values already: one token per request, chunks of prompts, or both in one call.

    q [N, heads, dim] (heads: groups of kv_heads; dim in multiples of 8 up to 256): rows starts[b] ..
    starts[b + 1] - 1 are the last tokens of request b, whose keys are ``lengths[b]`` in all, in the pages of row b of
    ``block_table`` [B, M] int32. Each attends to the keys up to its own, softmax(scale q k^T) v with scale
    dim^-1/2 by default, in 32 bits; a row without keys is 0. ``gate`` [N, heads, dim] multiplies the result by its sigmoid.
    Rows of no request (a padded batch) come back 0, or, with ``out`` given, are left as they were.
    ``max_new``: the most new tokens of one request, where the caller knows; it chooses kernels and no row's keys. By default
    every request is taken to bring one token at least, so a batch whose table has unused places, and whose tokens are no more
    than its places, is served as decoding requests: right, but a prompt in it takes up to four times as long.
    (In bf16 the kernel for many rows rounds the weights to bf16 for their product with v. It takes the requests of more than 16
    tokens times query heads per key head, 32 at head dims up to 64 where the average or max_new is 17 to 32 of them, of
    batches that may hold one by max_new or the default.)
    q, gate and out may be views whose rows start on 16 bytes (q and gate are copied where they do not); out is
    none of the inputs. What the cache holds elsewhere (NaN too) does not matter."""
    _lib.not_recorded("paged_attention")
    if _lib.dual_level() or (torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad or (
            gate is not None and gate.requires_grad) or (out is not None and out.requires_grad))):
        _lib.inference_only("paged_attention", q, k_cache, v_cache, gate, out)
    # (contiguous() would leave a contiguous view that starts off 16 bytes where it is)
    if q.dim() == 3 and not _aligned(q):
        q = q.clone(memory_format=torch.contiguous_format)
    if gate is not None and gate.dim() == 3 and not _aligned(gate):
        gate = gate.clone(memory_format=torch.contiguous_format)
    lib = _lib.load()
    p, need = _attention_params(
        lib, q.shape, q.stride(), q.dtype, k_cache.shape, k_cache.stride(), k_cache.dtype, v_cache.shape, v_cache.stride(), v_cache.dtype,
        block_table.shape, block_table.dtype, starts.shape, starts.dtype, lengths.shape, lengths.dtype, _like(gate), _like(out),
        None if scale is None else float(scale), None if max_new is None else int(max_new),
        (q.get_device(), k_cache.get_device(), v_cache.get_device(), block_table.get_device(), starts.get_device(), lengths.get_device(),
         _device(gate, q), _device(out, q)))
    starts, lengths, block_table, dev = _int32(starts), _int32(lengths), block_table.contiguous(), q.device
    y = torch.empty_like(q, memory_format=torch.contiguous_format) if out is None else out
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    with _lib.on_device(dev):
        _lib.check_status(lib.tjev_gdn_paged_attention(
            p, _lib.current_stream(dev), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), starts.data_ptr(),
            lengths.data_ptr(), None if gate is None else gate.data_ptr(), y.data_ptr(), ws.data_ptr(), need))
    return y


def _aligned(x: torch.Tensor) -> bool:
    """Whether the rows of x [N, heads, dim] start on 16 bytes."""
    s, e = x.stride(), 16 // x.element_size()
    return s[2] == 1 and (s[0] % e == 0 or x.shape[0] == 1) and (s[1] % e == 0 or x.shape[1] == 1) and x.data_ptr() % 16 == 0
