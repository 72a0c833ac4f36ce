"""The paged key/value cache and its attention on MI355X: the full-attention layers that stand between the
GDN layers of a served hybrid decoder, beside ``gdn_prefill`` and ``gdn_decode_step`` (serve.py). Inference
only, through the HIP library: there is no gradient, and tensors that carry one raise outside
torch.no_grad(). Nothing here waits for the GPU or reads a length on the host.

A step of a batch, with what every layer shares first:

    t = paged_tables(cached, new, block_table, free_pages, taken, page_size=P, tokens=N)
    q, k = rotary_axes(q, k, positions, inv_freq, sections=...)            (rotary.py)
    paged_append(k, v, k_cache, v_cache, t.slots)
    out = paged_attention(q, k_cache, v_cache, t.block_table, t.starts, t.lengths, gate=gate)

With trees of drafted tokens (drafts.py: their ancestors and positions, their verification) attention is
``paged_tree_attention``; ``paged_compact`` moves the accepted ones to their places in all layers, and
``paged_fork`` says which requests go on, with how much of what they hold: sharing pages, copying last ones and giving back what
nobody holds.

Caches are [pages, page_size, kv_heads, dim] with any strides whose last dim is contiguous (another order
of the dims, or keys and values in one tensor, are views of this). Token t of a request lies in page
block_table[request, t // page_size] at place t % page_size; its slot is page * page_size + place. A
table entry that is no page of the cache (-1) holds no keys. Every call runs on torch's current stream of the
tensors' device; workspaces come from torch's allocator, so calls on several streams, and captured
graphs, have their own. Calls recorded by jit tracing or make_fx raise.
"""

from __future__ import annotations

import array
import ctypes
import functools
import operator
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


def _int32_near(x: torch.Tensor) -> torch.Tensor:
    """_int32 of numbers that may be anything: those past 32 bits become the last of them, not their low half."""
    return _int32(x.clamp(-(1 << 31), (1 << 31) - 1) if x.dtype == torch.int64 else x)


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
                      s_shape, s_dtype, l_shape, l_dtype, gate, out, scale, max_new, devices, what):
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
    _lib.one_gpu(what, devices)
    p = _lib.PagedParams(tokens, requests, t_shape[1], kc_shape[0], kc_shape[1], heads, kv_heads, dim, _DTYPES[q_dtype], int(out is None),
                         dim ** -0.5 if scale is None else scale, _strides(q_shape, q_stride),
                         (0, 0) if gate is None else _strides(*gate[:2]), (heads * dim, dim) if out is None else _strides(*out[:2]),
                         _strides(kc_shape, kc_stride), _strides(vc_shape, vc_stride), max_new=max_new or 0)
    need = lib.tjev_gdn_paged_workspace_bytes if what == "paged_attention" else lib.tjev_gdn_paged_tree_workspace_bytes
    return ctypes.byref(p), need(ctypes.byref(p))


def _strides(shape, stride):
    """The strides of all dims but the last, 0 where a dim has one place: no distance between rows, which may be any number."""
    return tuple(s if n > 1 else 0 for n, s in zip(shape[:-1], stride))


def _like(x: torch.Tensor | None):
    return None if x is None else (x.shape, x.stride(), x.dtype)


def _attend(what: str, q, k_cache, v_cache, block_table, starts, lengths, ancestors, scale, gate, out, max_new) -> torch.Tensor:
    """paged_attention, and with ancestors paged_tree_attention."""
    _lib.not_recorded(what)
    if _lib.dual_level() or (torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad or (
            gate is not None and gate.requires_grad) or (out is not None and out.requires_grad))):
        _lib.inference_only(what, q, k_cache, v_cache, gate, out)
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
         _device(gate, q), _device(out, q), _device(ancestors, q)), what)
    starts, lengths, block_table, dev = _int32(starts), _int32(lengths), block_table.contiguous(), q.device
    y = torch.empty_like(q, memory_format=torch.contiguous_format) if out is None else out
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    gate_at = None if gate is None else gate.data_ptr()
    with _lib.on_device(dev):
        stream = _lib.current_stream(dev)
        if ancestors is None:
            status = lib.tjev_gdn_paged_attention(
                p, stream, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), starts.data_ptr(),
                lengths.data_ptr(), gate_at, y.data_ptr(), ws.data_ptr(), need)
        else:
            ancestors = ancestors.contiguous()
            status = lib.tjev_gdn_paged_tree_attention(
                p, stream, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), starts.data_ptr(),
                lengths.data_ptr(), ancestors.data_ptr(), ancestors.shape[1], gate_at, y.data_ptr(), ws.data_ptr(), need)
        _lib.check_status(status)
    return y


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
    return _attend("paged_attention", q, k_cache, v_cache, block_table, starts, lengths, None, scale, gate, out, max_new)


def paged_tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                         starts: torch.Tensor, lengths: torch.Tensor, ancestors: torch.Tensor, *, scale: float | None = None,
                         gate: torch.Tensor | None = None, out: torch.Tensor | None = None, max_new: int | None = None) -> torch.Tensor:
    """``paged_attention`` of trees of new tokens: each attends to all keys before its request's new tokens and, of those, to the
    ones that its row of ``ancestors`` [N, W] int64 names (bit j % 64 of word j / 64: the request's j-th), in whatever order they
    stand; as ``draft_tree`` makes them these are its ancestors and itself. A row may name any of them, or none (one that then
    has no keys is 0); a request's tokens from 64 W on cannot be named. ``max_new``: the most new tokens of one request; it
    chooses kernels and no row's keys. All else as for ``paged_attention``, but for which rows have their weights rounded in bf16:

    Kernels are chosen by the table's width too, the only bound on the keys that the host has. Batches that may hold a request of more
    than 16 tokens times query heads per key head (32 as there) go to the kernel for many rows, for those requests, except where all of
    them in tiles of 16 (32) rows, each counted as M * page_size keys in blocks of 128 and three blocks more, are at most four blocks to
    a workgroup, of which there are 512 (768 at head dims up to 64): small batches in tables not much wider than they need, which take up
    to a third less time for it (one tree of 12 over 4000, 16/4 heads of 256: 20 us, in a table for 16384 keys or more 26)."""
    if ancestors.dim() != 2 or ancestors.shape[0] != q.shape[0] or ancestors.shape[1] < 1 or ancestors.dtype != torch.int64:
        raise ValueError(f"ancestors are [{q.shape[0]}, words] int64, not {tuple(ancestors.shape)} {ancestors.dtype}")
    _check_sizes(ancestors.shape[1])
    return _attend("paged_tree_attention", q, k_cache, v_cache, block_table, starts, lengths, ancestors, scale, gate, out, max_new)


def _aligned(x: torch.Tensor) -> bool:
    """Whether the rows of x [N, heads, dim] start on 16 bytes."""
    s, e = x.stride(), 16 // x.element_size()
    return s[2] == 1 and (s[0] % e == 0 or x.shape[0] == 1) and (s[1] % e == 0 or x.shape[1] == 1) and x.data_ptr() % 16 == 0


# ---------------------------------------------------------------- who holds the pages
class Forked(NamedTuple):
    """What paged_fork leaves: the block table [B', M] int32 and lengths [B'] int32 of the places that go on, the free list [F], the
    pages taken of it [1] (more than there are: a shortage) and how many hold each page beside its first holder [pages], int32."""

    block_table: torch.Tensor
    lengths: torch.Tensor
    free_pages: torch.Tensor
    taken: torch.Tensor
    shared: torch.Tensor


_alike = operator.attrgetter("dtype", "requires_grad")
_size, _stride, _get_device, _address = torch.Tensor.size, torch.Tensor.stride, torch.Tensor.get_device, torch.Tensor.data_ptr


def _layers(what: str, caches):
    """The layers' caches as the library takes them: what they have in common (kept checks go by it), their number, and the addresses
    of all k's, then of all v's. A look at each tensor in C, for all at once: 0.5 us a layer."""
    pairs = list(caches)
    if not pairs:
        return None, 0, _NO_LAYERS
    if set(map(len, pairs)) != {2}:
        raise ValueError(f"{what} takes pairs of caches, k and v of every layer")
    ks, vs = zip(*pairs)
    flat = ks + vs
    sizes, k_strides, v_strides, alike, devices = (set(map(_size, flat)), set(map(_stride, ks)), set(map(_stride, vs)), set(map(_alike, flat)),
                                                   set(map(_get_device, flat)))
    if _lib.dual_level() or any(grad for _, grad in alike):
        _lib.inference_only(what, *flat)
    if len(sizes) > 1 or len(k_strides) > 1 or len(v_strides) > 1 or len({dt for dt, _ in alike}) > 1:
        raise ValueError(f"the layers' caches are alike in shape, strides and type, not {sizes} {k_strides} {v_strides} {[dt for dt, _ in alike]}")
    return (sizes.pop(), k_strides.pop(), v_strides.pop(), alike.pop()[0], *devices), len(pairs), array.array("Q", map(_address, flat))


def _of_layers(what: str, layers: int, addresses) -> tuple[int, int]:
    """Where the library finds the addresses of k's and of v's. Tokens of a cache that is listed twice would be moved twice, by
    workgroups at once."""
    if len(set(addresses)) < 2 * layers:
        raise ValueError(f"{what}: a cache is given twice (layers that share one name it once)")
    at = addresses.buffer_info()[0]
    return at, at + 8 * layers


_NO_LAYERS = array.array("Q", (0,))


def _pages_params(what: str, like, layers: int, page_size, pages, **kw):
    """The library's parameters, the caches' part from what they have in common (None: there are none)."""
    if like is None:
        return _lib.PagesParams(pages=1 if pages is None else pages, page_size=1 if page_size is None else page_size, **kw)
    shape, k_stride, v_stride, dtype = like[:4]
    if len(shape) != 4 or dtype not in _DTYPES:
        raise ValueError(f"caches are [pages, page_size, heads, dim], float32 or bfloat16, not {tuple(shape)} {dtype}")
    _check_caches(shape, k_stride, dtype, shape, v_stride, dtype, shape[2], shape[3])
    if min(shape) < 1:
        raise ValueError(f"caches {tuple(shape)} without pages, heads or values")
    if page_size not in (None, shape[1]) or pages not in (None, shape[0]):
        raise ValueError(f"{what}: {pages} pages of {page_size} tokens, and caches {tuple(shape)}")
    if any(s == 0 and n > 1 for strides in (k_stride, v_stride) for s, n in zip(strides, shape)):
        raise ValueError("an expanded cache cannot be written")
    return _lib.PagesParams(pages=shape[0], page_size=shape[1], kv_heads=shape[2], dim=shape[3], dtype=_DTYPES[dtype], layers=layers,
                            k_stride=k_stride[:3], v_stride=v_stride[:3], **kw)


@functools.lru_cache(maxsize=256)
def _compact_params(like, layers: int, t_shape, t_dtype, s_shape, s_dtype, l_shape, l_dtype, p_shape, p_dtype, k_shape, k_dtype, devices):
    if len(t_shape) != 2 or t_dtype != torch.int32 or not 1 <= t_shape[0] <= _lib.MAX_REQUESTS or t_shape[1] < 1:
        raise ValueError(f"block_table is [requests, pages] int32 of 1 to {_lib.MAX_REQUESTS} requests, not {tuple(t_shape)} {t_dtype}")
    requests = t_shape[0]
    _check_sizes(t_shape[1])
    if s_shape != (requests + 1,) or l_shape != (requests,) or k_shape != (requests,):
        raise ValueError(f"starts {tuple(s_shape)}, lengths {tuple(l_shape)} and kept {tuple(k_shape)} of {requests} requests")
    if len(p_shape) != 2 or p_shape[0] != requests or p_shape[1] < 1:
        raise ValueError(f"path is [{requests}, max_new], not {tuple(p_shape)}")
    _check_sizes(p_shape[1])
    for dt in (s_dtype, l_dtype, p_dtype, k_dtype):
        if dt not in (torch.int32, torch.int64):
            raise ValueError(f"starts, lengths, path and kept are int32 or int64, not {dt}")
    p = _pages_params("paged_compact", like, layers, None, None, max_new=p_shape[1], requests=requests, table_width=t_shape[1])
    _lib.one_gpu("paged_compact", (*devices, *like[4:]) if like else devices)
    return ctypes.byref(p)


def paged_compact(caches, block_table: torch.Tensor, starts: torch.Tensor, lengths: torch.Tensor, path: torch.Tensor,
                  kept: torch.Tensor) -> torch.Tensor:
    """Moves the kept ones of every request's new tokens to the front of them, in all layers' caches at once, in place, and
    returns the lengths that are left [B] int32: token path[b, j] becomes the j-th, j < kept[b], as ``verify_drafts`` names them.

    ``caches``: the (k_cache, v_cache) of every layer, alike in shape and strides, none of them twice or part of another (none: the
    lengths alone). ``starts`` and ``lengths`` are the step's, with the new tokens. A request's numbers in ``path`` [B, max_new] grow; those
    that are less than their place, or no new token, are left out. A page that holds new tokens is held by one request; those are distinct.
    What stands behind a request's kept tokens is left as it was."""
    _lib.not_recorded("paged_compact")
    like, layers, addresses = _layers("paged_compact", caches)
    p = _compact_params(
        like, layers, block_table.shape, block_table.dtype, starts.shape, starts.dtype, lengths.shape, lengths.dtype, path.shape, path.dtype,
        kept.shape, kept.dtype, (block_table.get_device(), starts.get_device(), lengths.get_device(), path.get_device(), kept.get_device()))
    k_at, v_at = _of_layers("paged_compact", layers, addresses)
    dev = block_table.device
    table, starts, lengths, path, kept = block_table.contiguous(), _int32(starts), _int32(lengths), _int32_near(path), _int32_near(kept)
    out = torch.empty_like(lengths)
    with _lib.on_device(dev):
        _lib.check_status(_lib.load().tjev_gdn_paged_compact(
            p, _lib.current_stream(dev), k_at, v_at, table.data_ptr(), starts.data_ptr(), lengths.data_ptr(),
            path.data_ptr(), kept.data_ptr(), out.data_ptr()))
    return out


@functools.lru_cache(maxsize=256)
def _fork_params(lib, like, layers: int, t_shape, t_dtype, l_shape, l_dtype, s_shape, s_dtype, keep, f_shape, f_dtype, taken, sh_shape, sh_dtype,
                 page_size: int, devices):
    """The library's view of a call and its workspace. keep: its (shape, dtype) or None; taken: its (size, dtype)."""
    if len(t_shape) != 2 or t_dtype != torch.int32 or not 1 <= t_shape[0] <= _lib.MAX_REQUESTS or t_shape[1] < 1:
        raise ValueError(f"block_table is [requests, pages] int32 of 1 to {_lib.MAX_REQUESTS} requests, not {tuple(t_shape)} {t_dtype}")
    if page_size < 1:
        raise ValueError(f"pages of at least one token, not {page_size}")
    if l_shape != (t_shape[0],):
        raise ValueError(f"lengths {tuple(l_shape)} of {t_shape[0]} requests")
    if len(s_shape) != 1 or not 1 <= s_shape[0] <= _lib.MAX_REQUESTS or (keep is not None and keep[0] != s_shape):
        raise ValueError(f"sources and keep are [new requests] of 1 to {_lib.MAX_REQUESTS}, not {tuple(s_shape)} and {keep and tuple(keep[0])}")
    if len(f_shape) != 1 or len(sh_shape) != 1 or sh_shape[0] < 1 or taken[0] != 1:
        raise ValueError("free_pages is a list of pages, taken one number, and shared a number for every page")
    for dt in (l_dtype, s_dtype, f_dtype, taken[1], sh_dtype, *(() if keep is None else (keep[1],))):
        if dt not in (torch.int32, torch.int64):
            raise ValueError(f"lengths, sources, keep, pages and their numbers are int32 or int64, not {dt}")
    _check_sizes(t_shape[0] * t_shape[1], s_shape[0] * t_shape[1], f_shape[0], sh_shape[0], page_size)
    p = ctypes.byref(_pages_params("paged_fork", like, layers, page_size, sh_shape[0], n_free=f_shape[0], requests=t_shape[0],
                                   new_requests=s_shape[0], table_width=t_shape[1]))
    _lib.one_gpu("paged_fork", (*devices, *like[4:]) if like else devices)
    return p, lib.tjev_gdn_fork_workspace_bytes(p)


def paged_fork(caches, block_table: torch.Tensor, lengths: torch.Tensor, sources: torch.Tensor, keep: torch.Tensor | None,
               free_pages: torch.Tensor, taken: torch.Tensor, shared: torch.Tensor, *, page_size: int) -> Forked:
    """Which requests go on, with what: place i of the new table with the first ``keep[i]`` tokens (None: all) of place
    ``sources[i]`` [B'] of ``block_table`` [B, M] (-1: it is unused). That is a batch's samples or beams (a source several times),
    a roll back behind rejected drafts (``keep`` shorter), requests that end (no place goes on from them) and a table made dense, all at
    once, on the GPU. ``lengths`` [B] are those that the places have pages for: after a step the step's own (``PagedTables.lengths``), not
    what was kept of it, or the pages of the rest would be nobody's.

    ``shared`` [pages]: how many hold each page beside its first holder (0 in the beginning). Places share pages; but a last page with room
    in it, where the next tokens go, has one holder: the first place that goes on in it where nobody holds it otherwise, and for each
    other one a page is taken and the tokens are copied in all layers' ``caches`` ((k_cache, v_cache) pairs, alike in shape and strides,
    none of them twice, in pages of up to 2^20 - 16 tokens; those may be none). Pages that nobody holds any more come back in front of index
    ``taken`` of ``free_pages`` [F], in the table's order, and are the first to be taken again; the list needs room for them there, as it
    has where all of them were taken from it. A copy that finds no page gets -1, and ``taken`` is over F.

    A call with ``keep`` is taken to be a step's roll back, where few pages change hands; it is right with any, but slower than one without
    where thousands do (64 places of 512 pages, all given back: 180 us instead of 27).

    Nothing given is changed but the caches: the new table, lengths, list, ``taken`` and ``shared`` come back."""
    _lib.not_recorded("paged_fork")
    lib = _lib.load()
    like, layers, addresses = _layers("paged_fork", caches)
    p, need = _fork_params(
        lib, like, layers, block_table.shape, block_table.dtype, lengths.shape, lengths.dtype, sources.shape, sources.dtype,
        None if keep is None else (keep.shape, keep.dtype), free_pages.shape, free_pages.dtype, (taken.numel(), taken.dtype), shared.shape,
        shared.dtype, int(page_size),
        (block_table.get_device(), lengths.get_device(), sources.get_device(), _device(keep, lengths), free_pages.get_device(),
         taken.get_device(), shared.get_device()))
    k_at, v_at = _of_layers("paged_fork", layers, addresses)
    dev = block_table.device
    table, lengths, sources, free, taken, shared = (block_table.contiguous(), _int32(lengths), _int32_near(sources), _int32(free_pages),
                                                    _int32(taken), _int32(shared))
    keep = None if keep is None else _int32_near(keep)
    # (tensors of their own: a part of a larger one takes longer to make)
    table_out, ws = table.new_empty((sources.shape[0], table.shape[1])), torch.empty(need, dtype=torch.uint8, device=dev)
    lengths_out, free_out, taken_out, shared_out = torch.empty_like(sources), torch.empty_like(free), taken.new_empty(1), torch.empty_like(shared)
    with _lib.on_device(dev):
        _lib.check_status(lib.tjev_gdn_paged_fork(
            p, _lib.current_stream(dev), k_at, v_at, table.data_ptr(), lengths.data_ptr(), sources.data_ptr(),
            None if keep is None else keep.data_ptr(), free.data_ptr(), taken.data_ptr(), shared.data_ptr(), table_out.data_ptr(),
            lengths_out.data_ptr(), free_out.data_ptr(), taken_out.data_ptr(), shared_out.data_ptr(), ws.data_ptr(), need))
    return Forked(table_out, lengths_out, free_out, taken_out, shared_out)
