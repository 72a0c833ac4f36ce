"""Rotary positions with several axes (time, height, width) on MI355X, computed by the HIP library.

The hybrid decoder whose GDN layers this package runs puts a full-attention layer after every third of
them; its queries and keys are turned by their positions before they meet. ``rotary_axes`` turns
the first 2 * len(inv_freq) lanes of every head of q and k in one launch: pair i by the angle
positions[axis of i] * inv_freq[i], the angle taken in 64 bits and the turn in 32, rounded once. The
axes divide the pairs by ``sections``. Differentiable in q and k (the gradient is the turn back and keeps
neither of them); positions and frequencies take no gradient. Forward-mode derivatives raise, as do recorded calls
(jit tracing, make_fx). A gradient
may be captured into a HIP graph when no eager graph of the same leaves is alive, as torch requires of any
operator. There is no fallback: without the HIP library, or on a CPU tensor, the operator raises.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
_POSITION_BITS = {torch.int32: 32, torch.int64: 64}
_FREQ_BITS = {torch.float32: 32, torch.float64: 64}


@functools.lru_cache(maxsize=256)
def _checked(q_shape, q_dtype, k_shape, k_dtype, p_shape, p_dtype, f_shape, f_dtype, sections, interleaved: bool, devices):
    """The checks of a call, kept by its shapes, types and options: the number of axes."""
    if q_dtype not in _DTYPES:
        raise ValueError(f"rotary_axes takes float32 or bfloat16 tensors, not {q_dtype}")
    if len(q_shape) < 3 or len(f_shape) != 1:
        raise ValueError(f"q is [..., T, heads, dim] and inv_freq [pairs], not {tuple(q_shape)} and {tuple(f_shape)}")
    if k_shape is not None and (len(k_shape) != len(q_shape) or k_shape[:-2] != q_shape[:-2] or k_shape[-1] != q_shape[-1]
                                or k_dtype != q_dtype):
        raise ValueError(f"k {tuple(k_shape)} {k_dtype} does not go with q {tuple(q_shape)} {q_dtype}")
    lead, half, dim = q_shape[:-2], f_shape[0], q_shape[-1]
    if sections is None and p_shape == lead:
        p_shape = (1, *p_shape)
    if p_shape[1:] != lead or len(p_shape) != len(lead) + 1:
        raise ValueError(f"positions {tuple(p_shape)} are not one of {tuple(lead)} per axis")
    if p_dtype not in _POSITION_BITS or f_dtype not in _FREQ_BITS:
        raise ValueError(f"positions are int32 or int64 and frequencies float32 or float64, not {p_dtype} and {f_dtype}")
    secs = [half] if sections is None else list(sections)
    if not 0 < 2 * half <= dim or dim % 2:
        raise ValueError(f"{half} frequencies turn {2 * half} lanes of heads of {dim}")
    if not 1 <= len(secs) <= _lib.MAX_AXES:
        raise ValueError(f"1 to {_lib.MAX_AXES} position axes, not {len(secs)}")
    if min(secs) < 0 or sum(secs) != half:
        raise ValueError(f"sections {secs} do not add up to {half} pairs")
    if p_shape[0] != len(secs):
        raise ValueError(f"positions of {p_shape[0]} axes for {len(secs)} sections")
    if interleaved and any(n and a + len(secs) * (n - 1) >= half for a, n in enumerate(secs) if a):
        raise ValueError(f"interleaved sections {secs}: an axis runs out of the {half} pairs")
    _lib.one_gpu("rotary_axes", devices)
    return len(secs)


@functools.lru_cache(maxsize=256)
def _params(q_shape, q_stride, dtype, k_shape, k_stride, half, axes, sections, interleaved, adjacent, inverse, p_dtype, f_dtype):
    """The library's view of a call (a reference to the struct; never changed): q [B, T, Hq, D], k [B, T, Hk, D] or None;
    [T, Hq, D] is a batch of one."""
    if len(q_shape) == 3:
        q_shape, q_stride = (1, *q_shape), (0, *q_stride)
        if k_shape is not None:
            k_shape, k_stride = (1, *k_shape), (0, *k_stride)
    batch, length, heads, dim = q_shape
    return ctypes.byref(_lib.RotaryParams(
        batch, length, heads, 0 if k_shape is None else k_shape[2], dim, 2 * half, axes, (ctypes.c_int32 * _lib.MAX_AXES)(*sections),
        interleaved, adjacent, inverse, _DTYPES[dtype], _POSITION_BITS[p_dtype], _FREQ_BITS[f_dtype], 0, q_stride[:3],
        (0, 0, 0) if k_shape is None else k_stride[:3]))


def _launch(q, k, positions, inv_freq, axes, sections, interleaved: bool, adjacent: bool, inverse: bool):
    """The library's call: q [B, T, Hq, D] or [T, Hq, D], k alike or None (the last dim contiguous)."""
    _lib.not_recorded("rotary_axes")
    dev = q.device
    p = _params(q.shape, q.stride(), q.dtype, None if k is None else k.shape, None if k is None else k.stride(), inv_freq.shape[0],
                axes, sections, interleaved, adjacent, inverse, positions.dtype, inv_freq.dtype)
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = None if k is None else torch.empty_like(k, memory_format=torch.contiguous_format)
    with _lib.on_device(dev):
        _lib.check_status(_lib.load().tjev_gdn_rotary(
            p, _lib.current_stream(dev), q.data_ptr(), None if k is None else k.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(),
            q_out.data_ptr(), None if k is None else k_out.data_ptr()))
    return q_out, k_out


def _rows(x):
    """x with its last dim contiguous (a copy only where it is not)."""
    return x if x.stride(-1) == 1 else x.contiguous()


class _Rotary(torch.autograd.Function):
    """The launch with its gradient, which is the turn the other way: the same Function again where the backward itself
    is differentiated."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, options, inverse: bool):
        ctx.options, ctx.inverse = options, inverse
        ctx.save_for_backward(positions, inv_freq)
        return _launch(q, k, positions, inv_freq, *options, inverse)

    @staticmethod
    def backward(ctx, d_q, d_k):
        positions, inv_freq = ctx.saved_tensors
        d_q = _rows(d_q)
        d_k = _rows(d_k) if ctx.needs_input_grad[1] else None
        d_q, d_k = _turned(d_q, d_k, positions, inv_freq, ctx.options, not ctx.inverse)
        return d_q, d_k, None, None, None, None


def _turned(q, k, positions, inv_freq, options, inverse: bool):
    """The launch, through its Function where q or k may carry a derivative: a gradient, or (whatever the grad mode) a tangent,
    which the Function refuses. Elsewhere without it, which is some us of host time."""
    if _lib.dual_level() or (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))):
        return _Rotary.apply(q, k, positions, inv_freq, options, inverse)
    return _launch(q, k, positions, inv_freq, *options, inverse)


def rotary_axes(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, *, sections=None,
                interleaved: bool = False, adjacent: bool = False):
    """q [..., T, Hq, D] and k [..., T, Hk, D] (or None) turned by their positions: (q', k'), new contiguous tensors.

    ``positions`` [A, ..., T] (int32 or int64): one position of every token per axis; [..., T] with one
    axis and no ``sections``. ``inv_freq`` [R/2] (float32 or float64), R <= D: lanes R and up are passed
    on. ``sections``: the pairs of each axis, up to 4, adding up to R/2; the first sections[0] pairs
    turn with axis 0 and so on, or (``interleaved``) pair i with axis i mod A while i < A * sections[i mod A] and with
    axis 0 from there. A pair is lanes i and i + R/2, or 2i and 2i + 1 (``adjacent``). q and k may be views
    with any strides whose last dim is contiguous; others are copied."""
    secs = None if sections is None else tuple([int(n) for n in sections])
    interleaved, adjacent = bool(interleaved), bool(adjacent)
    axes = _checked(q.shape, q.dtype, None if k is None else k.shape, None if k is None else k.dtype, positions.shape, positions.dtype,
                    inv_freq.shape, inv_freq.dtype, secs, interleaved,
                    (q.get_device(), positions.get_device(), inv_freq.get_device(), q.get_device() if k is None else k.get_device()))
    q4, k4 = q, k
    if q.dim() > 4:
        batch = math.prod(q.shape[:-3])
        q4 = q.reshape(batch, *q.shape[-3:])
        k4 = None if k is None else k.reshape(batch, *k.shape[-3:])
    options = (axes, (inv_freq.shape[0],) if secs is None else secs, interleaved, adjacent)
    q4, k4 = _turned(_rows(q4), None if k is None else _rows(k4), positions.contiguous(), inv_freq.contiguous(), options, False)
    if q.dim() <= 4:
        return q4, k4
    return q4.reshape(q.shape), None if k is None else k4.reshape(k.shape)
