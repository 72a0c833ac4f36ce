"""Rotary positions with several axes (time, height, width) on MI355X, computed by the HIP library.

The hybrid decoder whose GDN layers this package runs puts a full-attention layer after every third of
them; its queries and keys are turned by their positions before they meet. ``rotary_axes`` turns
the first 2 * len(inv_freq) lanes of every head of q and k in one launch: pair i by the angle
positions[axis of i] * inv_freq[i], the angle taken in 64 bits and the turn in 32, rounded once. The
axes divide the pairs by ``sections``. Differentiable in q and k (the gradient is the turn back and keeps
neither of them); positions and frequencies take no gradient. There is no fallback: without the
HIP library, or on a CPU tensor, the operator raises.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
_POSITION_BITS = {torch.int32: 32, torch.int64: 64}
_FREQ_BITS = {torch.float32: 32, torch.float64: 64}


@_lib.by_value
def _options(half: int, dim: int, axes: int, sections: str, interleaved: bool):
    """The sections as the library takes them, checked (``sections``: their text, kept by value)."""
    secs = [half] if sections == "None" else [int(s) for s in sections.split()]
    if not 0 < 2 * half <= dim or dim % 2:
        raise ValueError(f"{half} frequencies turn {2 * half} lanes of heads of {dim}")
    if not 1 <= len(secs) <= _lib.MAX_AXES:
        raise ValueError(f"1 to {_lib.MAX_AXES} position axes, not {len(secs)}")
    if min(secs) < 0 or sum(secs) != half:
        raise ValueError(f"sections {secs} do not add up to {half} pairs")
    if axes != len(secs):
        raise ValueError(f"positions of {axes} axes for {len(secs)} sections")
    if interleaved and any(n and a + len(secs) * (n - 1) >= half for a, n in enumerate(secs) if a):
        raise ValueError(f"interleaved sections {secs}: an axis runs out of the {half} pairs")
    return (ctypes.c_int32 * _lib.MAX_AXES)(*secs)


def _launch(q, k, positions, inv_freq, sections, interleaved: bool, adjacent: bool, inverse: bool):
    """The library's call: q [B, T, Hq, D], k [B, T, Hk, D] or None (the last dim contiguous)."""
    batch, length, heads, dim = q.shape
    k_heads = 0 if k is None else k.shape[2]
    p = _lib.RotaryParams(batch, length, heads, k_heads, dim, 2 * inv_freq.shape[0], positions.shape[0], sections,
                          interleaved, adjacent, inverse, _DTYPES[q.dtype], _POSITION_BITS[positions.dtype],
                          _FREQ_BITS[inv_freq.dtype], 0, q.stride()[:3], (0, 0, 0) if k is None else k.stride()[:3])
    q_out = torch.empty((batch, length, heads, dim), dtype=q.dtype, device=q.device)
    k_out = None if k is None else torch.empty((batch, length, k_heads, dim), dtype=q.dtype, device=q.device)
    with _lib.on_device(q.device):
        _lib.check_status(_lib.load().tjev_gdn_rotary(
            ctypes.byref(p), _lib.current_stream(q.device), q.data_ptr(), None if k is None else k.data_ptr(),
            positions.data_ptr(), inv_freq.data_ptr(), q_out.data_ptr(), None if k is None else k_out.data_ptr()))
    return q_out, k_out


def _rows(x):
    """x with its last dim contiguous (a copy only where it is not)."""
    return x if x.stride(-1) == 1 else x.contiguous()


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, sections, interleaved, adjacent):
        ctx.options = (sections, interleaved, adjacent)
        ctx.save_for_backward(positions, inv_freq)
        return _launch(q, k, positions, inv_freq, *ctx.options, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_q, d_k):
        positions, inv_freq = ctx.saved_tensors
        if not ctx.needs_input_grad[1]:
            d_k = None
        d_q, d_k = _launch(_rows(d_q), None if d_k is None else _rows(d_k), positions, inv_freq, *ctx.options, True)
        return d_q, d_k, None, None, None, None, None


def rotary_axes(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, *, sections=None,
                interleaved: bool = False, adjacent: bool = False):
    """q [..., T, Hq, D] and k [..., T, Hk, D] (or None) turned by their positions: (q', k'), new contiguous tensors.

    ``positions`` [A, ..., T] (int32 or int64): one position of every token per axis; [..., T] with one
    axis and no ``sections``. ``inv_freq`` [R/2] (float32 or float64), R <= D: lanes R and up are passed
    on. ``sections``: the pairs of each axis, up to 4, adding up to R/2; the first sections[0] pairs
    turn with axis 0 and so on, or (``interleaved``) pair i with axis i mod A while i < A * sections[i mod A] and with
    axis 0 from there. A pair is lanes i and i + R/2, or 2i and 2i + 1 (``adjacent``). q and k may be views
    with any strides whose last dim is contiguous; others are copied."""
    if q.dtype not in _DTYPES:
        raise ValueError(f"rotary_axes takes float32 or bfloat16 tensors, not {q.dtype}")
    if q.dim() < 3 or inv_freq.dim() != 1:
        raise ValueError(f"q is [..., T, heads, dim] and inv_freq [pairs], not {tuple(q.shape)} and {tuple(inv_freq.shape)}")
    if k is not None and (k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1] or k.dtype != q.dtype):
        raise ValueError(f"k {tuple(k.shape)} {k.dtype} does not go with q {tuple(q.shape)} {q.dtype}")
    lead = q.shape[:-2]
    if sections is None and positions.shape == lead:
        positions = positions[None]
    if positions.shape[1:] != lead or positions.dim() != len(lead) + 1:
        raise ValueError(f"positions {tuple(positions.shape)} are not one of {tuple(lead)} per axis")
    if positions.dtype not in _POSITION_BITS or inv_freq.dtype not in _FREQ_BITS:
        raise ValueError(f"positions are int32 or int64 and frequencies float32 or float64, not {positions.dtype} and {inv_freq.dtype}")
    secs = _options(inv_freq.shape[0], q.shape[-1], positions.shape[0],
                    "None" if sections is None else " ".join([str(int(s)) for s in sections]), bool(interleaved))
    for t in (q, k, positions, inv_freq):
        if t is not None and not t.is_cuda:
            raise RuntimeError("rotary_axes runs on the GPU (HIP); got a CPU tensor")
        if t is not None and t.device != q.device:
            raise ValueError(f"tensors on {q.device} and {t.device}")
    batch = math.prod(lead[:-1])
    q4 = _rows(q if q.dim() == 4 else q.reshape(batch, *q.shape[-3:]))
    k4 = None if k is None else _rows(k if k.dim() == 4 else k.reshape(batch, *k.shape[-3:]))
    args = (q4, k4, positions.contiguous(), inv_freq.contiguous(), secs, bool(interleaved), bool(adjacent))
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        q4, k4 = _Rotary.apply(*args)
    else:
        q4, k4 = _launch(*args, False)
    if q.dim() == 4:
        return q4, k4
    return q4.reshape(q.shape), None if k is None else k4.reshape(k.shape)
