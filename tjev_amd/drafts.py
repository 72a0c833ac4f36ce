"""Drafted tokens of a served batch on MI355X: a step that checks several guesses of the next tokens at once, over the paged cache
(paged.py). Inference only, through the HIP library, without a word from the host about what is on the GPU:

    t = paged_tables(cached, new, block_table, free_pages, taken, page_size=P, tokens=N)
    d = draft_tree(parents, t.starts, t.lengths, max_new=M)
    q, k = rotary_axes(q, k, d.positions, inv_freq)                       (each layer)
    paged_append(k, v, k_cache, v_cache, t.slots)
    out = paged_tree_attention(q, k_cache, v_cache, t.block_table, t.starts, t.lengths, d.ancestors, max_new=M)
    ...
    v = verify_drafts(tokens, target_probs, t.starts, uniforms, parents=parents, max_new=M)
    lengths = paged_compact(caches, t.block_table, t.starts, t.lengths, v.path, v.kept)
    f = paged_fork(caches, t.block_table, t.lengths, places, lengths[places], free_pages, t.taken, shared, page_size=P)

A request's new tokens are a tree. Token 0 is its root, the token that the last step ended with; ``parents`` holds for every other the
number within the request of the one that it was drafted behind, which comes before it.

GDN layers keep a state and no keys. They run such a step a level of the trees at a time with ``gdn_decode_step``, each token from its
parent's state and conv history; none of the calls above moves those, the caller does, who made the trees and knows their levels:

    for at, above in levels:       # rows of the batch, and their parents' (of the first level: the requests' places)
        out[at], conv[at], state[at] = gdn_decode_step(qkv[at], ..., conv[above], state[above], ...)

and after verification request b goes on with those of row t.starts[b] + v.path[b, v.kept[b] - 1], or, in place i of a fork, of request
places[i]. A level reads and writes whole states (4 H Dk Dv bytes a token), and its indexing copies them once more each way.
"""

from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from . import _lib
from .paged import _device, _int32, _int32_near

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}


class DraftTree(NamedTuple):
    """What a step's layers share: of every token its ancestors and itself as bits [N, W] int64 (bit j % 64 of word j / 64: its
    request's token j), and its position [N] int32."""

    ancestors: torch.Tensor
    positions: torch.Tensor


class Verified(NamedTuple):
    """A step's outcome, -1 behind: the tokens that each request goes on with [B, max_new], the drafts that were accepted and one
    more; the numbers of the tokens whose keys are kept, the root and the accepted ones [B, max_new]; how many those are [B].
    int32."""

    tokens: torch.Tensor
    path: torch.Tensor
    kept: torch.Tensor


@functools.lru_cache(maxsize=256)
def _tree_params(p_shape, p_dtype, s_shape, s_dtype, l_shape, l_dtype, max_new: int, devices):
    if len(p_shape) != 1 or len(s_shape) != 1 or s_shape[0] < 2 or l_shape != (s_shape[0] - 1,):
        raise ValueError(f"parents are [tokens], starts [requests + 1] and lengths [requests], not {tuple(p_shape)}, {tuple(s_shape)} and "
                         f"{tuple(l_shape)}")
    for dt in (p_dtype, s_dtype, l_dtype):
        if dt not in (torch.int32, torch.int64):
            raise ValueError(f"parents, starts and lengths are int32 or int64, not {dt}")
    if not 1 <= max_new < 1 << 30:
        raise ValueError(f"max_new is a number of tokens, not {max_new}")
    _lib.one_gpu("draft_tree", devices)
    return ctypes.byref(_lib.DraftParams(tokens=p_shape[0], max_new=max_new, requests=l_shape[0]))


def draft_tree(parents: torch.Tensor, starts: torch.Tensor, lengths: torch.Tensor, *, max_new: int) -> DraftTree:
    """The ancestors and positions of every request's new tokens: rows starts[b] .. starts[b + 1] - 1 of ``parents`` [N] are those of
    request b, of ``lengths[b]`` tokens in all. A parent is a number within the request, less than the token's own; anything else is
    none, and only the cached tokens stand before such a token. The position is the number of tokens before it: cached ones and
    ancestors. ``max_new``: the most new tokens of a request; W is a 64th of it. Rows of no request and of a request's tokens from
    max_new on are 0."""
    _lib.not_recorded("draft_tree")
    p = _tree_params(parents.shape, parents.dtype, starts.shape, starts.dtype, lengths.shape, lengths.dtype, int(max_new),
                     (parents.get_device(), starts.get_device(), lengths.get_device()))
    dev = parents.device
    parents, starts, lengths = _int32_near(parents), _int32(starts), _int32(lengths)
    ancestors, positions = torch.empty((parents.shape[0], (int(max_new) + 63) // 64), dtype=torch.int64, device=dev), torch.empty_like(parents)
    with _lib.on_device(dev):
        _lib.check_status(_lib.load().tjev_gdn_draft_tree(
            p, _lib.current_stream(dev), parents.data_ptr(), starts.data_ptr(), lengths.data_ptr(), ancestors.data_ptr(), positions.data_ptr()))
    return DraftTree(ancestors, positions)


@functools.lru_cache(maxsize=256)
def _verify_params(lib, x_shape, x_dtype, t_shape, t_stride, t_dtype, s_shape, s_dtype, u_shape, u_dtype, parents, draft, max_new: int, devices):
    """The library's view of a call and its workspace. parents: their (shape, dtype), draft: its (shape, stride, dtype), or None."""
    if len(t_shape) != 2 or t_dtype not in _DTYPES or t_shape[1] < 1:
        raise ValueError(f"target_probs are [tokens, vocabulary], float32 or bfloat16, not {tuple(t_shape)} {t_dtype}")
    tokens, vocab = t_shape
    if x_shape != (tokens,) or x_dtype not in (torch.int32, torch.int64):
        raise ValueError(f"tokens are [{tokens}] int32 or int64, not {tuple(x_shape)} {x_dtype}")
    if u_shape != (tokens,) or u_dtype != torch.float32:
        raise ValueError(f"uniforms are [{tokens}] float32, not {tuple(u_shape)} {u_dtype}")
    if len(s_shape) != 1 or s_shape[0] < 2 or s_dtype not in (torch.int32, torch.int64):
        raise ValueError(f"starts are [requests + 1] int32 or int64, not {tuple(s_shape)} {s_dtype}")
    if parents is not None and (parents[0] != (tokens,) or parents[1] not in (torch.int32, torch.int64)):
        raise ValueError(f"parents are [{tokens}] int32 or int64, not {tuple(parents[0])} {parents[1]}")
    if draft is not None and (draft[0] != t_shape or draft[2] != t_dtype):
        raise ValueError(f"draft_probs {tuple(draft[0])} {draft[2]} are not like target_probs {tuple(t_shape)} {t_dtype}")
    if draft is not None and parents is not None:
        raise ValueError("draft_probs are of chains (parents None): the tokens of a tree are chosen, not drawn")
    if not 1 <= max_new < 1 << 30:
        raise ValueError(f"max_new is a number of tokens, not {max_new}")
    if vocab >= 1 << 31:
        raise ValueError(f"vocabularies of less than 2^31, not {vocab}")
    _lib.one_gpu("verify_drafts", devices)
    p = ctypes.byref(_lib.DraftParams(tokens=tokens, max_new=max_new, target_stride=t_stride[0] if tokens > 1 else 0,
                                      draft_stride=0 if draft is None or tokens < 2 else draft[1][0], requests=s_shape[0] - 1, vocab=vocab,
                                      dtype=_DTYPES[t_dtype]))
    return p, lib.tjev_gdn_verify_workspace_bytes(p)


def verify_drafts(tokens: torch.Tensor, target_probs: torch.Tensor, starts: torch.Tensor, uniforms: torch.Tensor, *,
                  parents: torch.Tensor | None = None, draft_probs: torch.Tensor | None = None, max_new: int) -> Verified:
    """Which drafted tokens are kept, and the token that the request goes on with: each emitted token is distributed as the target's.

    ``target_probs`` [N, V]: row i is the target model's distribution behind token i of the batch, ``tokens`` [N] the drafted tokens
    (a root's is not read), ``uniforms`` [N] float32 numbers in [0, 1). From the root on, a node's children are looked at in order:
    with r the node's row, child c is accepted if uniforms[c] * (1 - what target_probs[r] gives its earlier siblings) < target_probs[r,
    tokens[c]]. So are trees of chosen tokens (the likeliest ones) checked, and with ``parents`` None chains, each token behind the
    one before. A chain whose tokens were drawn from ``draft_probs`` [N, V] (row c: token c's distribution) has uniforms[c] *
    draft_probs[c, tokens[c]] < target_probs[r, tokens[c]]; a tree cannot have them.

    Where no child is accepted a token is drawn with the root's number, from what is left: target_probs[r] without the rejected
    tokens, or the positive part of target_probs[r] - draft_probs[c]: the first token whose running sum is over the number times the whole,
    in 64 bits (a number of 1 or more: the last with a probability). Where nothing is left it is drawn from target_probs[r], and
    is -1 where that holds nothing. Rows add up to one; what is no positive finite number counts as 0; a token outside the vocabulary
    is not accepted. Greedy decoding is a target_probs of ones and zeros.

    ``max_new``: the most new tokens of a request, the outputs' width; further ones are not looked at. The probabilities'
    last dim is contiguous, or they are copied."""
    _lib.not_recorded("verify_drafts")
    if _lib.dual_level() or (torch.is_grad_enabled() and (target_probs.requires_grad or uniforms.requires_grad or (
            draft_probs is not None and draft_probs.requires_grad))):
        _lib.inference_only("verify_drafts", target_probs, draft_probs, uniforms)
    if target_probs.dim() == 2 and target_probs.stride(1) != 1:
        target_probs = target_probs.contiguous()
    if draft_probs is not None and draft_probs.dim() == 2 and draft_probs.stride(1) != 1:
        draft_probs = draft_probs.contiguous()
    lib = _lib.load()
    p, need = _verify_params(
        lib, tokens.shape, tokens.dtype, target_probs.shape, target_probs.stride(), target_probs.dtype, starts.shape, starts.dtype,
        uniforms.shape, uniforms.dtype, None if parents is None else (parents.shape, parents.dtype),
        None if draft_probs is None else (draft_probs.shape, draft_probs.stride(), draft_probs.dtype), int(max_new),
        (tokens.get_device(), target_probs.get_device(), starts.get_device(), uniforms.get_device(), _device(parents, tokens),
         _device(draft_probs, tokens)))
    dev, requests, most = target_probs.device, starts.shape[0] - 1, int(max_new)
    tokens, starts, uniforms = _int32_near(tokens), _int32(starts), uniforms.contiguous()
    parents = None if parents is None else _int32_near(parents)
    out, ws = tokens.new_empty((requests, most)), torch.empty(need, dtype=torch.uint8, device=dev)
    path, kept = torch.empty_like(out), tokens.new_empty(requests)
    with _lib.on_device(dev):
        _lib.check_status(lib.tjev_gdn_verify_drafts(
            p, _lib.current_stream(dev), tokens.data_ptr(), None if parents is None else parents.data_ptr(), starts.data_ptr(),
            uniforms.data_ptr(), target_probs.data_ptr(), None if draft_probs is None else draft_probs.data_ptr(), out.data_ptr(),
            path.data_ptr(), kept.data_ptr(), ws.data_ptr(), need))
    return Verified(out, path, kept)
