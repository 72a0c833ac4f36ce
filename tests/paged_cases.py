"""Plain 64-bit forms of the attention layers' operators, and the errors their kernels may have, for the
tests: loops over requests, heads and axes on the CPU.

Tolerances count roundings: to bf16 at most 2^-8 of the value, to fp32 2^-24."""

from __future__ import annotations

import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def pair_axes(half, sections, interleaved):
    """The axis of each pair, pair by pair."""
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    out = []
    for i in range(half):
        a = i % len(sections)
        out.append(a if i < len(sections) * sections[a] else 0)
    return out


def rotary64(x, positions, inv_freq, sections, interleaved=False, adjacent=False, sign=1.0):
    """x [B, T, H, D] turned in 64 bits, and |a| + |b| of every lane's pair (0 on the lanes passed on)."""
    half = inv_freq.shape[0]
    x, y, mag = x.double(), x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    for i, ax in enumerate(pair_axes(half, sections, interleaved)):
        t = sign * positions[ax].double()[..., None] * float(inv_freq[i].double())
        p, q = (2 * i, 2 * i + 1) if adjacent else (i, i + half)
        a, b = x[..., p], x[..., q]
        y[..., p] = a * torch.cos(t) - b * torch.sin(t)
        y[..., q] = b * torch.cos(t) + a * torch.sin(t)
        mag[..., p] = mag[..., q] = a.abs() + b.abs()
    return y, mag


def rotary_room(y, mag, dtype):
    """The fraction of a turn is rounded to fp32 (an angle off by pi 2^-25), sine and cosine are within 2 ulp
    (2^-23), the two products and their sum 2^-23: 3 * 2^-23 < 2^-21 of |a| + |b|; then the stored rounding."""
    room = mag * 2.0 ** -21
    return room + HALF_STEP[dtype] * (y.abs() + room)


def tables_walk(cached, new, table, free, taken, page, tokens, inplace=False):
    """The scheduler's walk over the requests: lists in, (table, slots, starts, lengths, taken) out."""
    width = len(table[0])
    table = [list(r) for r in table]
    slots, starts, at = [-1] * tokens, [0], 0
    for b, (c, n) in enumerate(zip(cached, new)):
        c, n = max(0, c), max(0, n)
        held, wanted = min(width, -(-c // page)), min(width, -(-(c + n) // page))
        for j in range(held, wanted):
            table[b][j] = free[taken] if taken < len(free) else -1
            taken += 1
        if not inplace:
            table[b][wanted:] = [-1] * (width - wanted)
        for pos in range(c, c + n):
            p = table[b][pos // page] if pos // page < width else -1
            if at < tokens and p >= 0:
                slots[at] = p * page + pos % page
            at += 1
        starts.append(at)
    return table, slots, starts, [max(0, c) + max(0, n) for c, n in zip(cached, new)], taken


def attention64(q, k_cache, v_cache, table, starts, lengths, scale=None, gate=None):
    """(out, room): the operator in 64 bits, row by row, and what a kernel's row may be off by (before the gate).
    NaN in the inputs comes out only where a row attends to it. CPU tensors."""
    n_rows, heads, dim = q.shape
    pages, page, kv, _ = k_cache.shape
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    room = torch.zeros(q.shape, dtype=torch.float64)
    half = HALF_STEP[q.dtype]
    for b in range(table.shape[0]):
        s0, s1, length = int(starts[b]), int(starts[b + 1]), int(lengths[b])
        places = [(int(table[b, t // page]), t % page) for t in range(min(max(0, length), table.shape[1] * page))]
        for j in range(s1 - s0):
            if s0 + j >= n_rows:
                break
            seen = [p for p in places[:max(0, length - (s1 - s0) + j + 1)] if 0 <= p[0] < pages]
            if not seen:
                continue
            ip, io = (torch.tensor(x) for x in zip(*seen))
            for h in range(heads):
                k, v = k_cache[ip, io, h * kv // heads].double(), v_cache[ip, io, h * kv // heads].double()
                x = q[s0 + j, h].double()
                w = torch.softmax(scale * (k @ x), 0)
                o, a = w @ v, w @ v.abs()
                # scores: products and their sums in fp32, off by delta; each weight by 4 delta at most (its own
                # power and the sum's); the sums over the keys; in bf16 the weights' rounding
                delta = (dim + 8) * 2.0 ** -24 * abs(scale) * float((k.abs() @ x.abs()).max())
                r = a * (4 * delta + (len(seen) + 64) * 2.0 ** -24 + 2.0 ** -20 + (half if q.dtype == torch.bfloat16 else 0.0))
                if gate is not None:
                    sg = torch.sigmoid(gate[s0 + j, h].double())
                    o, r = o * sg, r * sg + 2.0 ** -21 * (o * sg).abs()
                out[s0 + j, h], room[s0 + j, h] = o, r + half * (o.abs() + r)
    return out, room


def batch(gen, lens, *, heads, kv_heads, dim, page, dtype=torch.bfloat16, extra_pages=3, extra_width=1, pad_rows=0, gate=False):
    """A batch on the CPU: (cached, new) per request, pages in random order, values N(0, 1), NaN in every place of the
    cache that no token has."""
    rn = lambda *s: torch.randn(s, generator=gen).to(dtype)  # noqa: E731
    need = [-(-(c + n) // page) for c, n in lens]
    pool = sum(need) + extra_pages
    order = torch.randperm(pool, generator=gen)
    table = torch.full((len(lens), max(1, max(need)) + extra_width), -1, dtype=torch.int32)
    kc, vc = (torch.full((pool, page, kv_heads, dim), math.nan, dtype=dtype) for _ in range(2))
    at = 0
    for b, (c, n) in enumerate(lens):
        table[b, :need[b]] = order[at:at + need[b]].int()
        at += need[b]
        for cache in (kc, vc):
            t = torch.arange(c + n)
            cache[table[b].long()[t // page], t % page] = rn(c + n, kv_heads, dim)
    rows = sum(n for _, n in lens)
    starts = torch.zeros(len(lens) + 1, dtype=torch.int32)
    starts[1:] = torch.cumsum(torch.tensor([n for _, n in lens]), 0)
    lengths = torch.tensor([c + n for c, n in lens], dtype=torch.int32)
    q = rn(rows + pad_rows, heads, dim)
    return dict(q=q, k_cache=kc, v_cache=vc, block_table=table, starts=starts, lengths=lengths,
                gate=rn(rows + pad_rows, heads, dim) if gate else None)


def compare(got, want, room):
    err = (got.double().cpu() - want).abs()
    assert bool((torch.isnan(want) == torch.isnan(got.cpu())).all()), "NaN in other places"
    ok = (err <= room) | torch.isnan(want) | (got.double().cpu() == want)
    assert bool(ok.all()), f"off by {float((err / room.clamp(min=1e-300))[~ok].max()):.3g} times the tolerance"
