"""Measured operators of the attention layers that stand between the Gated DeltaNet layers: rotary
positions with several axes, the paged key/value cache (block tables and slot maps, the write of new
tokens) and attention of new tokens over it.

``draw`` gives more cases of the ranges that the listed ones stand for: 1 to 128 requests, 1 to 4096
new tokens, up to 32768 cached tokens per request, head dims 64, 128 and 256, groups of 1 to 8 query
heads per key head, pages of 8 to 128 tokens (ones that end inside a tile among them), bf16 and fp32,
rotary over one to three axes of part or all of the head, forward, and forward with backward. Lengths come
from the case alone; values and the order of the pages from the seed.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _case(name, kind, **kw):
    c = dict(kind=kind, **kw)
    return dict(name=name, **c) if name else c


def _rotary(name, batch, length, heads, kv_heads, dim, rotary, axes, interleaved, dtype, grad):
    return _case(name, "rotary", batch=batch, length=length, heads=heads, kv_heads=kv_heads, dim=dim, rotary=rotary, axes=axes,
                 interleaved=interleaved, dtype=dtype, grad=grad)


def _cache(name, kind, requests, cached, new, mix, page, heads=16, kv_heads=4, dim=256, dtype="bf16", gate=False):
    return _case(name, kind, requests=requests, cached=cached, new=new, mix=mix, page=page, heads=heads, kv_heads=kv_heads, dim=dim,
                 dtype=dtype, gate=gate)


def listed():
    return [
        # a decode batch's q and k, a quarter of each head rotated, text after images (three axes)
        _rotary("rotary_decode", 64, 1, 16, 4, 256, 64, 3, True, "bf16", False),
        # a training step's q and k over packed images and text, forward and backward
        _rotary("rotary_train", 2, 8192, 16, 4, 256, 64, 3, True, "bf16", True),
        # the scheduler's step of a decode batch: one new token a request, now and then a new page
        _cache("tables_decode", "tables", 64, 8192, 1, "ragged", 16),
        # the scheduler's step of a large batch with chunks of prompts among the decoding requests
        _cache("tables_chunks", "tables", 256, 32768, 1024, "mixed", 64),
        # the new key and value of every request of a decode batch
        _cache("append_decode", "append", 64, 4096, 1, "ragged", 16),
        # a long prompt's keys and values
        _cache("append_prompt", "append", 2, 512, 8000, "uniform", 64, heads=32, kv_heads=8, dim=128),
        # one interactive request's step: few rows, a cache of some thousand tokens
        _cache("attention_1row", "attention", 1, 4000, 1, "uniform", 16),
        # a full decode batch of very different lengths, with the layer's output gate
        _cache("attention_64rows", "attention", 64, 32768, 1, "ragged", 64, gate=True),
        # several drafted tokens a request, checked at once
        _cache("attention_draft", "attention", 32, 8192, 5, "ragged", 16, heads=32, kv_heads=8, dim=128),
        # a chunk of a long prompt over what is cached of it
        _cache("attention_chunk", "attention", 1, 30000, 2048, "uniform", 64, gate=True),
        # chunks of prompts beside decoding requests, pages that end inside a tile
        _cache("attention_mixed", "attention", 24, 6000, 1100, "mixed", 24, heads=32, kv_heads=4, dim=128),
        # a small full-precision run
        _cache("attention_fp32", "attention", 3, 1500, 200, "ragged", 16, heads=8, kv_heads=2, dim=64, dtype="fp32"),
    ]


def _spread(rng, lo, hi):
    """An integer in [lo, hi], uniform over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "tables", "append", "attention", "attention", "attention", "attention"])
    dtype = "fp32" if rng.random() < 0.2 else "bf16"
    dim = rng.choice([64, 128, 256])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 4, 5, 8])
    if kind == "rotary":
        batch = _spread(rng, 1, 4)
        return _rotary(None, batch, _spread(rng, 1, 8192 // batch), heads, kv, dim, rng.choice([dim, dim, dim // 2, dim // 4]),
                       rng.choice([1, 2, 3, 3]), rng.random() < 0.5, dtype, rng.random() < 0.5)
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    requests = _spread(rng, 1, 128)
    mix = rng.choice(["uniform", "ragged", "ragged", "mixed"])
    if kind == "tables":
        return _cache(None, kind, requests, _spread(rng, 1, 32768), _spread(rng, 1, 1024), mix, page)
    if kind == "append":
        requests = _spread(rng, 1, 32)
        return _cache(None, kind, requests, _spread(rng, 1, 1024), _spread(rng, 1, 4096 // requests), mix, page, heads, kv, dim, dtype)
    if rng.random() < 0.5:  # decoding, with drafted tokens or without: up to 2 GB of cache
        most = int(2e9 / (kv * dim * (4 if dtype == "bf16" else 8) * requests))
        cached, new = _spread(rng, 1, min(32768, most)), rng.choice([1, 1, 1, 2, 3, 6])
    else:  # chunks: as many keys as the largest listed chunk has work for (full precision: a twentieth of it)
        requests = _spread(rng, 1, 16)
        new = _spread(rng, 2, 2048 // requests)
        most = int((1e12 if dtype == "bf16" else 5e10) / (4 * requests * new * heads * dim))
        cached = _spread(rng, 1, min(32768 // requests, max(1, most - new)))
    return _cache(None, kind, requests, cached, new, mix, page, heads, kv, dim, dtype, rng.random() < 0.5)


# --------------------------------------------------------------------------- the case's lengths
def _lengths(case):
    """(cached, new) per request: alike; ragged (cached lengths spread over their logarithm); mixed: three
    of four requests decode one token, the others bring chunks, one brings nothing and the last is unused."""
    rng = random.Random(f"{case['requests']} {case['cached']} {case['new']} {case['mix']}")
    out = []
    for b in range(case["requests"]):
        c, n = case["cached"], case["new"]
        if case["mix"] != "uniform":
            c = _spread(rng, max(1, c // 64), c)
        if case["mix"] == "mixed":
            n = 1 if rng.random() < 0.75 else _spread(rng, 1, n)
            if b and b == case["requests"] // 3:
                n = 0
            if b and b == case["requests"] - 1:
                c = n = 0
        out.append((c, n))
    return out


def _pages(tokens, page):
    return -(-tokens // page)


def _sections(case):
    """The pairs of each axis: the first the rest, the others a third of them (as in text, height, width)."""
    half, a = case["rotary"] // 2, case["axes"]
    rest = [half // a] * (a - 1)
    return [half - sum(rest), *rest]


def _freqs(case):
    half = case["rotary"] // 2
    return 1e7 ** (-torch.arange(half, dtype=torch.float64) / half)


# --------------------------------------------------------------------------- inputs
def _rn(gen, *shape, dtype, std=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype) * std


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    rng = np.random.default_rng(int(seed))
    s = {"case": dict(case)}
    if case["kind"] == "rotary":
        dt, b, t = DTYPES[case["dtype"]], case["batch"], case["length"]
        s["q"], s["k"] = (_rn(gen, b, t, h, case["dim"], dtype=dt) for h in (case["heads"], case["kv_heads"]))
        if case["grad"]:
            s["dq"], s["dk"] = (_rn(gen, b, t, h, case["dim"], dtype=dt) for h in (case["heads"], case["kv_heads"]))
        # text positions go on from 0 (prefill) or stand far in (decode); the other axes lag behind the first
        base = rng.integers(0, 200000, (b, 1)) if t == 1 else rng.integers(0, 1000, (b, 1))
        time = base + np.arange(t)[None]
        axes = [time] + [np.maximum(0, time - rng.integers(0, 64, (b, t))) for _ in range(case["axes"] - 1)]
        s["positions"] = torch.from_numpy(np.stack(axes)).cuda()
        s["inv_freq"] = _freqs(case).cuda()
        return s
    page, lens = case["page"], _lengths(case)
    held = [_pages(c, page) for c, _ in lens]
    wanted = [_pages(c + n, page) for c, n in lens]
    tokens = sum(n for _, n in lens)
    width = max(1, max(wanted)) + 3  # a request may grow further
    pool = max(1, sum(wanted)) + 5
    order = rng.permutation(pool).astype(np.int32)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    s["cached"], s["new"] = i32([c for c, _ in lens]), i32([n for _, n in lens])
    if case["kind"] == "tables":
        table, at = np.full((len(lens), width), -1, np.int32), 0
        for b, n in enumerate(held):
            table[b, :n] = order[at:at + n]
            at += n
        s["table"], s["free"] = torch.from_numpy(table).cuda(), torch.from_numpy(order[at:].copy()).cuda()
        s["taken"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        s["tokens"] = tokens + 7  # the step's token buffer, a little larger than what is in it
        return s
    table, at = np.full((len(lens), width), -1, np.int32), 0
    for b, n in enumerate(wanted):
        table[b, :n] = order[at:at + n]
        at += n
    dt, hk, d = DTYPES[case["dtype"]], case["kv_heads"], case["dim"]
    s["k_cache"], s["v_cache"] = (_rn(gen, pool, page, hk, d, dtype=dt) for _ in range(2))
    if case["kind"] == "append":
        slots = np.concatenate([table[b, np.arange(c, c + n) // page].astype(np.int64) * page + np.arange(c, c + n) % page
                                for b, (c, n) in enumerate(lens)] + [np.full(3, -1)])
        s["slots"] = torch.from_numpy(slots).cuda()
        kv = _rn(gen, tokens + 3, 2, hk, d, dtype=dt)  # the projection's rows: k beside v
        s["k"], s["v"], s["tokens"] = kv[:, 0], kv[:, 1], tokens
        return s
    s["table"] = torch.from_numpy(table).cuda()
    s["starts"] = i32(np.concatenate([[0], np.cumsum([n for _, n in lens])]))
    s["lengths"] = i32([c + n for c, n in lens])
    qg = _rn(gen, tokens, case["heads"], 2 * d, dtype=dt)  # the projection's rows: each head's query beside its gate
    s["q"], s["gate"] = qg[..., :d], qg[..., d:] if case["gate"] else None
    s["lens"] = lens  # the scheduler's own copy
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "rotary" and case["grad"]:
        s["q"].requires_grad_(True)
        s["k"].requires_grad_(True)
    return s


# --------------------------------------------------------------------------- one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from tjev_amd.paged import paged_append, paged_attention, paged_tables
    from tjev_amd.rotary import rotary_axes

    case = s["case"]
    if case["kind"] == "rotary":
        q, k = rotary_axes(s["q"], s["k"], s["positions"], s["inv_freq"], sections=_sections(case), interleaved=case["interleaved"])
        if not case["grad"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
    if case["kind"] == "tables":
        t = paged_tables(s["cached"], s["new"], s["table"], s["free"], s["taken"], page_size=case["page"], tokens=s["tokens"])
        return {"table": t.block_table, "slots": t.slots, "starts": t.starts, "lengths": t.lengths, "taken": t.taken}
    if case["kind"] == "append":
        paged_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    return {"out": paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["starts"], s["lengths"], gate=s["gate"])}


def _pair_axis(case):
    """The axis of each pair: sections one after another, or the axes in turn while their sections last."""
    sec, half = _sections(case), case["rotary"] // 2
    if not case["interleaved"]:
        return [a for a, n in enumerate(sec) for _ in range(n)]
    a = len(sec)
    return [i % a if i < a * sec[i % a] else 0 for i in range(half)]


def _turn(x, cos, sin, rotary):
    """The pairs (i, i + rotary / 2) of every head turned, in 32 bits, rounded once."""
    f = x.detach().float()
    a, b, rest = f[..., :rotary // 2], f[..., rotary // 2:rotary], f[..., rotary:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1).to(x.dtype)


def _run_plain(s):
    case = s["case"]
    if case["kind"] == "rotary":
        axis = torch.tensor(_pair_axis(case)).to(s["positions"].device, non_blocking=True)
        angle = s["positions"].double().movedim(0, -1)[..., axis] * s["inv_freq"]  # [B, T, R/2], in 64 bits: far positions
        cos, sin = torch.cos(angle).float()[..., None, :], torch.sin(angle).float()[..., None, :]
        out = {n: _turn(s[n], cos, sin, case["rotary"]) for n in ("q", "k")}
        if case["grad"]:  # a turn's gradient is the turn back
            out.update({n: _turn(s[n], cos, -sin, case["rotary"]) for n in ("dq", "dk")})
        return out
    if case["kind"] == "tables":
        return _plain_tables(s, case["page"])
    if case["kind"] == "append":
        hk, d = case["kv_heads"], case["dim"]
        where = s["slots"][:s["tokens"]]  # without the token buffer's unused rows
        for n in ("k", "v"):
            s[n + "_cache"].view(-1, hk, d)[where] = s[n][:s["tokens"]]
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    out, at, g = torch.zeros_like(s["q"], memory_format=torch.contiguous_format), 0, case["heads"] // case["kv_heads"]
    for b, (c, n) in enumerate(s["lens"]):
        if not n:
            continue
        ids = s["table"][b, :_pages(c + n, case["page"])].long()
        k, v = (x[ids].flatten(0, 1)[:c + n].float().transpose(0, 1).contiguous() for x in (s["k_cache"], s["v_cache"]))  # [Hk, L, D]
        q = s["q"][at:at + n].float().reshape(n, -1, g, case["dim"]).permute(1, 2, 0, 3).flatten(1, 2)  # [Hk, g n, D]
        w = torch.matmul(q, k.transpose(1, 2)) * case["dim"] ** -0.5
        pos = torch.arange(c, c + n, device=w.device).repeat(g)
        w = w.masked_fill(torch.arange(c + n, device=w.device) > pos[:, None], -math.inf)
        w = torch.exp(w - w.amax(-1, keepdim=True))
        o = torch.matmul(w, v) / w.sum(-1, keepdim=True)
        o = o.view(-1, g, n, case["dim"]).permute(2, 0, 1, 3).flatten(1, 2)
        if s["gate"] is not None:
            o = o * torch.sigmoid(s["gate"][at:at + n].float())
        out[at:at + n] = o.to(out.dtype)
        at += n
    return {"out": out}


def _plain_tables(s, page):
    cached, new, table, free = s["cached"].long(), s["new"].long(), s["table"], s["free"]
    m, total = table.shape[1], cached + new
    held, wanted = ((x + page - 1) // page for x in (cached, total))
    held, wanted = held.clamp(max=m), wanted.clamp(max=m)
    want = wanted - held
    first = s["taken"].long() + torch.cumsum(want, 0) - want
    col = torch.arange(m, device=table.device)[None]
    at = first[:, None] + col - held[:, None]
    fresh = torch.where(at < len(free), free[at.clamp(0, len(free) - 1)], -1)
    table = torch.where(col < held[:, None], table, torch.where(col < wanted[:, None], fresh, -1)).int()
    ends = torch.cumsum(new, 0)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    t = torch.arange(s["tokens"], device=table.device)
    b = torch.searchsorted(ends, t, right=True).clamp(max=len(new) - 1)
    pos = cached[b] + t - starts[b]
    p = table[b, (pos // page).clamp(0, m - 1)].long()
    slots = torch.where((t < ends[-1]) & (p >= 0) & (pos // page < m), p * page + pos % page, -1)
    return {"table": table, "slots": slots, "starts": starts.int(), "lengths": total.int(), "taken": (s["taken"] + want.sum()).int()}


# --------------------------------------------------------------------------- work
def work(case):
    if case["kind"] == "rotary":
        e, n = (2 if case["dtype"] == "bf16" else 4), case["batch"] * case["length"]
        heads, both = case["heads"] + case["kv_heads"], 2 if case["grad"] else 1
        return {"bytes": both * (2 * n * heads * case["dim"] * e + n * case["axes"] * 8), "flops": 3.0 * both * n * heads * case["rotary"]}
    page, lens = case["page"], _lengths(case)
    tokens = sum(n for _, n in lens)
    if case["kind"] == "tables":
        width = max(1, max(_pages(c + n, page) for c, n in lens)) + 3
        return {"bytes": len(lens) * (4 * 4 + 2 * 4 * width) + 8 * (tokens + 7), "flops": 0.0}
    e, hk, d = (2 if case["dtype"] == "bf16" else 4), case["kv_heads"], case["dim"]
    if case["kind"] == "append":
        return {"bytes": tokens * (2 * 2 * hk * d * e + 8), "flops": 0.0}
    keys = sum(c + n for c, n in lens if n)
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in lens)
    rows = tokens * case["heads"] * d * e
    return {"bytes": 2 * keys * hk * d * e + rows * (3 if case["gate"] else 2) + 4 * sum(_pages(c + n, page) for c, n in lens),
            "flops": 4.0 * pairs * case["heads"] * d}


# --------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "rotary":
        inv, sec = _freqs(case).cuda(), _sections(case)
        a, half, rot = len(sec), case["rotary"] // 2, case["rotary"]
        angle = torch.empty(case["batch"], case["length"], half, dtype=torch.float64, device="cuda")
        left = list(sec)
        for i in range(half):  # pair by pair: whose section it is
            if case["interleaved"]:
                ax = i % a if i // a < sec[i % a] else 0
            else:
                ax = next(j for j in range(a) if left[j])
                left[ax] -= 1
            angle[..., i] = s["positions"][ax].double() * inv[i]
        z = torch.polar(torch.ones_like(angle), angle)[..., None, :]
        out = {}
        for n in ("q", "k") + (("dq", "dk") if case["grad"] else ()):
            x = s[n].double()
            y = torch.complex(x[..., :half].contiguous(), x[..., half:rot].contiguous()) * (z if n in ("q", "k") else z.conj())
            out[n] = torch.cat([y.real, y.imag, x[..., rot:]], -1)
        return out
    if case["kind"] == "tables":  # whole numbers: the scheduler's walk, request by request
        page, table, free = case["page"], s["table"].cpu().numpy().copy(), s["free"].cpu().tolist()
        slots, at, taken = [-1] * s["tokens"], 0, int(s["taken"])
        starts, lens = [0], _lengths(case)
        for b, (c, n) in enumerate(lens):
            table[b, _pages(c, page):] = -1
            for j in range(_pages(c, page), min(table.shape[1], _pages(c + n, page))):
                table[b, j] = free[taken] if taken < len(free) else -1
                taken += 1
            for pos in range(c, c + n):
                p = int(table[b, pos // page]) if pos // page < table.shape[1] else -1
                slots[at] = p * page + pos % page if p >= 0 else -1
                at += 1
            starts.append(at)
        return {"table": torch.from_numpy(table), "slots": torch.tensor(slots), "starts": torch.tensor(starts, dtype=torch.int32),
                "lengths": torch.tensor([c + n for c, n in lens], dtype=torch.int32), "taken": torch.tensor([taken], dtype=torch.int32)}
    page, lens = case["page"], _lengths(case)
    if case["kind"] == "append":
        out = {n: s[n].clone() for n in ("k_cache", "v_cache")}
        for n, y in out.items():
            kept = s["slots"] >= 0
            where = s["slots"][kept]
            y[torch.div(where, page, rounding_mode="floor"), where % page] = s[n[0]][kept]
        return {n: y.double() for n, y in out.items()}
    g, d = case["heads"] // case["kv_heads"], case["dim"]
    out, at = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for b, (c, n) in enumerate(lens):
        for h in range(case["kv_heads"] if n else 0):
            where = torch.arange(c + n, device="cuda")
            ids = s["table"][b].long()[where // page]
            k, v = (x[ids, where % page, h].double() for x in (s["k_cache"], s["v_cache"]))
            for j in range(h * g, h * g + g):
                w = (s["q"][at:at + n, j].double() / math.sqrt(d)) @ k.t()
                w = w.masked_fill(where[None] > torch.arange(c, c + n, device="cuda")[:, None], -math.inf)
                o = torch.softmax(w, -1) @ v
                out[at:at + n, j] = o / (1 + torch.exp(-s["gate"][at:at + n, j].double())) if case["gate"] else o
        at += n
    return {"out": out}
