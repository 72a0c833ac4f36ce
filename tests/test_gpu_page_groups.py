"""Compaction and forks (tjev_amd.paged) of caches whose tokens have more vectors than a workgroup has threads: several groups of columns, the last
of them whole or a part, against the plain forms (tests/draft_cases.py)."""

from __future__ import annotations

import random

import pytest
import torch

from draft_cases import compact_walk, starts_of
from test_gpu_drafts import _caches, _fork, _pool, _same, i32

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
# vectors of a token: 512, 320, 288, 600 (of one element), 1024 (of one element)
WIDE = [(F32, 2, 8, 256, "plain"), (F32, 1, 5, 256, "joint"), (BF, 2, 9, 256, "heads first"), (BF, 2, 8, 75, "odd"), (F32, 1, 16, 64, "odd")]


@pytest.mark.parametrize("dtype,layers,heads,dim,layout", WIDE)
@pytest.mark.parametrize("kind", ["samples", "beams", "roll back"])
@pytest.mark.parametrize("page", [1, 16, 40])
def test_forks_of_wide_tokens(dtype, layers, heads, dim, layout, kind, page):
    rng = random.Random(f"{kind} {page} {dim}")
    lens = [rng.randint(0, 4 * page) for _ in range(6)] + [3 * page, 3 * page + 1, 4 * page - 1]
    n = len(lens)
    sources = {"samples": [b for b in range(n) for _ in range(1 + b % 3)], "beams": [rng.randrange(n) for _ in range(n)], "roll back": list(range(n))}[kind]
    keep = None if kind == "samples" else [max(0, lens[b] - rng.choice([0, 1, page, page + 1])) for b in sources]
    table, free, taken, shared = _pool(rng, lens, page, 6, 30, common=2)
    caches = _caches(torch.Generator().manual_seed(dim), layers, len(shared), page, heads, dim, dtype, layout)
    print(f"fork of wide tokens {dtype} layers={layers} {heads}x{dim} {layout} {kind} page={page}", flush=True)
    _fork(caches, table, lens, sources, keep, free, taken, shared, page)


@pytest.mark.parametrize("dtype,layers,heads,dim,layout", WIDE)
def test_many_forks_of_wide_tokens(dtype, layers, heads, dim, layout):
    """More places than one workgroup's: the copies name their pages by the list."""
    rng, page = random.Random(dim), 3
    lens = [rng.randint(0, 6) for _ in range(40)]
    sources = [rng.randrange(-1, 40) for _ in range(1030)]
    table, free, taken, shared = _pool(rng, lens, page, 3, 900, common=1)
    caches = _caches(torch.Generator().manual_seed(dim), min(layers, 2), len(shared), page, heads, dim, dtype, layout)
    print(f"many forks of wide tokens {dtype} {heads}x{dim} {layout}", flush=True)
    _fork(caches, table, lens, sources, None, free, taken, shared, page)


@pytest.mark.parametrize("dtype,layers,heads,dim,layout", WIDE)
@pytest.mark.parametrize("kind", ["tree", "last", "every second"])
def test_compaction_of_wide_tokens(dtype, layers, heads, dim, layout, kind):
    from tjev_amd import paged_compact

    rng, gen, page = random.Random(dim), torch.Generator().manual_seed(dim), 12
    sizes, cached = [1, 9, 0, 30, 21], [5, 0, 31, 2, 12]
    path, kept = torch.full((len(sizes), 40), -1, dtype=torch.int32), []
    for b, n in enumerate(sizes):
        way = {"tree": sorted(rng.sample(range(n), min(n, 7))), "last": list(range(1, n)), "every second": list(range(0, n, 2))}[kind]
        path[b, :len(way)] = torch.tensor(way, dtype=torch.int32)
        kept.append(len(way))
    need = [-(-(c + n) // page) for c, n in zip(cached, sizes)]
    order = torch.randperm(sum(need) + 2, generator=gen).int()
    table, at = torch.full((len(sizes), max(need) + 1), -1, dtype=torch.int32), 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    caches = _caches(gen, layers, sum(need) + 2, page, heads, dim, dtype, layout)
    want = [tuple(c.cpu().clone() for c in pair) for pair in caches]
    starts, lengths = torch.tensor(starts_of(sizes)), torch.tensor([c + n for c, n in zip(cached, sizes)])
    left = compact_walk(want, table, starts, lengths, path, kept)
    print(f"compaction of wide tokens {dtype} layers={layers} {heads}x{dim} {layout} {kind}", flush=True)
    got = paged_compact(caches, table.cuda(), starts.cuda(), lengths.cuda(), path.cuda(), i32(kept))
    assert got.tolist() == left
    _same(caches, want)
