"""Draft trees, their verification, compaction and forks (tjev_amd.drafts, tjev_amd.paged) against their plain forms
(tests/draft_cases.py), at the sizes and values where they can go wrong."""

from __future__ import annotations

import math
import random

import pytest
import torch

from draft_cases import bits_of, compact_walk, fork_walk, random_tree, starts_of, tree_walk, verify_walk

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------- the tree
@pytest.mark.parametrize("kind", ["tree", "chain", "star", "any", "roots"])
@pytest.mark.parametrize("sizes,max_new,front,behind", [
    ([1], 1, 0, 0), ([5, 0, 1, 17], 17, 0, 3), ([64, 63, 65, 2], 65, 2, 1), ([200, 128, 129, 1], 200, 0, 0), ([40, 9, 30], 12, 1, 2),
    ([300], 64, 0, 5), ([3] * 700, 3, 0, 0), ([700], 1000, 0, 0),
])
def test_tree(kind, sizes, max_new, front, behind):
    from tjev_amd import draft_tree

    rng = random.Random(len(sizes))
    parents = [7] * front + [p for n in sizes for p in random_tree(rng, n, kind)[:n]] + [7] * behind
    starts = starts_of(sizes, front)
    lengths = [n + rng.choice([0, 1, 50, 2 ** 20, 2 ** 31 - 1 - n]) for n in sizes]
    want, pos = tree_walk(parents, starts, lengths, max_new)
    dt = torch.int64 if len(sizes) % 2 else torch.int32
    print(f"tree {kind} {sizes[:5]} max_new={max_new}", flush=True)
    t = draft_tree(i32(parents).to(dt), i32(starts).to(dt), i32(lengths).to(dt), max_new=max_new)
    assert torch.equal(t.ancestors.cpu(), bits_of(want, -(-max_new // 64)))
    assert t.positions.tolist() == pos


def test_tree_of_any_starts():
    """Starts and lengths that hold anything: nothing outside the batch is touched, what lies within is as the walk has it."""
    from tjev_amd import draft_tree

    parents = [i - 1 for i in range(12)]
    for starts, lengths in (([-5, 4, 99], [3, 200]), ([6, 2, 12], [0, 10]), ([0, 0, 0], [0, 0]), ([2 ** 31 - 1, 3, 5], [-4, 2])):
        print(f"tree of starts {starts}", flush=True)
        t = draft_tree(i32(parents), i32(starts), i32(lengths), max_new=20)
        want, pos = tree_walk(parents, starts, lengths, 20)
        assert torch.equal(t.ancestors.cpu(), bits_of(want, 1)) and t.positions.tolist() == pos


def test_tree_positions_of_far_parents():
    """int64 parents past 32 bits are none, and not what their low half says."""
    from tjev_amd import draft_tree

    t = draft_tree(torch.tensor([-1, 2 ** 32, -2 ** 32, 2 ** 40 + 1], device="cuda"), i32([0, 4]), i32([9]), max_new=4)
    assert t.ancestors.flatten().tolist() == [1, 2, 4, 8] and t.positions.tolist() == [5] * 4


def test_no_drafts():
    from tjev_amd import draft_tree, verify_drafts

    t = draft_tree(i32([]), i32([0, 0, 0]), i32([4, 0]), max_new=3)
    assert t.ancestors.shape == (0, 1) and t.positions.shape == (0,)
    e = torch.empty(0, 11, device="cuda")
    v = verify_drafts(i32([]), e, i32([0, 0, 0]), torch.empty(0, device="cuda"), max_new=3)
    assert v.kept.tolist() == [0, 0] and v.tokens.tolist() == v.path.tolist() == [[-1] * 3] * 2


# ---------------------------------------------------------------- verification
def _verify(rng, sizes, vocab, kind, dtype, drawn, sharp=2.0, front=0, behind=0):
    gen = torch.Generator().manual_seed(vocab + len(sizes))
    n = front + sum(sizes) + behind
    target = torch.softmax(sharp * torch.randn(n, vocab, generator=gen), -1)
    starts = starts_of(sizes, front)
    parents = [-1] * front + [p for k in sizes for p in random_tree(rng, k, kind)[:k]] + [-1] * behind
    tokens, draft = torch.randint(0, vocab, (n,), generator=gen), None
    for b, k in enumerate(sizes):  # likely tokens behind each parent, some of them twice
        for i in range(1, k):
            p = parents[starts[b] + i]
            if 0 <= p < i:
                top = torch.topk(target[starts[b] + p], min(4, vocab)).indices
                tokens[starts[b] + i] = top[rng.randrange(len(top))]
    if drawn:
        above = torch.arange(n) - 1
        draft = torch.softmax(torch.log(target[above.clamp(min=0)].clamp(min=1e-30)) + 0.8 * torch.randn(n, vocab, generator=gen), -1)
        tokens = torch.multinomial(draft, 1, generator=gen)[:, 0]
        draft = draft.to(dtype)
    u = torch.rand(n, generator=gen)
    return dict(tokens=tokens, target_probs=target.to(dtype), starts=torch.tensor(starts), uniforms=u,
                parents=None if kind == "chain" else torch.tensor(parents), draft_probs=draft)


def _check(case, max_new):
    from tjev_amd import verify_drafts

    v = verify_drafts(**{n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in case.items()}, max_new=max_new)
    out, path, kept = verify_walk(case["tokens"], case["target_probs"], case["starts"], case["uniforms"], case["parents"], case["draft_probs"],
                                  max_new)
    assert v.kept.tolist() == kept and v.path.tolist() == path and v.tokens.tolist() == out
    return v


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kind,drawn", [("tree", False), ("star", False), ("any", False), ("chain", False), ("chain", True)])
@pytest.mark.parametrize("sizes,vocab,max_new", [
    ([1], 1, 1), ([6, 1, 0, 3, 9], 7, 9), ([12] * 40, 33, 12), ([30, 64, 65, 130], 50, 130), ([9, 20, 5], 5003, 6), ([4, 7], 70001, 7),
    ([2], 4096, 2), ([3, 3], 4097, 3), ([5], 1100001, 5),
])
def test_verify(dtype, kind, drawn, sizes, vocab, max_new):
    print(f"verify {dtype} {kind} drawn={drawn} {sizes[:4]} vocab={vocab} max_new={max_new}", flush=True)
    case = _verify(random.Random(vocab), sizes, vocab, kind, dtype, drawn, front=1, behind=2)
    v = _check(case, max_new)
    if len(sizes) == 40:  # some paths end at once, some go on
        assert int(v.kept.min()) == 1 and int(v.kept.max()) > 1


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kind,drawn", [("tree", False), ("chain", False), ("chain", True)])
@pytest.mark.parametrize("requests,vocab", [(257, 1), (300, 6), (256, 33), (261, 1025), (270, 5000)])
def test_verify_many(dtype, kind, drawn, requests, vocab):
    """More requests than are verified by a workgroup each, of small vocabularies too."""
    rng = random.Random(requests + vocab)
    sizes = [rng.choice([0, 1, 1, 2, 3, 5]) for _ in range(requests)]
    print(f"verify {dtype} {kind} drawn={drawn} {requests} requests vocab={vocab}", flush=True)
    _check(_verify(rng, sizes, vocab, kind, dtype, drawn, front=2, behind=1), 4)


@pytest.mark.parametrize("dtype,drawn,vocab", [(F32, True, 32768), (F32, True, 32769), (F32, False, 65536), (BF, True, 65536), (BF, False, 65537)])
def test_verify_at_the_largest_rows_of_a_launch(dtype, drawn, vocab):
    print(f"verify {dtype} drawn={drawn} vocab={vocab}", flush=True)
    _check(_verify(random.Random(vocab), [3, 1, 4], vocab, "chain" if drawn else "tree", dtype, drawn, front=0, behind=0), 4)


@pytest.mark.parametrize("drawn", [False, True])
def test_verified_tokens_have_the_targets_distribution(drawn):
    """A grid of numbers for the draft and for the drawn token: the first emitted token has the target's probabilities up to the grid's
    step, whatever the draft. A column of the grid is off by a cell at the border of its acceptance and one at each end of its part of the running
    sum: three steps."""
    from tjev_amd import verify_drafts

    vocab, m = 6, 150
    gen = torch.Generator().manual_seed(3)
    p, q = (torch.softmax(1.5 * torch.randn(vocab, generator=gen), -1) for _ in range(2))
    got = torch.zeros(vocab, dtype=torch.float64)
    grid = (torch.arange(m) + 0.5) / m
    for x in range(vocab if drawn else 1):  # drawn: every draft, with its probability; chosen: always token 2
        u = torch.stack(torch.meshgrid(grid, grid, indexing="ij"), -1).view(-1, 2)
        n = u.shape[0]
        tokens = torch.tensor([0, x if drawn else 2]).repeat(n)
        target, draft = p.repeat(2 * n, 1).cuda(), q.repeat(2 * n, 1).cuda() if drawn else None
        print(f"distribution of a verified token drawn={drawn} draft={x}", flush=True)
        v = verify_drafts(tokens.cuda(), target, (2 * torch.arange(n + 1)).cuda(), u.flatten().cuda(), draft_probs=draft, max_new=2)
        first = torch.bincount(v.tokens[:, 0].cpu().long(), minlength=vocab).double() / n
        got += first * (float(q[x]) if drawn else 1.0)
    assert float((got - p.double()).abs().max()) < 3 / m


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", [300, 66000])
def test_verify_degenerate_rows(dtype, vocab):
    """Rows without a positive number, NaN, infinities and negative numbers, a draft like the target, tokens outside the vocabulary,
    the same token twice among siblings, numbers of 0, 1, over 1, below 0 and NaN."""
    nan, inf = math.nan, math.inf
    base = torch.softmax(torch.randn(vocab, generator=torch.Generator().manual_seed(1)), -1)
    one = torch.zeros(vocab)
    one[17] = 1.0
    odd = base.clone()
    odd[[3, 50, 99]] = torch.tensor([nan, inf, -1.0])
    for name, row in (("plain", base), ("zeros", torch.zeros(vocab)), ("nan", torch.full((vocab,), nan)), ("one", one), ("odd", odd),
                      ("tiny", base * 1e-38)):
        for u0 in (0.0, 0.3, 1.0, 7.0, -1.0, nan)[::1 if vocab < 1000 else 2]:
            for up, x in (([-1, 0, 0, 0, 1], [0, 17, 17, 5, 9]), ([-1, 0, 0, 0, 0], [0, -1, vocab, 2 ** 31 - 1, 17]), ([-1, -1, 1, 0, 3], [0, 3, 17, 50, 99])):
                u = torch.tensor([u0, 0.9999, 0.5, 0.01, 0.2])
                case = dict(tokens=torch.tensor(x), target_probs=row.repeat(5, 1).to(dtype), starts=torch.tensor([0, 5]), uniforms=u,
                            parents=torch.tensor(up), draft_probs=None)
                _check(case, 5)
            case = dict(tokens=torch.tensor([0, 17, 3, 9, 2 ** 40 + 17]), target_probs=row.repeat(5, 1).to(dtype), starts=torch.tensor([0, 5]),
                        uniforms=torch.tensor([u0, 0.2, 0.9, 0.9999, 0.0]), parents=None, draft_probs=None)
            _check(case, 5)
            for draft in (base, one, odd, torch.zeros(vocab), row):  # a draft of its own numbers leaves nothing
                print(f"verify {dtype} rows={name} u={u0}", flush=True)
                _check(dict(case, draft_probs=draft.repeat(5, 1).to(dtype)), 5)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bits", [14, 16, 17, 21])
def test_verify_borders(dtype, bits):
    """Powers of two, whose sums are exact: numbers on the border of a token take the next one, at both sides of a part's end."""
    vocab = 1 << bits
    row = torch.full((1, vocab), 2.0 ** -bits, dtype=dtype)
    ks = [0, 1, 2, 255, 256, 1023, 1024, 1025, 4094, 4095, 4096, 4097, 8191, 8192, 12288, vocab // 2, vocab // 2 + 1, vocab - 1]
    us = [k * 2.0 ** -bits for k in ks]
    print(f"verify borders {dtype} vocab={vocab}", flush=True)
    from tjev_amd import verify_drafts

    v = verify_drafts(torch.zeros(len(ks), dtype=torch.int32, device="cuda"), row.cuda().expand(len(ks), vocab), torch.arange(len(ks) + 1).cuda(),
                      torch.tensor(us).cuda(), max_new=1)
    assert v.tokens[:, 0].tolist() == ks
    below = torch.nextafter(torch.tensor(us[1:]), torch.tensor(0.0))
    v = verify_drafts(torch.zeros(len(below), dtype=torch.int32, device="cuda"), row.cuda().expand(len(below), vocab),
                      torch.arange(len(below) + 1).cuda(), below.cuda(), max_new=1)
    assert v.tokens[:, 0].tolist() == [k - 1 for k in ks[1:]]


@pytest.mark.parametrize("dtype", [BF, F32])
def test_verify_strides(dtype):
    """Rows of a wider tensor that start on any element, and a last dim that is not contiguous."""
    case = _verify(random.Random(5), [5, 3, 8], 4999, "chain", dtype, True)
    want = _check(case, 8)
    from tjev_amd import verify_drafts

    for off in (1, 3):
        views = {}
        for n in ("target_probs", "draft_probs"):
            wide = torch.full((16, 5011), math.nan, dtype=dtype, device="cuda")
            views[n] = wide[:, off:off + 4999]
            views[n].copy_(case[n])
        print(f"verify strided {dtype} off={off}", flush=True)
        dev = {n: x.cuda() for n, x in case.items() if isinstance(x, torch.Tensor)}
        for kw in (views, {n: x.cuda().t().contiguous().t() for n, x in case.items() if n in views}):
            v = verify_drafts(**{**dev, **kw}, max_new=8)
            assert all(torch.equal(a, b) for a, b in zip(v, want))


def test_verify_of_far_rows():
    """Probabilities past 2^32 bytes and 2^31 elements from the first."""
    from tjev_amd import verify_drafts

    vocab = 200001
    n = 11000
    print("verify past 2^31 elements", flush=True)
    p = torch.zeros(n, vocab, dtype=BF, device="cuda")
    assert p.numel() > 2 ** 31
    p[n - 2, 7], p[n - 1, 199999] = 1.0, 1.0
    tokens = torch.zeros(n, dtype=torch.int32, device="cuda")
    tokens[n - 1] = 7
    v = verify_drafts(tokens, p, i32([n - 2, n]), torch.full((n,), 0.5, device="cuda"), max_new=2)
    assert v.tokens.tolist() == [[7, 199999]] and v.path.tolist() == [[0, 1]] and v.kept.tolist() == [2]


# ---------------------------------------------------------------- compaction
def _caches(gen, layers, pages, page, heads, dim, dtype, layout="plain"):
    out = []
    for _ in range(layers):
        if layout == "heads first":
            out.append(tuple(torch.randn(pages, heads, page, dim, generator=gen).to(dtype).cuda().transpose(1, 2) for _ in range(2)))
        elif layout == "joint":
            out.append(torch.randn(pages, 2, page, heads, dim, generator=gen).to(dtype).cuda().unbind(1))
        elif layout == "odd":
            out.append(tuple(torch.randn(pages * page * heads * dim + 1, generator=gen).to(dtype).cuda()[1:].view(pages, page, heads, dim)
                             for _ in range(2)))
        else:
            out.append(tuple(torch.randn(pages, page, heads, dim, generator=gen).to(dtype).cuda() for _ in range(2)))
    return out


def _same(caches, want):
    for pair, cpu in zip(caches, want):
        for c, w in zip(pair, cpu):
            assert torch.equal(c.cpu(), w)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("layers,heads,dim,page,layout", [(1, 2, 64, 16, "plain"), (3, 1, 8, 3, "heads first"), (2, 3, 20, 5, "joint"),
                                                          (18, 2, 16, 8, "plain"), (2, 5, 7, 1, "odd"), (1, 16, 256, 24, "plain")])
@pytest.mark.parametrize("kind", ["tree", "all", "last", "every second", "none"])
def test_compact(dtype, layers, heads, dim, page, layout, kind):
    """Moves over places that other moves read: a request's tokens shifted by one, every second one, and up to the last."""
    from tjev_amd import paged_compact

    rng = random.Random(dim)
    gen = torch.Generator().manual_seed(dim)
    sizes = [1, 9, 0, 70, 16, 200]
    cached = [5, 0, 31, 2, 16, 100]
    path = torch.full((len(sizes), 200), -1, dtype=torch.int32)
    kept = []
    for b, n in enumerate(sizes):
        way = {"tree": sorted(rng.sample(range(n), min(n, rng.randint(1, 12)))), "all": list(range(n)), "last": list(range(1, n)),
               "every second": list(range(0, n, 2)), "none": []}[kind]
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
    print(f"compact {dtype} layers={layers} {heads}x{dim} page={page} {layout} {kind}", flush=True)
    got = paged_compact(caches, table.cuda(), starts.cuda(), lengths.cuda(), path.cuda(), i32(kept))
    assert got.tolist() == left == [c + k for c, k in zip(cached, kept)]
    _same(caches, want)


def test_compact_of_anything():
    """Numbers that are no new token or less than their place, kept over what there is, missing pages, lengths shorter than the new tokens
    or past the table: left out, and nothing outside is touched."""
    from tjev_amd import paged_compact

    gen = torch.Generator().manual_seed(2)
    table = torch.tensor([[0, 1, -1, 3], [4, 99, 5, 6], [7, -7, 8, 9], [10, 11, 12, 13], [14, 15, 16, 17]], dtype=torch.int32)
    path = torch.tensor([[0, 3, 5, 200, -9], [2, 2 ** 31 - 1, 3, 4, 5], [1, 0, 1, 9, 20], [4, 5, 6, 7, 8], [1, 2, 3, 4, 5]], dtype=torch.int32)
    kept, starts, lengths = [5, 99, 4, -3, 5], [0, 10, 20, 30, 40, 50], [14, 16, 12, 12, 4]
    caches = _caches(gen, 2, 18, 4, 2, 8, F32)
    want = [tuple(c.cpu().clone() for c in pair) for pair in caches]
    left = compact_walk(want, table, starts, lengths, path, kept)
    print("compact of anything", flush=True)
    got = paged_compact(caches, table.cuda(), i32(starts).long(), i32(lengths).long(), path.cuda().long(), i32(kept).long())
    assert got.tolist() == left
    _same(caches, want)
    assert paged_compact([], table.cuda(), i32(starts), i32(lengths), path.cuda(), i32(kept)).tolist() == left


# ---------------------------------------------------------------- forks
def _pool(rng, lens, page, width, extra, common=0):
    """A table of requests with their pages in random order, some of them starting with the same `common` pages; the list and counts
    that go with it."""
    need = [min(width, -(-n // page)) for n in lens]
    order = list(range(sum(need) + extra))
    rng.shuffle(order)
    table, shared, at = [], [0] * len(order), 0
    for b, k in enumerate(need):
        row = order[at:at + k]
        at += k
        if b and common and rng.random() < 0.5 and min(lens[0], lens[b]) // page >= common:
            order.extend(row[:common]), row.__setitem__(slice(0, common), table[0][:common])
            for p in row[:common]:
                shared[p] += 1
        table.append(row + [-1] * (width - k))
    held = {p for row in table for p in row if p >= 0}
    rest = [p for p in dict.fromkeys(order) if p not in held]
    list_ = [0] * len(held) + rest
    return table, list_, len(held), shared


def _fork(caches, table, lens, sources, keep, free, taken, shared, page, dt=torch.int32):
    from tjev_amd import paged_fork

    want_caches = [tuple(c.cpu().clone() for c in pair) for pair in caches]
    want = fork_walk(want_caches, table, lens, sources, keep, free, taken, shared, page)
    given = [i32(x) for x in (table, lens, sources, free, [taken], shared)]
    before = [x.clone() for x in given]
    f = paged_fork(caches, given[0], given[1].to(dt), given[2].to(dt), None if keep is None else i32(keep).to(dt), given[3], given[4], given[5],
                   page_size=page)
    assert f.block_table.tolist() == want[0] and f.lengths.tolist() == want[1]
    assert f.free_pages.tolist() == want[2] and int(f.taken) == want[3] and f.shared.tolist() == want[4]
    _same(caches, want_caches)
    assert all(torch.equal(x, y) for x, y in zip(given, before))
    return f


@pytest.mark.parametrize("dtype,layers,heads,dim,layout", [(BF, 2, 2, 64, "plain"), (F32, 1, 3, 20, "heads first"), (BF, 17, 1, 8, "plain"),
                                                           (BF, 1, 5, 7, "odd"), (F32, 2, 4, 256, "joint"), (BF, 0, 1, 8, "plain")])
@pytest.mark.parametrize("kind", ["same", "roll back", "samples", "beams", "end", "dense", "mixed"])
@pytest.mark.parametrize("page", [1, 16, 24])
def test_fork(dtype, layers, heads, dim, layout, kind, page):
    rng = random.Random(f"{kind} {page}")
    lens = [rng.randint(0, 9 * page) for _ in range(12)] + [3 * page, 3 * page + 1]
    n = len(lens)
    sources = {"same": list(range(n)), "roll back": list(range(n)), "samples": [b for b in range(n) for _ in range(1 + b % 4)],
               "beams": [rng.randrange(n) for _ in range(n)], "end": [-1] * n, "dense": [b for b in range(n) if b % 3], "mixed":
               [rng.choice([-1, 0, 3, 3, 7, n, 2 ** 31 - 1, rng.randrange(n)]) for _ in range(25)]}[kind]
    keep = None if kind in ("same", "samples") else [max(0, lens[b] - rng.choice([0, 1, page, 2 * page + 1])) if 0 <= b < n else 5 for b in sources]
    if kind == "mixed":
        keep = [rng.choice([k, -3, 10 ** 6]) for k in keep]
    table, free, taken, shared = _pool(rng, lens, page, 10, 60, common=2)
    caches = _caches(torch.Generator().manual_seed(dim), layers, len(shared), page, heads, dim, dtype, layout)
    print(f"fork {dtype} layers={layers} {heads}x{dim} {layout} {kind} page={page}", flush=True)
    _fork(caches, table, lens, sources, keep, free, taken, shared, page, torch.int64 if layers == 1 else torch.int32)


@pytest.mark.parametrize("requests,new,width,page", [(1, 1, 1, 16), (1, 64, 40, 4), (300, 700, 20, 8), (2000, 1500, 3, 5), (8192, 8192, 2, 2),
                                                     (3, 2, 3000, 1)])
def test_fork_of_many(requests, new, width, page):
    rng = random.Random(requests)
    lens = [rng.randint(0, width * page) for _ in range(requests)]
    sources = [rng.randrange(-1, requests) for _ in range(new)]
    keep = [rng.randint(0, width * page) for _ in range(new)]
    table, free, taken, shared = _pool(rng, lens, page, width, new, common=1)
    print(f"fork of {requests} places into {new}", flush=True)
    _fork([], table, lens, sources, keep, free, taken, shared, page)


@pytest.mark.parametrize("requests,new,width,page", [
    (64, 1000, 4, 4), (1000, 64, 4, 4), (16, 3, 256, 1), (1, 2, 2048, 1), (1024, 1024, 4, 3), (5, 1, 819, 2), (64, 1000, 65, 4), (1000, 64, 65, 4),
    (16, 3, 4096, 1), (1, 2, 20000, 1), (1024, 1024, 64, 3), (1025, 9, 4, 3), (70, 70, 300, 2),
])
@pytest.mark.parametrize("kind", ["end", "any", "twice", "all kept"])
def test_fork_of_many_pages(requests, new, width, page, kind):
    """Pages given back and shared by the thousand, in and past what one workgroup does."""
    rng = random.Random(requests + new)
    lens = [rng.randint(width * page // 2, width * page) for _ in range(requests)]
    sources = [-1 if kind == "end" and i % 9 else rng.randrange(-1, requests) if kind == "any" else i // 2 % requests for i in range(new)]
    keep = None if kind == "all kept" else [rng.randint(0, width * page) for _ in range(new)]
    table, free, taken, shared = _pool(rng, lens, page, width, new, common=3)
    print(f"fork of {requests} places into {new} of {width} pages, {kind}", flush=True)
    _fork([], table, lens, sources, keep, free, taken, shared, page)


def test_fork_writes_back_and_forth():
    """Steps of forks, growth, roll backs into shared pages and ends, over one list: every page is held or on the list, once, and everybody
    reads the tokens that were written for them."""
    from tjev_amd import paged_append, paged_fork, paged_tables

    rng, page, width, pages = random.Random(4), 4, 12, 120
    kc = torch.zeros(pages, page, 1, 8, device="cuda")
    vc = torch.zeros_like(kc)
    table = torch.full((8, width), -1, dtype=torch.int32, device="cuda")
    free, taken, shared = torch.randperm(pages).int().cuda(), i32([0]), i32([0] * pages)
    texts, lengths, stamp = [[] for _ in range(8)], i32([0] * 8), 0
    for step in range(40):
        print(f"fork step {step}", flush=True)
        new = [min(rng.randint(0, 6), width * page - len(t)) for t in texts]
        t = paged_tables(lengths, i32(new), table, free, taken, page_size=page, tokens=sum(new) + 1)
        marks = list(range(stamp + 1, stamp + sum(new) + 1))
        stamp += len(marks)
        rows = torch.tensor(marks + [0], dtype=torch.float32, device="cuda")[:, None, None].expand(-1, 1, 8)
        paged_append(rows, -rows, kc, vc, t.slots)
        at = 0
        for b, n in enumerate(new):
            texts[b] = texts[b] + marks[at:at + n]
            at += n
        sources = [rng.choice([b, b, b, rng.randrange(8), -1]) for b in range(8)]
        keep = [rng.choice([10 ** 6, max(0, len(texts[b]) - rng.randint(0, 9))]) if b >= 0 else 0 for b in sources]
        f = paged_fork([(kc, vc)], t.block_table, t.lengths, i32(sources), i32(keep), free, t.taken, shared, page_size=page)
        texts = [texts[b][:k] if b >= 0 else [] for b, k in zip(sources, keep)]
        table, lengths, free, taken, shared = f
        assert lengths.tolist() == [len(x) for x in texts]
        held = {}
        for b, text in enumerate(texts):
            for j, x in enumerate(text):
                p = int(table[b, j // page])
                assert float(kc[p, j % page, 0, 0]) == x and float(vc[p, j % page, 0, 7]) == -x
            for p in table[b].tolist():
                if p >= 0:
                    held[p] = held.get(p, 0) + 1
        assert [held.get(p, 1) - 1 for p in range(pages)] == shared.tolist()
        rest = free[int(taken):].tolist()
        assert len(set(rest)) == len(rest) and not set(rest) & set(held) and len(rest) + len(held) == pages


def test_fork_without_room():
    """Copies that find the list at its end get -1; pages given back are the first to be taken; a list without room loses them."""
    c = lambda: _caches(torch.Generator().manual_seed(1), 1, 6, 4, 1, 8, F32)  # noqa: E731
    print("fork without room", flush=True)
    f = _fork(c(), [[0, 1]], [6], [0, 0, 0, 0], None, [0, 1, 5], 2, [0] * 6, 4)
    assert f.block_table.tolist() == [[0, 1], [0, 5], [0, -1], [0, -1]] and int(f.taken) == 5
    f = _fork(c(), [[0, 1], [2, 3]], [6, 8], [0, 0, 0], None, [0, 1, 2, 3], 4, [0] * 6, 4)
    assert f.block_table.tolist() == [[0, 1], [0, 2], [0, 3]] and int(f.taken) == 4
    f = _fork(c(), [[0, 1], [2, 3]], [8, 8], [-1], None, [9, 9], 1, [0] * 6, 4)
    assert f.free_pages.tolist() == [0, 9] and int(f.taken) == 0
    _fork(c(), [[0, 1], [2, 3]], [8, 7], [1, 1, 0], [7, 6, 5], [9, -1, 4], 2, [0] * 6, 4)
    _fork([], [[0, 1], [2, 3]], [8, 7], [1, 1, 0], [7, 6, 5], [], 0, [0] * 6, 4)


# ---------------------------------------------------------------- the calls
def _calls():
    """Each operator's call with its outputs as a list, on inputs of a few requests."""
    from tjev_amd import draft_tree, paged_compact, paged_fork, verify_drafts

    rng = random.Random(8)
    sizes = [7, 70, 0, 12]
    starts, lengths = i32(starts_of(sizes)), i32([n + 9 for n in sizes])
    parents = i32([p for n in sizes for p in random_tree(rng, n)[:n]])
    case = {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in _verify(random.Random(9), sizes, 9001, "tree", F32, False).items()}
    drawn = {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in _verify(random.Random(9), sizes, 9001, "chain", BF, True).items()}
    large = {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in _verify(random.Random(9), sizes, 70001, "tree", BF, False).items()}
    large_drawn = {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in _verify(random.Random(9), sizes, 70001, "chain", F32, True).items()}
    lens = [30, 11, 64, 90]
    table, free, taken, shared = _pool(rng, lens, 8, 12, 20, common=1)
    given = [i32(x) for x in (table, lens, [0, 0, 1, 3, 3, 3], [30, 29, 5, 90, 88, 3], free, [taken], shared)]
    base = _caches(torch.Generator().manual_seed(5), 2, len(shared), 8, 2, 64, BF)

    def fork(*_):
        caches = [tuple(c.clone() for c in pair) for pair in base]
        f = paged_fork(caches, *given, page_size=8)
        return [*f, *(c for pair in caches for c in pair)]

    many = [rng.randint(0, 40) for _ in range(1500)]
    table, free, taken, shared = _pool(rng, many, 4, 10, 900, common=1)
    given_many = [i32(x) for x in (table, many, [rng.randrange(-1, 1500) for _ in range(1200)], [rng.randint(0, 40) for _ in range(1200)], free, [taken],
                                   shared)]
    small = _caches(torch.Generator().manual_seed(6), 1, len(shared), 4, 1, 8, BF)

    def fork_many(*_):
        caches = [tuple(c.clone() for c in pair) for pair in small]
        return [*paged_fork(caches, *given_many, page_size=4), *caches[0]]

    path = i32([[0, 2, 3, -1], [0, 3, 6, 7], [-1] * 4, [0, 1, 2, 10]])
    kept = i32([3, 4, 0, 4])
    wide = i32([table[b][:11] for b in range(4)])

    def compact(*_):
        caches = [tuple(c.clone() for c in pair) for pair in base]
        return [paged_compact(caches, wide, starts, lengths, path, kept), *(c for pair in caches for c in pair)]

    return {"tree": lambda: list(draft_tree(parents, starts, lengths, max_new=70)), "verify": lambda: list(verify_drafts(**case, max_new=70)),
            "drawn": lambda: list(verify_drafts(**drawn, max_new=70)), "verify, large": lambda: list(verify_drafts(**large, max_new=70)),
            "drawn, large": lambda: list(verify_drafts(**large_drawn, max_new=70)), "fork": fork, "fork, many": fork_many, "compact": compact}


@pytest.mark.parametrize("what", ["tree", "verify", "drawn", "verify, large", "drawn, large", "fork", "fork, many", "compact"])
def test_calls_at_once_and_captured(monkeypatch, what):
    """Calls on two streams without a wait, captured ones replayed with eager work between, poisoned workspaces and LDS: the same bits."""
    from tjev_amd import _lib

    call = _calls()[what]
    print(f"calls of {what}", flush=True)
    want = [x.clone() for x in call()]
    same = lambda got: all(torch.equal(a, b) for a, b in zip(got, want))  # noqa: E731
    monkeypatch.setenv("TJEV_GDN_POISON", "1")
    assert same(call())
    monkeypatch.delenv("TJEV_GDN_POISON")
    with _lib.library(_lib.LDS_POISON_PATH):
        assert same(call())
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(call())
    torch.cuda.synchronize()
    assert all(same(g) for g in got)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = call()
        graphs.append((g, y))
    for _ in range(3):
        for _, y in graphs:
            for x in y:
                x.zero_()
        call()
        torch.cuda.synchronize()
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(same(y) for _, y in graphs)
