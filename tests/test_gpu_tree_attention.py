"""Attention for trees of drafted tokens over the paged cache (tjev_amd.paged_tree_attention) against its plain 64-bit form
(tests/draft_cases.py), and a drafted step from its tables to the next one's."""

from __future__ import annotations

import math
import random

import pytest
import torch

from draft_cases import bits_of, random_tree, starts_of, tree_attention64, tree_walk
from paged_cases import attention64, batch, compare

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
NAMES = ("q", "k_cache", "v_cache", "block_table", "starts", "lengths", "ancestors")


def _case(seed, lens, kind="tree", words=None, **kw):
    case = batch(torch.Generator().manual_seed(seed), lens, **kw)
    rng = random.Random(seed)
    parents = [p for _, n in lens for p in random_tree(rng, n, kind)[:n]]
    most = max(1, max(n for _, n in lens))
    sets, _ = tree_walk(parents, case["starts"].tolist(), case["lengths"].tolist(), most)
    sets += [set()] * (case["q"].shape[0] - len(sets))
    case["ancestors"] = bits_of(sets, words or -(-most // 64))
    return case


def _attend(case, **kw):
    from tjev_amd import paged_tree_attention

    return paged_tree_attention(**{n: x.cuda() if isinstance(x, torch.Tensor) and not x.is_cuda else x for n, x in {**case, **kw}.items()})


LENS = {
    "one": [(0, 1)], "small": [(31, 5), (0, 3), (64, 2), (200, 4), (16, 1)], "ragged": [(40, 17), (0, 0), (3, 1), (0, 33), (70, 1), (0, 0)],
    "wide": [(130, 150), (5, 64)], "words": [(100, 129), (63, 65), (1, 200)],
}


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [
    (4, 1, 64, 16), (2, 2, 128, 24), (16, 4, 256, 16), (5, 1, 40, 5), (20, 1, 96, 64), (3, 3, 8, 1), (6, 2, 200, 48),
])
@pytest.mark.parametrize("lens", sorted(LENS))
@pytest.mark.parametrize("kind", ["tree", "star"])
def test_tree_attention(dtype, heads, kv_heads, dim, page, lens, kind):
    """Every place of the cache that no token has holds NaN; rows behind the last request come back 0."""
    print(f"tree attention {dtype} heads={heads}/{kv_heads} dim={dim} page={page} {lens} {kind}", flush=True)
    case = _case(dim, LENS[lens], kind, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, pad_rows=3, gate=len(lens) % 2 == 0)
    want, room = tree_attention64(*(case[n] for n in NAMES), gate=case["gate"])
    got = _attend(case, max_new=max(n for _, n in LENS[lens]) if kind == "star" else None)
    compare(got, want, room)
    assert bool((got[-3:] == 0).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,lens", [(4, 2, 64, [(40, 17), (0, 5), (90, 70)]), (16, 4, 256, [(300, 9), (20, 40)]),
                                                     (8, 2, 128, [(0, 200), (77, 3)])])
def test_a_chain_is_causal(dtype, heads, kv_heads, dim, lens):
    """The rows of a chain are paged_attention's."""
    print(f"chains {dtype} {heads}/{kv_heads} of {dim} {lens}", flush=True)
    case = _case(3, lens, "chain", heads=heads, kv_heads=kv_heads, dim=dim, page=16, dtype=dtype, gate=True)
    want, room = attention64(*(case[n] for n in NAMES[:-1]), gate=case["gate"])
    compare(_attend(case), want, room)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads", [4, 24])
@pytest.mark.parametrize("words", [1, 2, 3])
def test_rows_may_name_any_token(dtype, heads, words):
    """Bits at random: tokens behind a row's own, not its own, none at all; more words than tokens, and fewer."""
    lens = [(0, 40), (30, 130), (0, 3), (17, 64), (64, 1)]
    case = _case(4, lens, heads=heads, kv_heads=2, dim=64, page=16, dtype=dtype, pad_rows=1)
    gen = torch.Generator().manual_seed(words)
    case["ancestors"] = torch.randint(-2 ** 63, 2 ** 63 - 1, (case["q"].shape[0], words), generator=gen)
    case["ancestors"][::7] = 0
    case["ancestors"][3::7] = -1
    print(f"any tokens {dtype} heads={heads} words={words}", flush=True)
    want, room = tree_attention64(*(case[n] for n in NAMES))
    got = _attend(case)
    compare(got, want, room)
    assert bool((got[::7][:3] == 0).all())  # rows of the first request without keys


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,lens,requests", [
    (8, 2, 64, [(700, 6), (0, 1), (90, 40)], 60), (16, 4, 256, [(1200, 64)], 64), (6, 3, 40, [(2000, 90), (5, 9)], 200),
    (4, 4, 200, [(77, 50), (1, 1)], 120), (16, 2, 128, [(4000, 3), (0, 200)], 9),
])
def test_unused_requests_and_the_most_new_tokens(dtype, heads, kv_heads, dim, lens, requests):
    """More places than trees, and bounds on a tree's tokens: the true one, none, and (which costs time alone) wrong ones."""
    case = _case(24, lens, heads=heads, kv_heads=kv_heads, dim=dim, page=16, dtype=dtype, gate=True)
    want, room = tree_attention64(*(case[n] for n in NAMES), gate=case["gate"])
    starts, lengths = torch.zeros(requests + 1, dtype=torch.int32), torch.zeros(requests, dtype=torch.int32)
    table = torch.full((requests, case["block_table"].shape[1]), -1, dtype=torch.int32)
    for b in range(len(lens)):
        at = b * (requests - 1) // max(1, len(lens) - 1)
        starts[at + 1:] = case["starts"][b + 1]
        lengths[at], table[at] = case["lengths"][b], case["block_table"][b]
    case.update(starts=starts, lengths=lengths, block_table=table)
    for max_new in (None, max(n for _, n in lens), 1, 5, 10 ** 6):
        print(f"tree attention {dtype} {heads}/{kv_heads} of {dim} {lens} in {requests} places, max_new={max_new}", flush=True)
        compare(_attend(case, max_new=max_new), want, room)


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(16, 4, 256, 16), (16, 4, 256, 64), (16, 4, 256, 24), (16, 4, 200, 16), (16, 4, 128, 32),
                                                     (24, 4, 64, 16)])
@pytest.mark.parametrize("longest", [128, 385, 900])
def test_many_trees_in_tiles_of_both_kinds(heads, kv_heads, dim, page, longest):
    """Trees of a few tokens beside ones of up to 40, more of them than are streamed; keys that end in the first and the second
    block of a pair, one key, and none."""
    rng = random.Random(longest + page)
    lens = [(rng.choice((0, 1, 127, 128, 129, 255, 256, 257, longest)) % (longest + 1), rng.choice((0, 1, 2, 4, 5, 9, 33, 40))) for _ in range(44)]
    print(f"many trees, {heads}/{kv_heads} of {dim}, page={page}, up to {longest} keys", flush=True)
    case = _case(longest, lens, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=BF, gate=dim == 256, pad_rows=2)
    want, room = tree_attention64(*(case[n] for n in NAMES), gate=case["gate"])
    compare(_attend(case), want, room)


def test_no_tokens():
    from tjev_amd import paged_tree_attention

    c = torch.zeros(2, 16, 2, 64, device="cuda")
    z = torch.zeros(3, dtype=torch.int32, device="cuda")
    table = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    got = paged_tree_attention(torch.empty(0, 4, 64, device="cuda"), c, c, table, z, z[:2], torch.empty(0, 1, dtype=torch.int64, device="cuda"))
    assert got.shape == (0, 4, 64)
    got = paged_tree_attention(torch.ones(5, 4, 64, device="cuda"), c, c, table, z, z[:2], torch.full((5, 1), -1, device="cuda"))
    assert bool((got == 0).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("page", [16, 10])
@pytest.mark.parametrize("heads", [4, 16])
def test_pages_that_are_none(dtype, page, heads):
    """Entries that are no page, lengths past the table's width or shorter than the new tokens."""
    case = _case(5, [(200, 4), (90, 20), (33, 1), (0, 7)], heads=heads, kv_heads=2, dim=64, page=page, dtype=dtype)
    t = case["block_table"]
    t[0, 1], t[0, 3], t[1, 0], t[2, :] = -1, case["k_cache"].shape[0], 2 ** 31 - 1, -2 ** 31
    case["lengths"][0] += 3000
    case["lengths"][3] = 4      # three of its seven tokens stand before the first
    t[0][t[0] == -1] = 10 ** 6
    print(f"tree attention over pages that are none {dtype} page={page} heads={heads}", flush=True)
    want, room = tree_attention64(*(case[n] for n in NAMES))
    compare(_attend(case), want, room)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lens,dim", [([(20, 40)], 64), ([(100, 3), (5, 30)], 128), ([(0, 150)], 256), ([(9, 100)], 64), ([(60, 4)], 256)])
def test_bad_values_reach_only_their_rows(dtype, lens, dim):
    """NaN and infinities in the keys and values of some new tokens: the rows that do not name them are as if they were not there."""
    case = _case(6, lens, heads=4, kv_heads=2, dim=dim, page=16, dtype=dtype)
    c, n = lens[-1]
    table, b = case["block_table"], len(lens) - 1
    at = lambda t: (int(table[b, t // 16]), t % 16)  # noqa: E731
    clean = _attend(case)
    bad = (n // 2, n - 2, n - 1)
    case["v_cache"][at(c + bad[0])][0, 3] = math.nan
    case["v_cache"][at(c + bad[1])][1, 5] = math.inf
    case["k_cache"][at(c + bad[2])][0, 2] = math.nan
    print(f"tree attention with bad values {dtype} {lens} dim={dim}", flush=True)
    got = _attend(case)
    first = int(case["starts"][b])
    free = [r for r in range(n) if not any(int(case["ancestors"][first + r, j // 64]) >> j % 64 & 1 for j in bad)]
    assert free and len(free) < n
    assert torch.equal(got[:first], clean[:first]) and all(torch.equal(got[first + r], clean[first + r]) for r in free)
    want, room = tree_attention64(*(case[x] for x in NAMES))
    compare(got, want, room)
    assert bool(torch.isnan(got[first + n - 1, :2]).all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_layouts_views_and_scales(dtype):
    """Caches with the heads before the places or keys beside values, q beside its gate, a given out whose rows of no request stay, rows in
    front, int64 lengths, a negative scale and 0."""
    from tjev_amd import paged_tree_attention

    case = _case(7, [(40, 3), (100, 40), (7, 1)], heads=4, kv_heads=2, dim=64, page=16, dtype=dtype, pad_rows=4, gate=True)
    case["starts"] += 2
    case["ancestors"] = case["ancestors"].roll(2, 0)
    for scale in (0.3, -0.2, 0.0):
        want, room = tree_attention64(*(case[n] for n in NAMES), scale, case["gate"])
        qg = torch.cat([case["q"], case["gate"]], -1).cuda()
        dev = {n: x.cuda() for n, x in case.items()}
        dev.update(q=qg[..., :64], gate=qg[..., 64:], starts=dev["starts"].long(), lengths=dev["lengths"].long(),
                   ancestors=torch.stack([dev["ancestors"]] * 2, 1)[:, 0])
        kc, vc = dev["k_cache"], dev["v_cache"]
        for name, (k, v) in {"plain": (kc, vc), "heads first": tuple(c.transpose(1, 2).contiguous().transpose(1, 2) for c in (kc, vc)),
                             "joint": tuple(torch.stack([kc, vc], 1).unbind(1))}.items():
            print(f"tree attention layout {name} {dtype} scale={scale}", flush=True)
            got = paged_tree_attention(**dict(dev, k_cache=k, v_cache=v), scale=scale)
            compare(got, want, room)
            wide = torch.full((got.shape[0], 4, 128), 7.0, dtype=dtype, device="cuda")
            out = wide[..., 64:]
            assert paged_tree_attention(**dict(dev, k_cache=k, v_cache=v), scale=scale, out=out) is out
            assert torch.equal(out[2:-2], got[2:-2]) and bool((out[:2] == 7).all()) and bool((out[-2:] == 7).all())
            assert bool((wide[..., :64] == 7).all())


# tiles whose keys one range holds or several, joined in each of the ways
SPLIT = {
    "streamed, few": ([(9000, 2)], 8, 2, 128, None), "streamed, many": ([(900, 2)] * 70, 8, 2, 128, None),
    "wide, few": ([(3000, 64)], 16, 4, 256, None), "wide, many": ([(1500, 70)] * 6, 16, 4, 128, None),
    "wide, counted": ([(3000, 64)] + [(0, 0)] * 63, 16, 4, 256, 64), "32 rows": ([(700, 5)] * 40, 8, 2, 64, 8),
    "32 rows, many": ([(50, 20)] * 40, 8, 8, 64, None), "small, streamed": ([(1500, 12)], 16, 4, 256, None),
}


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kind", sorted(SPLIT))
def test_long_contexts(monkeypatch, dtype, kind):
    """Many workgroups a tile, joined: right, the same bits twice, in the poison modes, on streams at once, and captured."""
    from tjev_amd import _lib

    lens, heads, kv_heads, dim, max_new = SPLIT[kind]
    case = _case(8, lens, heads=heads, kv_heads=kv_heads, dim=dim, page=16, dtype=dtype, gate=True)
    dev = dict({n: x.cuda() for n, x in case.items()}, max_new=max_new)
    print(f"long contexts: {kind} {dtype}", flush=True)
    got = _attend(dev)
    # a few requests against the plain form, each alone
    for b in (0, len(lens) // 2) if lens[-1][1] else (0,):
        s0, s1 = int(case["starts"][b]), int(case["starts"][b + 1])
        rows = sorted({s0, s0 + 1, (s0 + s1) // 2, s1 - 1})
        for r in rows:
            one = dict(case, q=case["q"][r:r + 1], gate=case["gate"][r:r + 1])
            # one row of the tree: its own keys as a batch of one whose table holds the named tokens alone, in their order
            first = int(case["lengths"][b]) - (s1 - s0)
            named = [j for j in range(s1 - s0) if int(case["ancestors"][r, j // 64]) >> j % 64 & 1]
            t = torch.tensor([*range(first), *(first + j for j in named)])
            page = case["block_table"][b].long()[t // 16]
            k, v = (case[n][page, t % 16][:, None] for n in ("k_cache", "v_cache"))
            want, room = attention64(one["q"], k, v, torch.arange(len(t), dtype=torch.int32)[None], torch.tensor([0, 1]), torch.tensor([len(t)]),
                                     gate=one["gate"])
            compare(got[r:r + 1], want, room)
    assert torch.equal(_attend(dev), got)
    monkeypatch.setenv("TJEV_GDN_POISON", "1")
    assert torch.equal(_attend(dev), got)
    monkeypatch.delenv("TJEV_GDN_POISON")
    with _lib.library(_lib.LDS_POISON_PATH):
        assert torch.equal(_attend(dev), got)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    ys = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                ys.append(_attend(dev))
    torch.cuda.synchronize()
    assert all(torch.equal(y, got) for y in ys)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = _attend(dev)
        graphs.append((g, y))
    for i in range(3):
        dev["q"].mul_(-1.25)
        dev["ancestors"].copy_(dev["ancestors"].roll(1, 0))
        torch.cuda.synchronize()
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, _attend(dev)) for _, y in graphs)


def test_tree_attention_past_32_bits():
    """A cache of 2^32 elements: trees in its last pages, moved and forked there too."""
    from tjev_amd import paged_compact, paged_fork

    pages, page, heads, dim = 131073 + 4, 16, 8, 256
    print("trees past 2^32 elements", flush=True)
    kc, vc = (torch.zeros(pages, page, heads, dim, dtype=BF, device="cuda") for _ in range(2))
    assert kc.numel() > 2 ** 32
    case = _case(9, [(9, 30)], heads=heads, kv_heads=heads, dim=dim, page=page, extra_pages=0, extra_width=0)
    far = torch.tensor([[pages - 1, 2, pages - 3]])
    for big, n in ((kc, "k_cache"), (vc, "v_cache")):
        big[far[0].cuda()] = case[n][case["block_table"][0].long()].cuda()
    want, room = tree_attention64(*(case[n] for n in NAMES))
    compare(_attend(dict(case, k_cache=kc, v_cache=vc, block_table=far.int())), want, room)
    dev = {n: x.cuda() for n, x in case.items() if isinstance(x, torch.Tensor)}
    path = torch.tensor([[0, 5, 9, 29]], dtype=torch.int32, device="cuda")
    lengths = paged_compact([(kc, vc)], far.int().cuda(), dev["starts"], dev["lengths"], path, torch.tensor([4], device="cuda"))
    assert lengths.tolist() == [13]
    shared = torch.zeros(pages, dtype=torch.int32, device="cuda")
    f = paged_fork([(kc, vc)], far.int().cuda(), dev["lengths"], torch.tensor([0, 0], device="cuda"), lengths.repeat(2),
                   torch.tensor([pages - 1, 2, pages - 3, pages - 2], dtype=torch.int32, device="cuda"), torch.tensor([3], device="cuda"), shared,
                   page_size=page)
    # (the two pages behind the kept tokens come back, in order, and the copy takes the first of them)
    assert f.block_table.tolist() == [[pages - 1, -1, -1], [2, -1, -1]] and f.free_pages.tolist() == [pages - 1, 2, pages - 3, pages - 2]
    assert int(f.taken) == 2
    for big, n in ((kc, "k_cache"), (vc, "v_cache")):
        for j, t in enumerate([*range(9), 9, 14, 18, 38]):
            w = case[n][case["block_table"][0, t // 16].long(), t % 16]
            assert torch.equal(big[pages - 1, j].cpu(), w) and torch.equal(big[2, j].cpu(), w)


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("captured", [False, True])
def test_drafted_steps(captured):
    """Prompts, then steps of drafted trees in two layers: tables, ancestors, rotary positions, the write, attention, verification,
    compaction, and forks that roll back, sample one request twice and end another; then the same again. What a request reads is at
    every step what its own tokens, one after the other, make it: the rows on the accepted path against attention over that sequence
    in 64 bits. Captured: a step recorded once and replayed for every other."""
    from tjev_amd import (draft_tree, paged_append, paged_attention, paged_compact, paged_fork, paged_tables, paged_tree_attention, rotary_axes,
                          verify_drafts)

    heads, kv, dim, page, half, vocab, most, places, layers = 8, 2, 64, 16, 16, 50, 12, 4, 2
    rng, gen = random.Random(1), torch.Generator().manual_seed(1)
    inv = (1e4 ** (-torch.arange(half, dtype=torch.float64) / half)).cuda()
    # the model: token x at position t has these q, k, v in each layer (before the turn), and the target's distribution
    table_q, table_k, table_v = (torch.randn(layers, vocab, h, dim, generator=gen).to(BF).cuda() for h in (heads, kv, kv))
    probs = torch.softmax(2 * torch.randn(vocab, vocab, generator=gen), -1).cuda()
    pages = 60
    caches = [tuple(torch.full((pages, page, kv, dim), math.nan, dtype=BF, device="cuda") for _ in range(2)) for _ in range(layers)]
    s = dict(table=torch.full((places, 10), -1, dtype=torch.int32), cached=torch.zeros(places, dtype=torch.int32), taken=torch.zeros(1, dtype=torch.int32),
             free=torch.randperm(pages, generator=gen).int(), shared=torch.zeros(pages, dtype=torch.int32))
    s = {n: x.cuda() for n, x in s.items()}
    rows = places * most

    def layer_rows(tokens, positions, slots):
        for i, (kc, vc) in enumerate(caches):
            q, k = rotary_axes(table_q[i][tokens], table_k[i][tokens], positions, inv)
            paged_append(k, table_v[i][tokens], kc, vc, slots)
            yield q, kc, vc

    # prompts
    prompt = [[rng.randrange(vocab) for _ in range(n)] for n in (20, 16, 33, 5)]
    flat = torch.tensor([x for p in prompt for x in p]).cuda()
    new = torch.tensor([len(p) for p in prompt], dtype=torch.int32).cuda()
    t = paged_tables(s["cached"], new, s["table"], s["free"], s["taken"], page_size=page, tokens=len(flat))
    pos = torch.cat([torch.arange(len(p)) for p in prompt]).cuda()
    for q, kc, vc in layer_rows(flat, pos, t.slots):
        paged_attention(q, kc, vc, t.block_table, t.starts, t.lengths)
    s.update(table=t.block_table, cached=t.lengths, taken=t.taken)
    texts = [list(p) for p in prompt]  # the tokens whose keys are cached
    roots = [7, 8, 9, 10]

    x = dict(tokens=torch.zeros(rows, dtype=torch.int64), parents=torch.zeros(rows, dtype=torch.int32), new=torch.zeros(places, dtype=torch.int32),
             uniforms=torch.zeros(rows), sources=torch.zeros(places, dtype=torch.int32), cut=torch.zeros(places, dtype=torch.int32))
    x = {n: v.cuda() for n, v in x.items()}

    def step():
        t = paged_tables(s["cached"], x["new"], s["table"], s["free"], s["taken"], page_size=page, tokens=rows)
        d = draft_tree(x["parents"], t.starts, t.lengths, max_new=most)
        outs = [paged_tree_attention(q, kc, vc, t.block_table, t.starts, t.lengths, d.ancestors, max_new=most)
                for q, kc, vc in layer_rows(x["tokens"], d.positions, t.slots)]
        v = verify_drafts(x["tokens"], probs[x["tokens"]], t.starts, x["uniforms"], parents=x["parents"], max_new=most)
        left = paged_compact(caches, t.block_table, t.starts, t.lengths, v.path, v.kept)
        f = paged_fork(caches, t.block_table, t.lengths, x["sources"], left[x["sources"].long().clamp(min=0)] - x["cut"], s["free"], t.taken, s["shared"],
                       page_size=page)
        return outs, v, f

    graph = None
    for n in range(6):
        print(f"drafted step {n} captured={captured}", flush=True)
        sizes = [rng.randint(1, most) if text else 0 for text in texts]
        trees = [random_tree(rng, k) if k else [] for k in sizes]
        toks = []
        for b, tree in enumerate(trees):
            mine = []
            for i, p in enumerate(tree):
                top = torch.topk(probs[mine[p]], 3).indices.tolist() if i else None
                mine.append(roots[b] if i == 0 else rng.choice(top))
            toks.append(mine)
        pad = rows - sum(sizes)
        sources = [[0, 1, 2, 3], [0, 1, 2, 0], [2, 1, -1, 3], [0, 1, 1, 3], [0, 1, 2, 3], [3, 2, 1, 0]][n]
        x["tokens"].copy_(torch.tensor([v for m in toks for v in m] + [0] * pad))
        x["parents"].copy_(torch.tensor([v for m in trees for v in m] + [5] * pad))
        x["new"].copy_(torch.tensor(sizes))
        x["uniforms"].copy_(torch.rand(rows, generator=gen))
        x["sources"].copy_(torch.tensor(sources))
        x["cut"].copy_(torch.tensor([0, 0, 1, 0]) if n == 3 else torch.zeros(4))
        saved = [tuple(c.clone() for c in pair) for pair in caches]
        outs, v, f = step()
        if captured:
            eager = [*outs, *v, *f, *(c.clone() for pair in caches for c in pair)]
            if graph is None:
                for pair, old in zip(caches, saved):
                    for c, o in zip(pair, old):
                        c.copy_(o)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    recorded = step()
            for pair, old in zip(caches, saved):
                for c, o in zip(pair, old):
                    c.copy_(o)
            graph.replay()
            outs, v, f = recorded
            for a, e in zip([*outs, *v, *f, *(c for pair in caches for c in pair)], eager):
                assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(e))
        # every request's accepted rows, as the last rows of the sequence that they continue
        lo = 0
        for b, text in enumerate(texts):
            kept = int(v.kept[b])
            assert (kept > 0) == (sizes[b] > 0)
            way = v.path[b, :kept].tolist()
            seq = text + [toks[b][i] for i in way]
            said = v.tokens[b, :kept].tolist()
            assert said[:-1] == [toks[b][i] for i in way[1:]] and 0 <= (said[-1] if kept else 0) < vocab
            if kept:
                ids = torch.tensor(seq).cuda()
                for i in range(layers):
                    q, k = rotary_axes(table_q[i][ids], table_k[i][ids], torch.arange(len(seq)).cuda(), inv)
                    want, room = attention64(q[-kept:].cpu(), k[:, None].cpu(), table_v[i][ids][:, None].cpu(), torch.arange(len(seq), dtype=torch.int32)[None],
                                             torch.tensor([0, kept]), torch.tensor([len(seq)]))
                    compare(outs[i][lo:lo + sizes[b]][way], want, room)
                roots[b] = said[-1]
            texts[b] = seq
            lo += sizes[b]
        texts, roots = [texts[b] if b >= 0 else [] for b in sources], [roots[b] if b >= 0 else 0 for b in sources]
        if n == 3:
            texts[2] = texts[2][:-1]
        # (in place: a captured step reads them where they are)
        s["table"].copy_(f.block_table), s["cached"].copy_(f.lengths), s["free"].copy_(f.free_pages), s["taken"].copy_(f.taken), s["shared"].copy_(f.shared)
        assert s["cached"].tolist() == [len(text) for text in texts]
        held = {}
        for b in range(places):
            row = [p for p in s["table"][b].tolist() if p >= 0]
            assert len(row) == -(-len(texts[b]) // page)
            for p in row:
                held[p] = held.get(p, 0) + 1
        rest = s["free"][int(s["taken"]):].tolist()
        assert not set(rest) & set(held) and len(rest) + len(held) == pages
        assert [held.get(p, 1) - 1 for p in range(pages)] == s["shared"].tolist()
