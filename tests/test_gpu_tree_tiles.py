"""Trees in tiles of 128 rows (tjev_amd.paged_tree_attention in bf16): block tables as wide as a server's, where no batch of them is
streamed, against the plain 64-bit form. That a case takes these tiles is read from the size of its workspace."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from draft_cases import tree_attention64
from paged_cases import attention64, compare
from test_gpu_tree_attention import LENS, NAMES, _attend, _case

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _place(rows, dim):
    """The bytes of a range's two unfinished tiles and its note."""
    return 2 * rows * ((64 if dim <= 64 else 128 if dim <= 128 else 256) + 2) * 4 + 32


def _workspace(case, max_new=None):
    from tjev_amd import _lib

    (tokens, heads, dim), (pages, page, kv_heads, _) = case["q"].shape, case["k_cache"].shape
    requests, width = case["block_table"].shape
    p = _lib.PagedParams(tokens=tokens, requests=requests, table_width=width, pages=pages, page_size=page, heads=heads, kv_heads=kv_heads, dim=dim,
                         dtype=_lib.BF16, scale=1.0, max_new=max_new or 0)
    return _lib.load().tjev_gdn_paged_tree_workspace_bytes(ctypes.byref(p))


def _wide(case, tokens=1 << 17, max_new=None):
    """The case with a table for `tokens` keys a request, whose tiles have 128 rows in as many ranges as there are."""
    table, page = case["block_table"], case["k_cache"].shape[1]
    case["block_table"] = torch.nn.functional.pad(table, (0, max(0, tokens // page - table.shape[1])), value=-1)
    dim = case["q"].shape[2]
    assert _workspace(case, max_new) == (768 if dim <= 64 else 512) * _place(128, dim)
    return case


@pytest.mark.parametrize("heads,kv_heads,dim,page", [
    (4, 1, 64, 16), (2, 2, 128, 24), (16, 4, 256, 16), (5, 1, 40, 5), (20, 1, 96, 64), (3, 3, 8, 1), (6, 2, 200, 48), (12, 2, 64, 24), (8, 2, 256, 8),
    (6, 2, 256, 20),
])
@pytest.mark.parametrize("lens,kind", [("ragged", "star"), ("wide", "tree"), ("words", "any")])
def test_tiles_of_128_rows(heads, kv_heads, dim, page, lens, kind):
    """Every place of the cache that no token has holds NaN; rows behind the last request come back 0."""
    print(f"wide trees heads={heads}/{kv_heads} dim={dim} page={page} {lens} {kind}", flush=True)
    case = _wide(_case(dim + page, LENS[lens], kind, heads=heads, kv_heads=kv_heads, dim=dim, page=page, pad_rows=3, gate=kind != "star"))
    want, room = tree_attention64(*(case[n] for n in NAMES), gate=case["gate"])
    got = _attend(case)
    compare(got, want, room)
    assert bool((got[-3:] == 0).all())


@pytest.mark.parametrize("heads,kv_heads,dim,lens", [(4, 2, 64, [(40, 17), (0, 5), (90, 70)]), (16, 4, 256, [(300, 9), (20, 40)]),
                                                     (8, 2, 128, [(0, 200), (77, 3)])])
def test_a_chain_in_them_is_causal(heads, kv_heads, dim, lens):
    print(f"wide chains {heads}/{kv_heads} of {dim} {lens}", flush=True)
    case = _wide(_case(3, lens, "chain", heads=heads, kv_heads=kv_heads, dim=dim, page=16, gate=True))
    want, room = attention64(*(case[n] for n in NAMES[:-1]), gate=case["gate"])
    compare(_attend(case), want, room)


@pytest.mark.parametrize("heads,dim,page", [(4, 64, 16), (24, 64, 24), (4, 128, 24), (24, 128, 64), (4, 256, 10), (24, 256, 16), (4, 72, 8)])
@pytest.mark.parametrize("words", [1, 2, 3])
def test_rows_in_them_may_name_any_token(heads, dim, page, words):
    """Bits at random: tokens behind a row's own, not its own, none at all; more words than tokens, and fewer."""
    lens = [(0, 40), (30, 130), (0, 3), (17, 64), (64, 1)]
    case = _wide(_case(4, lens, heads=heads, kv_heads=2, dim=dim, page=page, pad_rows=1))
    gen = torch.Generator().manual_seed(words)
    case["ancestors"] = torch.randint(-2 ** 63, 2 ** 63 - 1, (case["q"].shape[0], words), generator=gen)
    case["ancestors"][::7] = 0
    case["ancestors"][3::7] = -1
    print(f"any tokens, wide, heads={heads} of {dim} page={page} words={words}", flush=True)
    want, room = tree_attention64(*(case[n] for n in NAMES))
    got = _attend(case)
    compare(got, want, room)
    assert bool((got[:40:7] == 0).all())  # rows of the first request without keys


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 10, 24])
@pytest.mark.parametrize("heads", [4, 16])
def test_pages_of_them_that_are_none(dim, page, heads):
    """Entries that are no page, lengths past the table's width or shorter than the new tokens, trees that have lost their own keys."""
    case = _case(5, [(200, 14), (90, 40), (33, 11), (0, 27), (50, 60)], heads=heads, kv_heads=2, dim=dim, page=page)
    t = case["block_table"]
    t[0, 1], t[0, 3], t[1, 0], t[2, :] = -1, case["k_cache"].shape[0], 2 ** 31 - 1, -2 ** 31
    case["lengths"][0] += 3000
    case["lengths"][3] = 4      # all but four of its new tokens stand before the first
    t[4, 60 // page:] = -1
    t[0][t[0] == -1] = 10 ** 6
    print(f"wide trees over pages that are none, dim={dim} page={page} heads={heads}", flush=True)
    want, room = tree_attention64(*(case[n] for n in NAMES))
    compare(_attend(_wide(case)), want, room)


@pytest.mark.parametrize("lens,dim,page", [([(20, 40)], 64, 16), ([(100, 3), (5, 30)], 128, 16), ([(0, 150)], 256, 16), ([(9, 100)], 64, 24),
                                           ([(60, 33)], 256, 24), ([(300, 130)], 128, 10), ([(129, 90)], 40, 8), ([(33, 70)], 200, 5)])
@pytest.mark.parametrize("kind", ["tree", "any"])
def test_bad_values_in_them_reach_only_their_rows(lens, dim, page, kind):
    """NaN and infinities in the keys and values of some new tokens, of both signs in one column, and in a cached token's value: the
    rows that do not name them are as if they were not there."""
    case = _wide(_case(6, lens, kind, heads=4, kv_heads=2, dim=dim, page=page))
    c, n = lens[-1]
    table, b = case["block_table"], len(lens) - 1
    at = lambda t: (int(table[b, t // page]), t % page)  # noqa: E731
    clean = _attend(case)
    bad = (n // 2, n - 4, n - 3, n - 2, n - 1)
    case["v_cache"][at(c + bad[0])][0, 3] = math.nan
    case["v_cache"][at(c + bad[1])][1, 5] = math.inf
    case["v_cache"][at(c + bad[2])][1, 5] = -math.inf
    case["v_cache"][at(c + bad[3])][0, dim - 1] = -math.inf
    case["k_cache"][at(c + bad[4])][0, 2] = math.nan
    print(f"wide trees with bad values {lens} dim={dim} page={page} {kind}", flush=True)
    got = _attend(case)
    first = int(case["starts"][b])
    free = [r for r in range(n) if not any(int(case["ancestors"][first + r, j // 64]) >> j % 64 & 1 for j in bad)]
    assert free and len(free) < n
    assert torch.equal(got[:first], clean[:first]) and all(torch.equal(got[first + r], clean[first + r]) for r in free)
    want, room = tree_attention64(*(case[x] for x in NAMES))
    compare(got, want, room)
    assert bool(torch.isnan(got[first + n - 1, :2]).all())
    gen = torch.Generator().manual_seed(dim)  # the same of bits at random
    case["ancestors"] = torch.randint(-2 ** 63, 2 ** 63 - 1, case["ancestors"].shape, generator=gen)
    want, room = tree_attention64(*(case[x] for x in NAMES))
    compare(_attend(case), want, room)


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 24), (256, 16), (256, 12)])
def test_layouts_views_and_scales_of_them(dim, page):
    """Caches with the heads before the places or keys beside values, q beside its gate, a given out whose rows of no request stay, rows in
    front, int64 lengths, a negative scale and 0."""
    from tjev_amd import paged_tree_attention

    case = _wide(_case(7, [(40, 3), (100, 40), (7, 31)], heads=4, kv_heads=2, dim=dim, page=page, pad_rows=4, gate=True))
    case["starts"] += 2
    case["ancestors"] = case["ancestors"].roll(2, 0)
    for scale in (0.3, -0.2, 0.0):
        want, room = tree_attention64(*(case[n] for n in NAMES), scale, case["gate"])
        qg = torch.cat([case["q"], case["gate"]], -1).cuda()
        dev = {n: x.cuda() for n, x in case.items()}
        dev.update(q=qg[..., :dim], gate=qg[..., dim:], starts=dev["starts"].long(), lengths=dev["lengths"].long(),
                   ancestors=torch.stack([dev["ancestors"]] * 2, 1)[:, 0])
        kc, vc = dev["k_cache"], dev["v_cache"]
        for name, (k, v) in {"plain": (kc, vc), "heads first": tuple(c.transpose(1, 2).contiguous().transpose(1, 2) for c in (kc, vc)),
                             "joint": tuple(torch.stack([kc, vc], 1).unbind(1))}.items():
            print(f"wide trees, layout {name} dim={dim} page={page} scale={scale}", flush=True)
            got = paged_tree_attention(**dict(dev, k_cache=k, v_cache=v), scale=scale)
            compare(got, want, room)
            wide = torch.full((got.shape[0], 4, 2 * dim), 7.0, dtype=BF, device="cuda")
            out = wide[..., dim:]
            assert paged_tree_attention(**dict(dev, k_cache=k, v_cache=v), scale=scale, out=out) is out
            assert torch.equal(out[2:-2], got[2:-2]) and bool((out[:2] == 7).all()) and bool((out[-2:] == 7).all())
            assert bool((wide[..., :dim] == 7).all())


# tiles whose keys several ranges hold, joined in each of the ways: slices of few tiles, as many as the lengths say, and by ranges
SPLIT = {
    "sliced, 64": ([(3000, 64)], 8, 2, 64, 16, None), "sliced, 128": ([(2000, 130)], 4, 2, 128, 24, None),
    "sliced, 256": ([(3000, 64)], 16, 4, 256, 16, None), "sliced, 200": ([(1000, 21), (700, 5)], 8, 2, 200, 16, None),
    "counted, 64": ([(2500, 50)] + [(0, 0)] * 40, 8, 2, 64, 16, 50), "counted, 128": ([(2500, 50)] + [(0, 0)] * 40, 8, 2, 128, 10, 50),
    "counted, 256": ([(3000, 64)] + [(0, 0)] * 63, 16, 4, 256, 16, 64), "ranges, 64": ([(900, 40)] * 9, 16, 4, 64, 24, None),
    "ranges, 128": ([(1500, 70)] * 6, 16, 4, 128, 16, None), "ranges, 256": ([(1200, 33), (4, 2)] * 5, 16, 4, 256, 16, None),
}


@pytest.mark.parametrize("kind", sorted(SPLIT))
def test_long_contexts_in_them(monkeypatch, kind):
    """Many workgroups a tile: right, the same bits twice, in the poison modes, and captured."""
    from tjev_amd import _lib

    lens, heads, kv_heads, dim, page, max_new = SPLIT[kind]
    case = _wide(_case(8, lens, heads=heads, kv_heads=kv_heads, dim=dim, page=page, gate=True), max_new=max_new)
    dev = dict({n: x.cuda() for n, x in case.items()}, max_new=max_new)
    print(f"long contexts, wide: {kind}", flush=True)
    got = _attend(dev)
    # some rows of the first and of a middle request, each as the last token of a sequence of the tokens that it names
    for b in sorted({0, len(lens) // 2}):
        s0, s1 = int(case["starts"][b]), int(case["starts"][b + 1])
        first = int(case["lengths"][b]) - (s1 - s0)
        for r in sorted({s0, (s0 + s1) // 2, s1 - 1} if s1 > s0 else ()):
            named = [j for j in range(s1 - s0) if int(case["ancestors"][r, j // 64]) >> j % 64 & 1]
            t = torch.tensor([*range(first), *(first + j for j in named)])
            at = case["block_table"][b].long()[t // page]
            k, v = (case[n][at, t % page][:, None] for n in ("k_cache", "v_cache"))
            want, room = attention64(case["q"][r:r + 1], k, v, torch.arange(len(t), dtype=torch.int32)[None], torch.tensor([0, 1]),
                                     torch.tensor([len(t)]), gate=case["gate"][r:r + 1])
            compare(got[r:r + 1], want, room)
    assert torch.equal(_attend(dev), got)
    monkeypatch.setenv("TJEV_GDN_POISON", "1")
    assert torch.equal(_attend(dev), got)
    monkeypatch.delenv("TJEV_GDN_POISON")
    with _lib.library(_lib.LDS_POISON_PATH):
        assert torch.equal(_attend(dev), got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = _attend(dev)
    for _ in range(2):
        dev["q"].mul_(-1.25)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, _attend(dev))
