"""Paged attention (tjev_amd.paged) where pages end inside a tile, at every head dim's own tile: against the plain 64-bit forms
of tests/paged_cases.py, with missing pages, bad values, and weights held to the bits that the streamed tiles keep."""

from __future__ import annotations

import math

import pytest
import torch

from paged_cases import HALF_STEP, attention64, batch, compare

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
NAMES = ("q", "k_cache", "v_cache", "block_table", "starts", "lengths")
# one token each, drafts, a chunk of few and one of many rows
LENS = {"decode": [(15, 1), (16, 1), (0, 1), (127, 1), (129, 1), (500, 1)], "drafts": [(31, 5), (0, 3), (64, 2), (200, 4)],
        "ragged": [(40, 17), (0, 0), (3, 1), (0, 33), (70, 1), (0, 0)], "chunk": [(130, 150)]}


def _attend(case, **kw):
    from tjev_amd import paged_attention

    return paged_attention(**{n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in {**case, **kw}.items()})


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [
    (16, 4, 256, 24), (8, 2, 256, 8), (8, 2, 256, 10), (8, 2, 200, 10), (8, 2, 200, 8), (8, 2, 128, 8), (8, 2, 96, 8), (8, 2, 64, 8),
    (8, 2, 40, 24), (4, 4, 256, 1), (16, 4, 256, 100),
])
@pytest.mark.parametrize("lens", sorted(LENS))
def test_pages_that_end_inside_a_tile(dtype, heads, kv_heads, dim, page, lens):
    gate = len(lens) % 2 == 0
    print(f"attention {dtype} heads={heads}/{kv_heads} dim={dim} page={page} {lens} gate={gate}", flush=True)
    case = batch(torch.Generator().manual_seed(dim + page), LENS[lens], heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype,
                 pad_rows=3, gate=gate)
    want, room = attention64(*(case[n] for n in NAMES), gate=case["gate"])
    got = _attend(case)
    compare(got, want, room)
    assert bool((got[-3:] == 0).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("page", [8, 10, 16, 24])
@pytest.mark.parametrize("dim", [128, 200, 256])
def test_missing_pages(dtype, page, dim):
    """Entries that are no page of the cache, in the first, middle and last places of requests of few and many rows."""
    case = batch(torch.Generator().manual_seed(31), [(200, 4), (90, 60), (33, 1), (5, 90)], heads=8, kv_heads=2, dim=dim, page=page, dtype=dtype)
    t = case["block_table"]
    t[0, 0], t[0, 3], t[1, 0], t[1, 2], t[2, :], t[3, 1] = -1, case["k_cache"].shape[0], 2 ** 31 - 1, -7, -2 ** 31, -1
    t[1, -(-150 // page) - 1] = -1  # the last keys of many rows
    print(f"attention over missing pages {dtype} page={page} dim={dim}", flush=True)
    want, room = attention64(*(case[n] for n in NAMES))
    compare(_attend(case), want, room)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("page", [8, 10, 24])
@pytest.mark.parametrize("dim", [64, 128, 200, 256])
def test_bad_values_reach_only_their_rows(dtype, page, dim):
    """NaN and infinities in later tokens' keys and values, beside rows that do not attend to them."""
    lens = [(100, 3), (30, 60)]
    case = batch(torch.Generator().manual_seed(32), lens, heads=4, kv_heads=2, dim=dim, page=page, dtype=dtype)
    c, n = lens[-1]
    at = lambda t: (int(case["block_table"][1, t // page]), t % page)  # noqa: E731
    clean = _attend(case)
    case["v_cache"][at(c + n // 2)][0, 3] = math.nan
    case["v_cache"][at(c + n - 2)][1, 5] = math.inf
    case["v_cache"][at(c + n - 5)][1, 5] = math.inf
    case["k_cache"][at(c + n - 1)][0, 2] = math.nan
    print(f"attention with bad values {dtype} page={page} dim={dim}", flush=True)
    got = _attend(case)
    first = int(case["starts"][1])
    assert torch.equal(got[:first + n // 2], clean[:first + n // 2])
    want, room = attention64(*(case[x] for x in NAMES))
    compare(got, want, room)
    assert bool(torch.isnan(got[-1, :2]).all()) and bool(torch.isinf(got[-1, 2:, 5]).all())


# ---------------------------------------------------------------- the weights' bits
def cancelling(gen, tokens, keys, heads, kv_heads, dim):
    """A request whose values cancel in pairs of nearly equal weight: what is left of a sum is small beside what went into it, and
    so is its rounding to bf16."""
    k, v = torch.randn(keys, kv_heads, dim, generator=gen), torch.randn(keys, kv_heads, dim, generator=gen)
    k[1::2] = k[::2] + 0.02 * torch.randn(keys // 2, kv_heads, dim, generator=gen)
    v[1::2] = -v[::2]
    return torch.randn(tokens, heads, dim, generator=gen).to(BF), k.to(BF), v.to(BF)


def weighted(q, k, v, round_weights=None):
    """(out, room) of one request's rows q [T, H, D], all of which attend to all keys, in 64 bits. The room is attention64's
    (paged_cases.py) with two bf16 terms to a weight: the first its upper 8 bits, the second the rest (below 2^-7 of it) rounded
    by half a step, 2^-8 of that: 2^-15."""
    heads, kv, dim = q.shape[1], k.shape[1], q.shape[2]
    out, room = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for h in range(heads):
        x, kk, vv = q[:, h].double(), k[:, h * kv // heads].double(), v[:, h * kv // heads].double()
        s = dim ** -0.5 * (x @ kk.t())
        w = torch.exp(s - s.amax(-1, keepdim=True))
        o, a = (w if round_weights is None else round_weights(w)) @ vv / w.sum(-1, keepdim=True), w @ vv.abs() / w.sum(-1, keepdim=True)
        delta = (dim + 8) * 2.0 ** -24 * dim ** -0.5 * (x.abs() @ kk.abs().t()).amax(-1, keepdim=True)
        r = a * (4 * delta + (k.shape[0] + 64) * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -15)
        out[:, h], room[:, h] = o, r + HALF_STEP[BF] * (o.abs() + r)
    return out, room


SHAPES = [(16, 4, 64, 16), (16, 4, 128, 16), (16, 4, 256, 16), (8, 1, 96, 10), (8, 1, 256, 24), (20, 1, 64, 16)]


@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
def test_streamed_weights_keep_their_bits(heads, kv_heads, dim, page):
    from tjev_amd import paged_attention

    gen, keys = torch.Generator().manual_seed(33), 12
    q, k, v = cancelling(gen, 1, keys, heads, kv_heads, dim)
    pages = -(-keys // page)
    kc, vc = (torch.zeros(pages * page, kv_heads, dim, dtype=BF) for _ in range(2))
    kc[:keys], vc[:keys] = k, v
    print(f"weights of streamed rows {heads}/{kv_heads} of {dim} page={page}", flush=True)
    got = paged_attention(q.cuda(), *(c.view(pages, page, kv_heads, dim).cuda() for c in (kc, vc)),
                          torch.arange(pages, dtype=torch.int32, device="cuda")[None], torch.tensor([0, 1], dtype=torch.int32, device="cuda"),
                          torch.tensor([keys], dtype=torch.int32, device="cuda"))
    compare(got, *weighted(q, k, v))
