"""The paged cache's operators (tjev_amd.paged) against their plain 64-bit forms (tests/paged_cases.py), at the sizes
where they can go wrong: requests and pages that end inside a tile, rows without keys, pages that are none, NaN in
every place that no row attends to, other cache layouts, one long request over many workgroups, offsets past 2^32."""

from __future__ import annotations

import math

import pytest
import torch

from paged_cases import attention64, batch, compare, rotary64, tables_walk

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _cuda(x):
    return x.cuda() if isinstance(x, torch.Tensor) else x


def _attend(case, **kw):
    from tjev_amd import paged_attention

    return paged_attention(**{n: _cuda(x) for n, x in {**case, **kw}.items()})


# ---------------------------------------------------------------- tables and slots
@pytest.mark.parametrize("page,lens,free,taken,tokens", [
    (16, [(0, 1)], 3, 0, 1), (16, [(16, 1), (15, 1), (17, 0), (0, 0)], 5, 1, 4), (1, [(3, 4), (0, 2)], 9, 0, 9),
    (24, [(50, 100), (0, 0), (23, 1), (24, 1)], 12, 2, 110), (64, [(0, 200)], 2, 0, 205),  # a shortage
    (16, [(5, 300)], 40, 0, 300),  # past the table's width
    (7, [(i % 19, i % 5) for i in range(700)], 900, 3, 1500), (16, [(0, 0)] * 3, 0, 0, 0), (16, [(-4, 3), (2, -1)], 4, 0, 5),
    (32, [(100, 50)] * 20, 60, 0, 400),  # fewer slots than tokens
])
@pytest.mark.parametrize("inplace", [False, True])
def test_tables(page, lens, free, taken, tokens, inplace):
    from tjev_amd import paged_tables

    gen = torch.Generator().manual_seed(len(lens))
    width = 12
    ids = torch.randperm(5000, generator=gen).int()
    table = ids[:len(lens) * width].view(len(lens), width).clone() if len(lens) * width <= 5000 else torch.randint(
        0, 5000, (len(lens), width), generator=gen).int()
    pages = ids[-free:] if free else ids[:0]
    c, n = ([x[i] for x in lens] for i in (0, 1))
    want = tables_walk(c, n, table.tolist(), pages.tolist(), taken, page, tokens, inplace)
    dt = torch.int64 if len(lens) % 2 else torch.int32
    print(f"tables page={page} requests={len(lens)} inplace={inplace}", flush=True)
    dev = table.cuda()
    t = paged_tables(torch.tensor(c, dtype=dt).cuda(), torch.tensor(n, dtype=dt).cuda(), dev, pages.cuda(),
                     torch.tensor([taken], dtype=dt).cuda() if taken else None, page_size=page, tokens=tokens, inplace=inplace)
    assert (t.block_table.data_ptr() == dev.data_ptr()) == inplace
    for got, exp in zip(t, want):
        assert got.cpu().tolist() == exp if isinstance(exp, list) else int(got) == exp


def test_tables_of_many_requests():
    from tjev_amd import paged_tables

    gen = torch.Generator().manual_seed(0)
    c, n = (torch.randint(0, m, (8192,), generator=gen).int() for m in (60, 4))
    table, free = torch.randint(0, 99999, (8192, 8), generator=gen).int(), torch.randperm(99999, generator=gen).int()
    print("tables of 8192 requests", flush=True)
    t = paged_tables(c.cuda(), n.cuda(), table.cuda(), free.cuda(), page_size=8, tokens=20000)
    want = tables_walk(c.tolist(), n.tolist(), table.tolist(), free.tolist(), 0, 8, 20000)
    for got, exp in zip(t, want):
        assert got.cpu().tolist() == exp if isinstance(exp, list) else int(got) == exp


# ---------------------------------------------------------------- the write
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads,dim,page,layout", [(2, 64, 16, "plain"), (1, 8, 3, "heads first"), (3, 20, 5, "joint"), (8, 128, 64, "plain"),
                                                   (5, 7, 1, "odd"), (16, 256, 24, "heads first")])
@pytest.mark.parametrize("tokens", [1, 7, 300])
def test_append(dtype, heads, dim, page, layout, tokens):
    from tjev_amd import paged_append

    gen = torch.Generator().manual_seed(dim + tokens)
    pages = 2 + tokens // page
    print(f"append {dtype} heads={heads} dim={dim} page={page} {layout} tokens={tokens}", flush=True)
    shape = (pages, page, heads, dim)
    if layout == "heads first":
        kc, vc = (torch.randn(pages, heads, page, dim, generator=gen).to(dtype).cuda().transpose(1, 2) for _ in range(2))
    elif layout == "joint":
        kc, vc = torch.randn(pages, 2, page, heads, dim, generator=gen).to(dtype).cuda().unbind(1)
    elif layout == "odd":
        kc, vc = (torch.randn(math.prod(shape) + 1, generator=gen).to(dtype).cuda()[1:].view(shape) for _ in range(2))
    else:
        kc, vc = (torch.randn(shape, generator=gen).to(dtype).cuda() for _ in range(2))
    kv = torch.randn(tokens, 2, heads, dim, generator=gen).to(dtype)
    slots = torch.randperm(pages * page, generator=gen)[:tokens]
    slots[::3] = torch.tensor([-1, pages * page, 2 ** 40, -2 ** 40])[torch.arange(len(slots[::3])) % 4]
    want_k, want_v = kc.cpu().clone(), vc.cpu().clone()
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            want_k[s // page, s % page], want_v[s // page, s % page] = kv[t, 0], kv[t, 1]
    dev = kv.cuda()
    paged_append(dev[:, 0], dev[:, 1], kc, vc, slots.cuda())
    assert torch.equal(kc.cpu(), want_k) and torch.equal(vc.cpu(), want_v)


def test_append_of_nothing():
    from tjev_amd import paged_append

    c = torch.ones(2, 16, 2, 64, device="cuda")
    e = torch.empty(0, 2, 64, device="cuda")
    paged_append(e, e, c, c, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert bool((c == 1).all())


# ---------------------------------------------------------------- attention
LENS = {
    "one": [(0, 1)], "decode": [(15, 1), (16, 1), (0, 1), (127, 1), (128, 1), (129, 1), (500, 1)],
    "drafts": [(31, 5), (0, 3), (64, 2), (200, 4)], "ragged": [(40, 17), (0, 0), (3, 1), (0, 33), (70, 1), (0, 0)],
    "chunk": [(130, 150)],
}


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [
    (4, 1, 64, 16), (2, 2, 128, 24), (16, 4, 256, 16), (5, 1, 40, 5), (20, 1, 96, 64), (3, 3, 8, 1), (6, 2, 200, 48), (8, 8, 64, 100),
])
@pytest.mark.parametrize("lens", sorted(LENS))
def test_attention(dtype, heads, kv_heads, dim, page, lens):
    """Every place of the cache that no token has holds NaN; rows behind the last request come back 0."""
    gate = len(lens) % 2 == 0
    print(f"attention {dtype} heads={heads}/{kv_heads} dim={dim} page={page} {lens} gate={gate}", flush=True)
    case = batch(torch.Generator().manual_seed(dim), LENS[lens], heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype,
                 pad_rows=3, gate=gate)
    got = _attend(case)
    want, room = attention64(case["q"], case["k_cache"], case["v_cache"], case["block_table"], case["starts"], case["lengths"],
                             gate=case["gate"])
    compare(got, want, room)
    assert bool((got[-3:] == 0).all())


@pytest.mark.parametrize("dtype,dim,page,heads,kv_heads,lens", [
    (BF, 64, 16, 8, 1, [(31, 3), (0, 4), (200, 3), (77, 2)]), (BF, 40, 24, 8, 1, [(700, 4)]), (BF, 64, 10, 16, 2, [(31, 1), (5, 1), (64, 9)]),
    (BF, 64, 64, 5, 1, [(3000, 5), (9, 5), (0, 5)]), (F32, 64, 16, 16, 8, [(130, 260)]), (F32, 96, 24, 16, 8, [(30, 200), (9, 65)]),
])
def test_tiles_of_32_rows(dtype, dim, page, heads, kv_heads, lens):
    """Requests of 17 to 32 rows on average (bf16, head dims up to 64) and large fp32 batches."""
    print(f"attention {dtype} heads={heads}/{kv_heads} dim={dim} page={page} {lens}", flush=True)
    case = batch(torch.Generator().manual_seed(20), lens, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, pad_rows=1, gate=True)
    want, room = attention64(case["q"], case["k_cache"], case["v_cache"], case["block_table"], case["starts"], case["lengths"],
                             gate=case["gate"])
    compare(_attend(case), want, room)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("page", [16, 10])
@pytest.mark.parametrize("heads", [4, 16])
def test_pages_that_are_none(dtype, page, heads):
    """A table's entries -1 or past the cache hold no keys: what is left is attended to, and a row without
    any is 0. Lengths past the table's width end there; lengths shorter than the new tokens leave rows empty."""
    case = batch(torch.Generator().manual_seed(5), [(200, 4), (90, 20), (33, 1), (0, 7)], heads=heads, kv_heads=2, dim=64, page=page, dtype=dtype)
    t = case["block_table"]
    t[0, 1], t[0, 3], t[1, 0], t[2, :] = -1, case["k_cache"].shape[0], 2 ** 31 - 1, -2 ** 31
    case["lengths"][0] += 3000  # behind the table: the keys end with it
    case["lengths"][3] = 4      # three of its seven tokens stand before the first
    t[0][t[0] == -1] = 10 ** 6
    print(f"attention over pages that are none {dtype} page={page} heads={heads}", flush=True)
    want, room = attention64(*(case[n] for n in ("q", "k_cache", "v_cache", "block_table", "starts", "lengths")))
    got = _attend(case)
    compare(got, want, room)
    empty = int(case["starts"][2])
    assert bool((got[empty] == 0).all()) and bool((got[empty + 1:empty + 4] == 0).all()) and bool((got[empty + 4:] != 0).any())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lens,dim", [([(20, 40)], 64), ([(100, 3), (5, 30)], 128), ([(0, 150)], 256)])
def test_bad_values_reach_only_their_rows(dtype, lens, dim):
    """NaN and infinities in the keys and values of a request's later tokens: the rows before them, which do not
    attend to them, are as if they were not there; the rows that do are NaN or infinite as the sums are."""
    case = batch(torch.Generator().manual_seed(6), lens, heads=4, kv_heads=2, dim=dim, page=16, dtype=dtype)
    c, n = lens[-1]
    table, b = case["block_table"], len(lens) - 1
    at = lambda t: (int(table[b, t // 16]), t % 16)  # noqa: E731
    clean = _attend(case)
    case["v_cache"][at(c + n // 2)][0, 3] = math.nan
    case["v_cache"][at(c + n - 2)][1, 5] = math.inf
    case["k_cache"][at(c + n - 1)][0, 2] = math.nan
    print(f"attention with bad values {dtype} {lens} dim={dim}", flush=True)
    got = _attend(case)
    first = int(case["starts"][b])
    assert torch.equal(got[:first + n // 2], clean[:first + n // 2])
    want, room = attention64(*(case[n_] for n_ in ("q", "k_cache", "v_cache", "block_table", "starts", "lengths")))
    compare(got, want, room)
    assert bool(torch.isnan(got[-1, :2]).all()) and bool(torch.isinf(got[-1, 2:, 5]).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lens,dim", [([(50, 1)], 64), ([(600, 3), (7, 1)], 128), ([(40, 40)], 256), ([(3000, 1)], 128)])
def test_infinities_that_all_rows_attend_to(dtype, lens, dim):
    """Infinities among the values of a request's first tokens come out as such: no weight is or has a part that is 0."""
    case = batch(torch.Generator().manual_seed(16), lens, heads=4, kv_heads=2, dim=dim, page=16, dtype=dtype)
    for b in range(len(lens)):
        page = int(case["block_table"][b, 0])
        case["v_cache"][page, 0, 0, 3], case["v_cache"][page, 1, 1, 5] = math.inf, -math.inf
    print(f"attention with infinities {dtype} {lens} dim={dim}", flush=True)
    want, room = attention64(*(case[n] for n in ("q", "k_cache", "v_cache", "block_table", "starts", "lengths")))
    assert bool((want[:, :2, 3] == math.inf).all()) and bool((want[:, 2:, 5] == -math.inf).all()) and bool((~torch.isnan(want)).all())
    compare(_attend(case), want, room)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_layouts_and_views(dtype):
    """Caches with the heads before the places, or keys and values in one tensor; q beside its gate; a given out
    whose rows of no request stay; another scale; int64 lengths; starts that leave rows in front."""
    gen = torch.Generator().manual_seed(7)
    case = batch(gen, [(40, 3), (100, 20), (7, 1)], heads=4, kv_heads=2, dim=64, page=16, dtype=dtype, pad_rows=4, gate=True)
    case["starts"] += 2  # two rows before the first request, two behind the last
    want, room = attention64(case["q"], case["k_cache"], case["v_cache"], case["block_table"], case["starts"], case["lengths"], 0.3, case["gate"])
    qg = torch.cat([case["q"], case["gate"]], -1).cuda()
    dev = {n: _cuda(x) for n, x in case.items()}
    dev.update(q=qg[..., :64], gate=qg[..., 64:], starts=dev["starts"].long(), lengths=dev["lengths"].long())
    kc, vc = dev["k_cache"], dev["v_cache"]
    joint = torch.stack([kc, vc], 1)
    layouts = {"plain": (kc, vc), "heads first": tuple(c.transpose(1, 2).contiguous().transpose(1, 2) for c in (kc, vc)),
               "joint": tuple(joint.unbind(1)), "wide": tuple(torch.cat([c, c], -1)[..., :64] for c in (kc, vc))}
    from tjev_amd import paged_attention

    for name, (k, v) in layouts.items():
        print(f"attention layout {name} {dtype}", flush=True)
        got = paged_attention(**dict(dev, k_cache=k, v_cache=v), scale=0.3)
        compare(got, want, room)
        assert bool((got[:2] == 0).all()) and bool((got[-2:] == 0).all())
        wide = torch.full((got.shape[0], 4, 128), 7.0, dtype=dtype, device="cuda")
        out = wide[..., 64:]
        assert paged_attention(**dict(dev, k_cache=k, v_cache=v), scale=0.3, out=out) is out
        assert torch.equal(out[2:-2], got[2:-2]) and bool((out[:2] == 7).all()) and bool((out[-2:] == 7).all())
        assert bool((wide[..., :64] == 7).all())
    k = torch.empty(kc.numel() + 1, dtype=dtype, device="cuda")[1:].view(kc.shape)
    with pytest.raises(RuntimeError, match="16-byte"):
        paged_attention(**dict(dev, k_cache=k))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lens,heads,dim", [([(20000, 1)], 4, 64), ([(9000, 2), (3, 1), (5000, 1)], 8, 128), ([(2500, 300), (700, 1)], 2, 256)])
def test_long_requests_over_many_workgroups(dtype, lens, heads, dim):
    """Tiles whose keys are spread over many workgroups, and joined; twice the same bits."""
    print(f"long attention {dtype} {lens} dim={dim}", flush=True)
    case = batch(torch.Generator().manual_seed(8), lens, heads=heads, kv_heads=1, dim=dim, page=16, dtype=dtype)
    got = _attend(case)
    # the same in 64 bits on the GPU, a request at a time
    dev = {n: _cuda(x) for n, x in case.items()}
    for b, (c, n) in enumerate(lens):
        t = torch.arange(c + n, device="cuda")
        ids = dev["block_table"][b].long()[t // 16]
        k, v = (dev[x][ids, t % 16, 0].double() for x in ("k_cache", "v_cache"))
        s0 = int(case["starts"][b])
        for h in range(heads):
            x = dev["q"][s0:s0 + n, h].double()
            mask = t[None] > (c + torch.arange(n, device="cuda"))[:, None]
            w = torch.softmax((x @ k.t() * dim ** -0.5).masked_fill(mask, -math.inf), -1)
            want, a = w @ v, w @ v.abs()
            delta = (dim + 8) * 2.0 ** -24 * dim ** -0.5 * (x.abs() @ k.abs().t()).amax(-1, keepdim=True)
            half = 2.0 ** -8 if dtype == BF else 0.0
            room = a * (4 * delta + (c + n + 64) * 2.0 ** -24 + 2.0 ** -20 + half)
            room = room + (2.0 ** -8 if dtype == BF else 2.0 ** -24) * (want.abs() + room)
            compare(got[s0:s0 + n, h], want.cpu(), room.cpu())
    assert torch.equal(got, _attend(case))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("requests,lens,heads,kv_heads,dim", [
    (700, lambda b: (b * 7 % 40, 0 if b % 5 == 3 else 1), 2, 1, 64),      # more requests than a workgroup reads at once
    (300, lambda b: (b % 23, b % 4), 8, 2, 40), (40, lambda b: (600 - b, 1), 4, 2, 128),
    (3, lambda b: (900 + b, 200), 8, 4, 128), (9, lambda b: (400, 1 + 60 * (b % 2)), 10, 5, 64),
])
def test_many_requests(dtype, requests, lens, heads, kv_heads, dim):
    """Batches of many tiles, whose parts are joined a tile to a workgroup."""
    print(f"attention of {requests} requests {dtype} heads={heads}/{kv_heads} dim={dim}", flush=True)
    lens = [lens(b) for b in range(requests)]
    case = batch(torch.Generator().manual_seed(14), lens, heads=heads, kv_heads=kv_heads, dim=dim, page=16, dtype=dtype, pad_rows=2)
    got = _attend(case).cpu()
    assert bool(torch.isfinite(got).all()) and bool((got[-2:] == 0).all())
    # every 40th request against the plain form (its rows alone, as a batch of one)
    for b in range(0, requests, max(1, requests // 40)):
        s0, s1 = int(case["starts"][b]), int(case["starts"][b + 1])
        if s1 == s0:
            continue
        rows = slice(max(s0, s1 - 3), s1) if requests > 3 else slice(s1 - 2, s1)
        n = rows.stop - rows.start
        want, room = attention64(case["q"][rows], case["k_cache"], case["v_cache"], case["block_table"][b:b + 1], torch.tensor([0, n]),
                                 case["lengths"][b:b + 1])
        compare(got[rows], want, room)


def test_uninitialised_lds():
    """The debug build whose kernels first fill their LDS with NaN: the same bits."""
    from tjev_amd import _lib, paged_tables

    for lens, dim, dtype in (("ragged", 64, BF), ("chunk", 128, BF), ("chunk", 256, BF), ("drafts", 200, BF), ("decode", 128, F32), ("ragged", 256, F32)):
        case = batch(torch.Generator().manual_seed(15), LENS[lens], heads=8, kv_heads=2, dim=dim, page=16, dtype=dtype, gate=True)
        print(f"poisoned LDS {lens} dim={dim} {dtype}", flush=True)
        want = _attend(case)
        with _lib.library(_lib.LDS_POISON_PATH):
            assert torch.equal(_attend(case), want)
    i = torch.tensor([5, 0, 40], dtype=torch.int32, device="cuda")
    args = (i, i.flip(0), torch.arange(12, dtype=torch.int32, device="cuda").view(3, 4), torch.arange(9, dtype=torch.int32, device="cuda"))
    want = paged_tables(*args, page_size=16, tokens=60)
    with _lib.library(_lib.LDS_POISON_PATH):
        for x, y in zip(paged_tables(*args, page_size=16, tokens=60), want):
            assert torch.equal(x, y)


def test_offsets_past_32_bits():
    """A cache of 2^32 elements: its last pages written and read."""
    from tjev_amd import paged_append, paged_attention

    pages, page, heads, dim = 131073 + 4, 16, 8, 256
    print("attention past 2^32 elements", flush=True)
    kc, vc = (torch.empty(pages, page, heads, dim, dtype=BF, device="cuda") for _ in range(2))
    assert kc.numel() > 2 ** 32
    gen = torch.Generator().manual_seed(9)
    n = 40
    k, v, q = (torch.randn(n, heads, dim, generator=gen).to(BF) for _ in range(3))
    table = torch.tensor([[pages - 1, 2, pages - 3]], dtype=torch.int32)
    t = torch.arange(n)
    slots = table[0].long()[t // page] * page + t % page
    paged_append(k.cuda(), v.cuda(), kc, vc, slots.cuda())
    small = [torch.zeros(3, page, heads, dim, dtype=BF) for _ in range(2)]
    for c, x, big in zip(small, (k, v), (kc, vc)):
        c[t // page, t % page] = x
        assert torch.equal(big.view(-1, heads, dim)[slots.cuda()].cpu(), x)
    starts, lengths = torch.tensor([0, n], dtype=torch.int32), torch.tensor([n], dtype=torch.int32)
    got = paged_attention(q.cuda(), kc, vc, table.cuda(), starts.cuda(), lengths.cuda())
    want, room = attention64(q, *small, torch.tensor([[0, 1, 2]], dtype=torch.int32), starts, lengths)
    compare(got, want, room)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads", [4, 24])
def test_shared_pages(dtype, heads):
    """Requests whose first pages are the same (a common prompt), one of them with a page twice, gate and rows broadcast."""
    case = batch(torch.Generator().manual_seed(17), [(70, 3), (64, 9), (90, 1)], heads=heads, kv_heads=2, dim=64, page=16, dtype=dtype)
    table = case["block_table"]
    table[1, :3], table[2, 1:4], table[2, 4] = table[0, :3], table[0, 1:4], table[0, 1]
    case["gate"] = torch.randn(1, 1, 64, generator=torch.Generator().manual_seed(18)).to(dtype).expand(13, heads, 64)
    case["q"] = case["q"][:, :1].expand(13, heads, 64)
    print(f"attention over shared pages {dtype} heads={heads}", flush=True)
    want, room = attention64(*(case[n] for n in ("q", "k_cache", "v_cache", "block_table", "starts", "lengths")), gate=case["gate"])
    compare(_attend(case), want, room)


def test_as_many_keys_as_there_can_be():
    """A table whose entries are all one page, up to the last key that the operator takes."""
    from tjev_amd import paged_attention

    page, width = 65536, 32767
    gen = torch.Generator().manual_seed(19)
    kc, vc = (torch.randn(1, page, 1, 8, generator=gen).to(BF).cuda() for _ in range(2))
    q = torch.randn(1, 1, 8, generator=gen).to(BF).cuda()
    table, starts = torch.zeros(1, width, dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    print(f"attention over {width * page} keys", flush=True)
    got = paged_attention(q, kc, vc, table, starts, torch.tensor([width * page], dtype=torch.int32, device="cuda"))
    k, v, x = kc[0, :, 0].double(), vc[0, :, 0].double(), q[0, 0].double()
    w = torch.softmax(8 ** -0.5 * (k @ x), 0)
    want, a = w @ v, w @ v.abs()
    # sums of 2^31 numbers in 32 bits: a wave of a range adds fewer than 2^15 steps into one number, the weights' sum in
    # two additions a step and the result in eight (two products of 32 keys, a rounding for every 8), each off
    # by 2^-24 of it; the weights and the rounding as in attention64
    delta = 16 * 2.0 ** -24 * 8 ** -0.5 * float((k.abs() @ x.abs()).max())
    room = a * (4 * delta + 10 * (2 ** 15 + 64) * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -8)
    compare(got[0, 0], want.cpu(), (room + 2.0 ** -8 * (want.abs() + room)).cpu())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30, 3.0])
def test_scales(dtype, scale):
    case = batch(torch.Generator().manual_seed(13), [(60, 2), (30, 90), (9, 1)], heads=4, kv_heads=2, dim=64, page=16, dtype=dtype)
    print(f"attention {dtype} scale={scale}", flush=True)
    want, room = attention64(*(case[n] for n in ("q", "k_cache", "v_cache", "block_table", "starts", "lengths")), scale)
    compare(_attend(case, scale=scale), want, room)


def test_no_tokens():
    from tjev_amd import paged_attention

    c = torch.zeros(2, 16, 2, 64, device="cuda")
    z = torch.zeros(3, dtype=torch.int32, device="cuda")
    got = paged_attention(torch.empty(0, 4, 64, device="cuda"), c, c, torch.zeros(2, 1, dtype=torch.int32, device="cuda"), z, z[:2])
    assert got.shape == (0, 4, 64)
    got = paged_attention(torch.ones(5, 4, 64, device="cuda"), c, c, torch.zeros(2, 1, dtype=torch.int32, device="cuda"), z, z[:2])
    assert bool((got == 0).all())


# ---------------------------------------------------------------- together
def test_a_layer_served_step_by_step():
    """Two prompts in chunks, then decoded tokens beside a new prompt: tables, rotary positions, the write and gated attention on
    the GPU, against the same layer over each request's whole sequence in 64 bits. The tokens, pages and lengths of a
    step stay on the GPU."""
    from tjev_amd import paged_append, paged_attention, paged_tables, rotary_axes

    heads, kv, dim, page, half, sec = 8, 2, 64, 16, 16, (6, 5, 5)
    steps = [[40, 0, 25], [1, 30, 20], [1, 1, 1], [2, 1, 3], [1, 0, 1]]
    gen = torch.Generator().manual_seed(10)
    inv = 1e4 ** (-torch.arange(half, dtype=torch.float64) / half)
    total = [sum(s[b] for s in steps) for b in range(3)]
    seq = [{n: torch.randn(t, h, dim, generator=gen).to(BF) for n, h in (("q", heads), ("k", kv), ("v", kv), ("gate", heads))} for t in total]
    pos = [torch.stack([torch.arange(t), torch.arange(t) // 2, torch.randint(0, 9, (t,), generator=gen)]) for t in total]
    kc, vc = (torch.full((20, page, kv, dim), math.nan, dtype=BF, device="cuda") for _ in range(2))
    table = torch.full((3, 8), -1, dtype=torch.int32, device="cuda")
    free, taken = torch.randperm(20, generator=gen).int().cuda(), None
    cached, at = torch.zeros(3, dtype=torch.int32, device="cuda"), [0, 0, 0]
    outs = [[] for _ in range(3)]
    for step, new in enumerate(steps):
        print(f"layer step {step}: {new}", flush=True)
        rows = sum(new) + 2  # a padded batch
        x = {n: torch.cat([seq[b][n][at[b]:at[b] + k] for b, k in enumerate(new)] + [torch.full((2, *seq[0][n].shape[1:]), math.nan).to(BF)]).cuda()
             for n in seq[0]}
        p = torch.cat([pos[b][:, at[b]:at[b] + k] for b, k in enumerate(new)] + [torch.zeros(3, 2, dtype=torch.int64)], 1).cuda()
        t = paged_tables(cached, torch.tensor(new, dtype=torch.int32).cuda(), table, free, taken, page_size=page, tokens=rows)
        q, k = rotary_axes(x["q"], x["k"], p, inv.cuda(), sections=sec, interleaved=True)
        paged_append(k, x["v"], kc, vc, t.slots)
        y = paged_attention(q, kc, vc, t.block_table, t.starts, t.lengths, gate=x["gate"])
        assert bool((y[-2:] == 0).all())
        lo = 0
        for b, n in enumerate(new):
            outs[b].append(y[lo:lo + n].cpu())
            lo, at[b] = lo + n, at[b] + n
        table, cached, taken = t.block_table, t.lengths, t.taken
    assert int(taken) == sum(-(-t // page) for t in total)
    for b in range(3):
        q, k = (rotary64(seq[b][n][None], pos[b][:, None], inv, sec, True)[0][0].to(BF) for n in ("q", "k"))
        n = total[b]
        cache = [torch.zeros(n, 1, kv, dim, dtype=BF) for _ in range(2)]
        cache[0][:, 0], cache[1][:, 0] = k, seq[b]["v"]
        want, room = attention64(q, *cache, torch.arange(n, dtype=torch.int32)[None], torch.tensor([0, n]), torch.tensor([n]), gate=seq[b]["gate"])
        # q and k may be rounded to the neighbouring bf16 value: one step (2^-7) of each, in the scores
        a = torch.stack([(q[:, h].double().abs() @ k[:, h // 4].double().abs().t()).amax(-1) for h in range(heads)], 1)[..., None]
        vmax = seq[b]["v"].double().abs().max()
        moved = 4 * (2 * 2.0 ** -7) * dim ** -0.5 * a * vmax * torch.sigmoid(seq[b]["gate"].double())
        compare(torch.cat(outs[b]), want, room + moved)


@pytest.mark.parametrize("lens", ["decode", "ragged", "chunk"])
def test_captured_step_and_streams(lens):
    """A step captured into a graph and replayed on new lengths and values, with eager calls in between; two captured graphs
    and a side stream have workspaces of their own."""
    from tjev_amd import paged_attention

    case = batch(torch.Generator().manual_seed(11), LENS[lens], heads=8, kv_heads=2, dim=128, page=16, gate=True)
    dev = {n: _cuda(x) for n, x in case.items()}
    other = {n: _cuda(x) for n, x in batch(torch.Generator().manual_seed(12), [(3000, 1), (77, 9)], heads=8, kv_heads=2, dim=128, page=16).items()}
    print(f"attention captured {lens}", flush=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = paged_attention(**dev)
        paged_attention(**other)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(on_side, paged_attention(**dev))
    graphs = []
    for kw in (dev, other):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = paged_attention(**kw)
        graphs.append((g, y, kw))
    lengths = dev["lengths"].clone()
    for i in range(3):
        dev["q"].mul_(-1.25)
        dev["lengths"].copy_((lengths - i).clamp(min=0))
        for g, y, kw in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, y, kw in graphs:
            assert torch.equal(y, paged_attention(**kw))
