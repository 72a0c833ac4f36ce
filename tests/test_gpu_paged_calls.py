"""The paged cache's operators (tjev_amd.paged) called in ways that a served batch comes to: views off 16 bytes, tables with
unused places, several streams, workspaces that hold anything; against their plain 64-bit forms (tests/paged_cases.py)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from paged_cases import attention64, batch, compare

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
NAMES = ("q", "k_cache", "v_cache", "block_table", "starts", "lengths")


def _attend(case, **kw):
    from tjev_amd import paged_attention

    return paged_attention(**{n: x.cuda() if isinstance(x, torch.Tensor) and not x.is_cuda else x for n, x in {**case, **kw}.items()})


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n", [1, 2])
def test_rows_off_16_bytes(dtype, n):
    """q and gate of one token, contiguous and off 16 bytes, and of two."""
    case = batch(torch.Generator().manual_seed(21), [(40, n)], heads=4, kv_heads=2, dim=64, page=16, dtype=dtype, gate=True)
    want, room = attention64(*(case[x] for x in NAMES), gate=case["gate"])
    off = {}
    for x in ("q", "gate"):
        wide = torch.zeros(n, 3 + 4 * 64, dtype=dtype, device="cuda")
        off[x] = wide[:, 3:].view(n, 4, 64)
        off[x].copy_(case[x])
    print(f"attention of rows off 16 bytes {dtype} n={n}", flush=True)
    compare(_attend(case, **off), want, room)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides_of_one_row(dtype):
    """One token into a row of a wider tensor, over a cache of one key head whose heads' stride is no multiple of 16 bytes."""
    case = batch(torch.Generator().manual_seed(22), [(70, 1)], heads=4, kv_heads=1, dim=64, page=16, dtype=dtype)
    want, room = attention64(*(case[x] for x in NAMES))
    wide = torch.full((1, 1003), 7.0, dtype=dtype, device="cuda")
    out = wide[:, 8:264].view(1, 4, 64)
    caches = {}
    for x in ("k_cache", "v_cache"):
        c = case[x].cuda()
        caches[x] = c.as_strided(c.shape, (*c.stride()[:2], 1003, 1))
    print(f"attention into one row {dtype}", flush=True)
    assert _attend(case, out=out, **caches) is out
    compare(out, want, room)
    assert bool((wide[:, :8] == 7).all()) and bool((wide[:, 264:] == 7).all())


def _with_idle(case, places, requests):
    """The case's requests at these places of a table of so many, the others unused."""
    starts, lengths = torch.zeros(requests + 1, dtype=torch.int32), torch.zeros(requests, dtype=torch.int32)
    table = torch.full((requests, case["block_table"].shape[1]), -1, dtype=torch.int32)
    for b, at in enumerate(places):
        starts[at + 1:] = case["starts"][b + 1]
        lengths[at], table[at] = case["lengths"][b], case["block_table"][b]
    return dict(case, block_table=table, starts=starts, lengths=lengths)


def _us(case, calls=10):
    """Microseconds of a call among others, the quickest of five runs."""
    a, b, best = torch.cuda.Event(True), torch.cuda.Event(True), float("inf")
    for _ in range(5):
        a.record()
        for _ in range(calls):
            _attend(case)
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b) * 1e3 / calls)
    return best


@pytest.mark.parametrize("new", [1, 40])
def test_gaps_of_unused_requests(new):
    """Requests a thousand unused ones apart: the same bits as side by side, and less than twice their time (55 and 60 us for one
    token each; looked at one by one, the unused ones took 360 us more)."""
    lens = [(80000, new), (79900, new), (80100, new)]
    case = batch(torch.Generator().manual_seed(23), lens, heads=4, kv_heads=1, dim=128, page=64, extra_pages=0)
    cases = [{n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in _with_idle(case, places, 2003).items()}
             for places in ((1000, 1001, 1002), (0, 1001, 2002))]
    print(f"attention over gaps of unused requests, {new} tokens each", flush=True)
    near, far = (_attend(c) for c in cases)
    assert torch.equal(near, far) and torch.equal(near[:new], _attend(cases[0])[:new])
    near, far = (_us(c) for c in cases)
    print(f"{near:.1f} us side by side, {far:.1f} us apart", flush=True)
    assert far < 2 * near


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(32, 2, 200, 1), (8, 2, 64, 16), (16, 4, 256, 16)])
def test_unused_requests_between_others(dtype, heads, kv_heads, dim, page):
    """Every second to fifth request unused, and ranges that go on behind them: right, and the same bits every time."""
    lens = [((b * 37) % 340, 0 if b % 5 in (0, 3) or b % 7 == 2 else 1 + (b * b) % 9) for b in range(90)]
    case = batch(torch.Generator().manual_seed(27), lens, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    print(f"attention between unused requests {dtype} {heads}/{kv_heads} of {dim} page={page}", flush=True)
    want, room = attention64(*(case[x] for x in NAMES))
    case = {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in case.items()}
    got = _attend(case)
    compare(got, want, room)
    for _ in range(50):
        assert torch.equal(_attend(case), got)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,lens,requests", [
    (8, 2, 64, [(700, 6), (0, 1), (90, 40)], 60), (16, 4, 256, [(3000, 64)], 64), (40, 2, 128, [(50, 1), (600, 1)], 9),
    (8, 1, 64, [(900, 3), (40, 1)], 300), (6, 3, 40, [(2000, 90), (5, 9)], 200), (4, 4, 200, [(77, 50), (1, 1)], 120),
])
def test_unused_requests_and_the_most_new_tokens(dtype, heads, kv_heads, dim, lens, requests):
    """More places than tokens, and bounds on a request's tokens: the true one, none, and (which costs time alone) wrong ones."""
    case = batch(torch.Generator().manual_seed(24), lens, heads=heads, kv_heads=kv_heads, dim=dim, page=16, dtype=dtype, gate=True)
    want, room = attention64(*(case[x] for x in NAMES), gate=case["gate"])
    case = _with_idle(case, [b * (requests - 1) // max(1, len(lens) - 1) for b in range(len(lens))], requests)
    most = max(n for _, n in lens)
    for max_new in (None, most, 1, 5, 10 ** 6):
        print(f"attention {dtype} {heads}/{kv_heads} of {dim} {lens} in {requests} places, max_new={max_new}", flush=True)
        compare(_attend(case, max_new=max_new), want, room)


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 4, 256), (32, 4, 128), (32, 8, 64)])
def test_a_prompt_among_unused_requests(heads, kv_heads, dim):
    """64 tokens over 30000 in one of 256 places of a table, with their bound: less than 1.5 times their time alone in it (74 and
    83 us at head dim 256; streamed, 283)."""
    case = batch(torch.Generator().manual_seed(25), [(30000, 64)], heads=heads, kv_heads=kv_heads, dim=dim, page=64, extra_pages=0)
    alone, among = ({n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in c.items()} for c in (case, _with_idle(case, [128], 256)))
    print(f"attention of one prompt {heads}/{kv_heads} of {dim}", flush=True)
    alone, among = _us(alone), _us(dict(among, max_new=64))
    print(f"{alone:.1f} us alone, {among:.1f} us among unused requests", flush=True)
    assert among < 1.5 * alone


# tiles of few rows and of many, whose parts are joined by several workgroups each, by one, and by as many as there are
SPLIT = {
    "streamed, few": ([(9000, 1)], 8, 2, 128, None, 0), "streamed, many": ([(900, 1)] * 70, 8, 2, 128, None, 0),
    "wide, few": ([(3000, 64)], 16, 4, 256, None, 0), "wide, many": ([(1500, 70)] * 6, 16, 4, 128, None, 0),
    "wide, counted": ([(3000, 64)], 16, 4, 256, 64, 64), "wide, counted, many": ([(700, 1)] * 40 + [(2000, 64)], 16, 4, 64, 64, 0),
}


def _split(kind, dtype=BF):
    lens, heads, kv_heads, dim, max_new, requests = SPLIT[kind]
    case = batch(torch.Generator().manual_seed(26), lens, heads=heads, kv_heads=kv_heads, dim=dim, page=16, dtype=dtype, gate=True)
    if requests:
        case = _with_idle(case, [requests // 2], requests)
    return {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in dict(case, max_new=max_new).items()}


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kind", sorted(SPLIT))
def test_poisoned_workspace(monkeypatch, dtype, kind):
    """The poison mode, and a workspace and an output that hold anything: the same bits."""
    case = _split(kind, dtype)
    print(f"poisoned workspace: {kind} {dtype}", flush=True)
    want = _attend(case)
    assert bool(torch.isfinite(want).all())
    monkeypatch.setenv("TJEV_GDN_POISON", "1")
    assert torch.equal(_attend(case), want)
    monkeypatch.delenv("TJEV_GDN_POISON")
    empty = torch.empty

    def filled(*args, **kw):
        x = empty(*args, **kw)
        return x.fill_(0xFF) if x.dtype == torch.uint8 else x  # the workspace: NaN, and notes of -1 parts

    monkeypatch.setattr(torch, "empty", filled)
    out = torch.full_like(want, float("nan"))
    assert torch.equal(_attend(case, out=out), want)


def test_poison_reaches_the_workspace(monkeypatch):
    """All of it but the ranges' notes, which are numbers."""
    from tjev_amd import _lib, paged

    case = _split("streamed, few")
    lib, held = _lib.load(), {}
    real = paged._attention_params

    def keep(*args):
        held["p"], held["need"] = real(*args)
        return held["p"], held["need"]

    monkeypatch.setattr(paged, "_attention_params", keep)
    want = _attend(case)
    ws, out = torch.zeros(held["need"], dtype=torch.uint8, device="cuda"), torch.empty_like(want)
    monkeypatch.setenv("TJEV_GDN_POISON", "1")
    print("poison in the workspace", flush=True)
    _lib.check_status(lib.tjev_gdn_paged_attention(
        held["p"], ctypes.c_void_p(_lib.current_stream(ws.device)), *(case[n].data_ptr() for n in NAMES), case["gate"].data_ptr(),
        out.data_ptr(), ws.data_ptr(), held["need"]))
    assert torch.equal(out, want)
    # ranges of two places of 16 rows (results, maximum, sum) and a note; places that no part went to are left NaN
    place, note = 16 * (128 + 2) * 4, 32
    notes = held["need"] // (2 * place + note) * note
    assert bool(torch.isnan(ws[:-notes].view(torch.float32)).any()) and not bool((ws[-notes:].view(torch.int32) == 0x7FC00000).any())


@pytest.mark.parametrize("kinds", [("streamed, few", "wide, few"), ("wide, many", "wide, counted"), ("streamed, many", "streamed, many")])
def test_two_calls_at_once(kinds):
    """Calls queued on two streams without a wait between them, and graphs replayed on both at once: a workspace of its own each."""
    cases = [_split(k) for k in kinds]
    want = [_attend(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    print(f"two calls at once: {kinds}", flush=True)
    torch.cuda.synchronize()
    got = [[] for _ in cases]
    for _ in range(12):
        for s, c, g in zip(streams, cases, got):
            with torch.cuda.stream(s):
                g.append(_attend(c))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(x, w) for x in g)
    graphs = []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ys = [_attend(c) for _ in range(3)]
        graphs.append((graph, ys))
    for _ in range(3):
        for _, ys in graphs:
            for y in ys:
                y.zero_()
        torch.cuda.synchronize()
        for s, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for w, (_, ys) in zip(want, graphs):
            assert all(torch.equal(y, w) for y in ys)
