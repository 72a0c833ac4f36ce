"""Rotary positions with several axes (tjev_amd.rotary) against the 64-bit form (tests/paged_cases.py): every pair
layout and section order, partial rotation, odd sizes that take the element-wise form, strided views, far
positions, and the gradient against the formula and against differences."""

from __future__ import annotations

import pytest
import torch

from paged_cases import rotary64, rotary_room

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _freqs(half, dtype=torch.float64):
    return (1e6 ** (-torch.arange(half, dtype=torch.float64) / max(1, half))).to(dtype)


def _check(got, x, pos, inv, sec, interleaved, adjacent, sign=1.0):
    want, mag = rotary64(x, pos, inv, sec, interleaved, adjacent, sign)
    room = rotary_room(want, mag, x.dtype)
    err = (got.double().cpu() - want).abs()
    assert bool((err <= room).all()), float((err / room.clamp(min=1e-30)).max())
    lanes = 2 * inv.shape[0]
    assert torch.equal(got[..., lanes:].cpu(), x[..., lanes:])  # passed on as they are


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape,half,sec", [
    ((2, 7, 4, 2, 64), 32, (12, 10, 10)), ((1, 1, 1, 1, 128), 64, (64,)), ((3, 33, 16, 4, 256), 32, (11, 11, 10)),
    ((1, 129, 5, 1, 128), 16, (4, 4, 4, 4)), ((2, 3, 3, 3, 40), 20, (10, 10)), ((1, 5, 2, 1, 38), 9, (3, 3, 3)),
    ((1, 4, 1, 1, 2), 1, (1,)), ((1, 2, 2, 2, 96), 40, (40, 0)), ((1, 1000, 24, 8, 64), 32, (16, 8, 8)),
])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("adjacent", [False, True])
def test_forward_and_gradient(dtype, shape, half, sec, interleaved, adjacent):
    from tjev_amd import rotary_axes

    if interleaved and any(n and a + len(sec) * (n - 1) >= half for a, n in enumerate(sec) if a):
        pytest.skip("not an interleaving")
    b, t, hq, hk, d = shape
    print(f"rotary {dtype} {shape} half={half} {sec} interleaved={interleaved} adjacent={adjacent}", flush=True)
    gen = torch.Generator().manual_seed(t + half)
    q, k, dq, dk = (torch.randn(b, t, h, d, generator=gen).to(dtype) for h in (hq, hk, hq, hk))
    pos = torch.randint(0, 5000, (len(sec), b, t), generator=gen)
    inv = _freqs(half)
    xq, xk = q.cuda().requires_grad_(True), k.cuda().requires_grad_(True)
    yq, yk = rotary_axes(xq, xk, pos.cuda(), inv.cuda(), sections=sec, interleaved=interleaved, adjacent=adjacent)
    gq, gk = torch.autograd.grad((yq, yk), (xq, xk), (dq.cuda(), dk.cuda()))
    for got, x, sign in ((yq, q, 1.0), (yk, k, 1.0), (gq, dq, -1.0), (gk, dk, -1.0)):
        _check(got.detach(), x, pos, inv, sec, interleaved, adjacent, sign)


@pytest.mark.parametrize("pos_dtype,freq_dtype", [(torch.int32, F32), (torch.int64, torch.float64)])
def test_far_positions(pos_dtype, freq_dtype):
    """Angles of 10^8 and more radians keep the bound: a 32-bit angle would be off by whole turns."""
    from tjev_amd import rotary_axes

    gen = torch.Generator().manual_seed(1)
    q = torch.randn(1, 64, 2, 64, generator=gen)
    pos = torch.randint(2 ** 30, 2 ** 31 - 1, (2, 1, 64), generator=gen).to(pos_dtype)
    pos[1] *= -1
    inv = _freqs(32, freq_dtype)
    print(f"far positions {pos_dtype} {freq_dtype}", flush=True)
    got, none = rotary_axes(q.cuda(), None, pos.cuda(), inv.cuda(), sections=(16, 16))
    assert none is None
    # the 64-bit angle itself is off by 2^-53 of 2^31 radians, in kernel and oracle: far below the room
    _check(got, q, pos, inv, (16, 16), False, False)


def test_views_and_shapes():
    """q, k as slices of one projection, without a batch dim, transposed to another order, empty."""
    from tjev_amd import rotary_axes

    gen = torch.Generator().manual_seed(2)
    qkv = torch.randn(19, (4 + 2 * 2) * 64, generator=gen).to(BF)
    pos, inv = torch.arange(19)[None], _freqs(32)
    dev = qkv.cuda()
    q, k = dev[:, :256].view(19, 4, 64), dev[:, 256:384].view(19, 2, 64)
    print("rotary of slices", flush=True)
    yq, yk = rotary_axes(q, k, pos[0].cuda(), inv.cuda())
    assert yq.shape == q.shape and yq.is_contiguous() and yk.is_contiguous()
    _check(yq[None], q.cpu()[None], pos[:, None], inv, (32,), False, False)
    _check(yk[None], k.cpu()[None], pos[:, None], inv, (32,), False, False)
    x = torch.randn(3, 5, 64, 7, generator=gen)  # [B, H, D, T]: its last dim is not the heads'
    v = x.permute(0, 3, 1, 2)
    print("rotary of a permuted view", flush=True)
    y, _ = rotary_axes(v.cuda(), None, torch.arange(7).expand(3, 7).cuda(), inv.cuda())
    _check(y, v, torch.arange(7).expand(1, 3, 7), inv, (32,), False, False)
    off = torch.randn(2 * 7 * 64 + 1, generator=gen).to(BF)[1:].view(1, 7, 2, 64)  # rows off 16 bytes
    print("rotary of a misaligned view", flush=True)
    y, _ = rotary_axes(off.cuda(), None, torch.arange(7)[None].cuda(), inv.cuda())
    _check(y, off, torch.arange(7)[None, None], inv, (32,), False, False)
    e, f = rotary_axes(torch.zeros(0, 4, 64, device="cuda"), torch.zeros(0, 2, 64, device="cuda"),
                       torch.zeros(0, dtype=torch.int64, device="cuda"), inv.cuda())
    assert e.shape == (0, 4, 64) and f.shape == (0, 2, 64)


def test_gradient_against_differences():
    """d/dq of a weighted sum by central differences, in fp32: the operator is linear in q, so a difference over
    2 is off by the forward's own rounding only."""
    from tjev_amd import rotary_axes

    gen = torch.Generator().manual_seed(3)
    q, w = torch.randn(1, 3, 2, 16, generator=gen), torch.randn(1, 3, 2, 16, generator=gen).cuda()
    pos, inv = torch.randint(0, 100, (2, 1, 3), generator=gen).cuda(), _freqs(6).cuda()
    f = lambda x: (rotary_axes(x, None, pos, inv, sections=(4, 2))[0].double() * w.double()).sum()  # noqa: E731
    x = q.cuda().requires_grad_(True)
    print("rotary differences", flush=True)
    (g,) = torch.autograd.grad(f(x), x)
    room = 2 * 2.0 ** -21 * float((q.abs().max() + 1) * 2 * w.abs().sum())
    for i in range(0, q.numel(), 7):
        e = torch.zeros_like(q).view(-1)
        e[i] = 1.0
        e = e.view(q.shape).cuda()
        with torch.no_grad():
            diff = float(f(q.cuda() + e) - f(q.cuda() - e)) / 2
        assert abs(diff - float(g.view(-1)[i])) <= room


def test_second_derivative():
    """The gradient's own gradient is the forward turn."""
    from tjev_amd import rotary_axes

    gen = torch.Generator().manual_seed(6)
    q, k, w = (torch.randn(1, 5, h, 32, generator=gen) for h in (2, 1, 2))
    pos, inv = torch.randint(0, 100, (2, 1, 5), generator=gen), _freqs(12)
    x, y, d = q.cuda().requires_grad_(True), k.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    print("rotary second derivative", flush=True)
    a, b = rotary_axes(x, y, pos.cuda(), inv.cuda(), sections=(7, 5))
    (g,) = torch.autograd.grad(a, x, d, create_graph=True)
    _check(g.detach(), w, pos, inv, (7, 5), False, False, -1.0)
    (h,) = torch.autograd.grad(g, d, q.cuda())
    _check(h, q, pos, inv, (7, 5), False, False)


def test_one_gradient_and_graph():
    """Only k needing one; a captured forward replayed on new values."""
    from tjev_amd import rotary_axes

    gen = torch.Generator().manual_seed(4)
    q, k = torch.randn(2, 9, 4, 64, generator=gen).to(BF), torch.randn(2, 9, 2, 64, generator=gen).to(BF)
    pos, inv = torch.randint(0, 100, (3, 2, 9), generator=gen), _freqs(32)
    xk = k.cuda().requires_grad_(True)
    print("rotary of one gradient", flush=True)
    _, yk = rotary_axes(q.cuda(), xk, pos.cuda(), inv.cuda(), sections=(12, 10, 10))
    (g,) = torch.autograd.grad(yk, xk, torch.ones_like(yk))
    _check(g, torch.ones_like(k), pos, inv, (12, 10, 10), False, False, -1.0)
    bq, bp, bi = q.cuda(), pos.cuda(), inv.cuda()
    call = lambda: rotary_axes(bq, None, bp, bi, sections=(12, 10, 10))[0]  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    print("rotary captured", flush=True)
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call()
    for i in range(3):
        bq.copy_((q.float() * (i + 1)).to(BF))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, call())


def test_captured_gradient():
    """Forward and gradient captured into a graph, replayed on new values beside eager calls."""
    from tjev_amd import rotary_axes

    gen = torch.Generator().manual_seed(7)
    q, k = (torch.randn(2, 40, h, 64, generator=gen).to(BF).cuda().requires_grad_(True) for h in (4, 2))
    dq, dk = torch.randn(2, 40, 4, 64, generator=gen).to(BF).cuda(), torch.randn(2, 40, 2, 64, generator=gen).to(BF).cuda()
    pos, inv = torch.randint(0, 1000, (3, 2, 40), generator=gen).cuda(), _freqs(32).cuda()

    def step():
        a, b = rotary_axes(q, k, pos, inv, sections=(12, 10, 10), interleaved=True)
        return [a.detach(), b.detach(), *torch.autograd.grad((a, b), (q, k), (dq, dk))]

    print("rotary gradient captured", flush=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        with torch.no_grad():
            q.mul_(-1.5)
            dq.mul_(1.25)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, step()):
            assert torch.equal(x, y)
