"""What the calls of the attention layers' operators hand to the library (CPU only, a stand-in takes its place): derivatives that
would be lost, recorded calls, views that are copied."""

from __future__ import annotations

import contextlib

import pytest
import torch
import torch.autograd.forward_ad as forward_ad


class _Library:
    """Notes the arguments of every call, and returns 0."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0

        return call


@pytest.fixture
def library(monkeypatch):
    from tjev_amd import _lib, paged, rotary

    lib = _Library()
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(_lib, "one_gpu", lambda what, devices: None)
    monkeypatch.setattr(_lib, "current_stream", lambda device: 0)
    monkeypatch.setattr(_lib, "on_device", lambda device: contextlib.nullcontext())
    yield lib
    for kept in (paged._tables_params, paged._append_params, paged._attention_params, rotary._checked, rotary._params):
        kept.cache_clear()  # checks that passed here alone


def _rotary(q, k=None):
    from tjev_amd import rotary_axes

    return rotary_axes(q, k, torch.zeros(1, 1, 3, dtype=torch.int64), torch.ones(8))


# ---------------------------------------------------------------- derivatives
@pytest.mark.parametrize("which", ["q", "k"])
@pytest.mark.parametrize("grad", [False, True])
def test_rotary_refuses_forward_derivatives(library, which, grad):
    """Dual inputs raise, as at the other differentiable operators: their tangents must not come back as none."""
    x = {n: torch.randn(1, 3, 2, 16) for n in "qk"}
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        x[which] = forward_ad.make_dual(x[which], torch.ones(1, 3, 2, 16))
        with pytest.raises(NotImplementedError, match="jvp"):
            _rotary(**x)


def test_rotary_refuses_forward_derivatives_of_its_gradient(library):
    x = torch.randn(1, 3, 2, 16, requires_grad=True)
    y, _ = _rotary(x)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(NotImplementedError, match="jvp"):
            torch.autograd.grad(y, x, d)


def test_rotary_within_a_dual_level(library):
    """Inputs without a tangent are turned as elsewhere."""
    with forward_ad.dual_level():
        y, _ = _rotary(torch.randn(1, 3, 2, 16))
        assert forward_ad.unpack_dual(y).tangent is None
    assert [n for n, _ in library.calls] == ["tjev_gdn_rotary"]


# ---------------------------------------------------------------- recorded calls
def _calls():
    """Each operator as a function of one tensor."""
    from tjev_amd import paged_append, paged_attention, paged_tables

    i = torch.zeros(2, dtype=torch.int32)
    table, starts = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    cache = torch.zeros(4, 16, 2, 64)

    def append(k):
        paged_append(k, k, cache, cache, torch.zeros(3, dtype=torch.int64))
        return cache + 0

    return {"rotary_axes": (lambda q: _rotary(q)[0], torch.randn(1, 3, 2, 16)),
            "paged_tables": (lambda t: paged_tables(i, i, t, i, page_size=16, tokens=4).slots, table),
            "paged_append": (append, torch.randn(3, 2, 64)),
            "paged_attention": (lambda q: paged_attention(q, cache, cache, table, starts, i), torch.randn(3, 4, 64))}


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("what", ["rotary_axes", "paged_tables", "paged_append", "paged_attention"])
@pytest.mark.parametrize("record", ["jit", "make_fx", "pre_dispatch"])
def test_recorded_calls_are_refused(library, what, record):
    """A launch is no operator of torch's: a record of it would be of its uninitialised output."""
    from torch.fx.experimental.proxy_tensor import make_fx

    f, x = _calls()[what]
    with pytest.raises(RuntimeError, match=f"{what}.*recorded"):
        torch.jit.trace(f, (x,), check_trace=False) if record == "jit" else make_fx(f, pre_dispatch=record == "pre_dispatch")(x)
    assert not library.calls


@pytest.mark.filterwarnings("ignore")
def test_a_recorded_rotary_gradient_is_refused(library):
    from torch.fx.experimental.proxy_tensor import make_fx

    q = torch.randn(1, 3, 2, 16, requires_grad=True)
    y, _ = _rotary(q)
    with pytest.raises(RuntimeError, match="rotary_axes.*recorded"):
        make_fx(lambda d: torch.autograd.grad(y, q, d)[0])(torch.ones_like(y))


@pytest.mark.parametrize("what", ["rotary_axes", "paged_tables", "paged_append", "paged_attention"])
def test_modes_that_only_look_on(library, what):
    """A dispatch mode that records nothing (a FLOP counter) lets the calls through."""
    from torch.utils.flop_counter import FlopCounterMode

    f, x = _calls()[what]
    library.tjev_gdn_paged_workspace_bytes = lambda p: 256
    with FlopCounterMode(display=False):
        f(x)
    assert len(library.calls) == 1


# ---------------------------------------------------------------- views
def _attend(**kw):
    from tjev_amd import paged_attention

    n = kw["q"].shape[0]
    cache = torch.zeros(4, 16, 2, 64, dtype=kw["q"].dtype)
    a = dict(k_cache=cache, v_cache=cache, block_table=torch.zeros(1, 3, dtype=torch.int32), starts=torch.tensor([0, n], dtype=torch.int32),
             lengths=torch.tensor([n], dtype=torch.int32))
    return paged_attention(**{**a, **kw})


Q, GATE, OUT = 2, 8, 9  # places in the library's call


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 2])
@pytest.mark.parametrize("which", ["q", "gate"])
def test_rows_off_16_bytes_are_copied(library, dtype, n, which):
    """One row of a wider tensor is contiguous, and no less a row off 16 bytes."""
    x = {"q": torch.zeros(n, 4, 64, dtype=dtype), "gate": torch.zeros(n, 4, 64, dtype=dtype)}
    x[which] = torch.zeros(n, 3 + 4 * 64, dtype=dtype)[:, 3:].view(n, 4, 64)
    assert x[which].data_ptr() % 16 and (n > 1 or x[which].is_contiguous())
    _attend(**x)
    (_, args), = [c for c in library.calls if c[0] == "tjev_gdn_paged_attention"]
    at, other = (Q, "gate") if which == "q" else (GATE, "q")
    assert args[at] % 16 == 0 and args[at] != x[which].data_ptr() and args[Q + GATE - at] == x[other].data_ptr()


@pytest.mark.parametrize("which", ["q", "gate", "out", "k_cache", "v_cache"])
def test_strides_of_one_row_do_not_matter(library, which):
    """Where a dim has one place its stride is no row's distance: such a view is neither copied nor refused."""
    x = {n: torch.zeros(1, 4, 64) for n in ("q", "gate", "out")}
    x.update({n: torch.zeros(4, 16, 1, 64) for n in ("k_cache", "v_cache")})
    old = x[which]
    x[which] = old.as_strided(old.shape, tuple(s if n > 1 else 1003 for n, s in zip(old.shape, old.stride())))
    _attend(**x)
    (_, args), = [c for c in library.calls if c[0] == "tjev_gdn_paged_attention"]
    p = args[0]._obj
    assert [args[i] for i in (Q, 3, 4, GATE, OUT)] == [x[n].data_ptr() for n in ("q", "k_cache", "v_cache", "gate", "out")]
    for s in (p.q_stride, p.gate_stride, p.out_stride, p.k_stride, p.v_stride):
        assert all(v % 4 == 0 for v in s)


# ---------------------------------------------------------------- gradients that there are none of
@pytest.mark.parametrize("which", ["q", "gate", "out", "k_cache", "v_cache"])
def test_attention_refuses_to_lose_a_gradient(library, which):
    x = {n: torch.zeros(2, 4, 64) for n in ("q", "gate", "out")}
    x.update({n: torch.zeros(4, 16, 2, 64) for n in ("k_cache", "v_cache")})
    with forward_ad.dual_level(), torch.no_grad():
        with pytest.raises(RuntimeError, match="paged_attention has no gradient"):
            _attend(**{**x, which: forward_ad.make_dual(x[which], torch.ones_like(x[which]))})
    x[which].requires_grad_(True)
    with pytest.raises(RuntimeError, match="paged_attention has no gradient"):
        _attend(**x)
    assert not [c for c in library.calls if c[0] == "tjev_gdn_paged_attention"]
    with torch.no_grad():
        _attend(**x)
    x[which] = x[which].detach()
    _attend(**x)
    assert len([c for c in library.calls if c[0] == "tjev_gdn_paged_attention"]) == 2


@pytest.mark.parametrize("which", ["k", "v", "k_cache", "v_cache"])
def test_append_refuses_to_lose_a_gradient(library, which):
    from tjev_amd import paged_append

    x = {n: torch.zeros(3, 2, 64) for n in ("k", "v")}
    x.update({n: torch.zeros(4, 16, 2, 64) for n in ("k_cache", "v_cache")})
    slots = torch.zeros(3, dtype=torch.int64)
    with forward_ad.dual_level(), torch.no_grad():
        with pytest.raises(RuntimeError, match="paged_append has no gradient"):
            paged_append(**{**x, which: forward_ad.make_dual(x[which], torch.ones_like(x[which]))}, slots=slots)
    x[which].requires_grad_(True)
    with pytest.raises(RuntimeError, match="paged_append has no gradient"):
        paged_append(**x, slots=slots)
    assert not library.calls
    with torch.no_grad():
        paged_append(**x, slots=slots)
    assert len(library.calls) == 1


# ---------------------------------------------------------------- sizes past 32 bits
FAR = 2 ** 32 + 16


def test_tables_refuse_pages_past_32_bits(library):
    from tjev_amd import paged_tables

    i, table = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32)
    for kw in (dict(page_size=FAR), dict(page_size=2 ** 31), dict(block_table=torch.zeros(1, 1, dtype=torch.int32).expand(2, FAR))):
        with pytest.raises(ValueError, match="2\\^31"):
            paged_tables(**{**dict(cached=i, new=i, block_table=table, free_pages=i, page_size=16, tokens=4), **kw})
    assert not library.calls


@pytest.mark.parametrize("shape", [(FAR, 16, 2, 64), (4, FAR, 2, 64)])
def test_caches_past_32_bits_are_refused(library, shape):
    from tjev_amd import paged

    cache = torch.zeros(1, 1, 1, 64).expand(shape)
    with pytest.raises(ValueError, match="2\\^31"):
        _attend(q=torch.zeros(1, 4, 64), k_cache=cache, v_cache=cache)
    # (no tensor of this size: a call's checks take the shape alone)
    like = lambda s: (s, (1 << 40, 128, 64, 1), torch.float32)  # noqa: E731
    with pytest.raises(ValueError, match="2\\^31"):
        paged._append_params(*(2 * ((3, 2, 64), (128, 64, 1), torch.float32)), *like(shape), *like(shape), (3,), torch.int64, (0,))
    assert not [c for c in library.calls if c[0] != "tjev_gdn_paged_workspace_bytes"]


def test_table_widths_past_32_bits_are_refused(library):
    with pytest.raises(ValueError, match="2\\^31"):
        _attend(q=torch.zeros(1, 4, 64), block_table=torch.zeros(1, 1, dtype=torch.int32).expand(1, FAR))


# ---------------------------------------------------------------- the kernels chosen by what one request may bring
def _workspace(**kw):
    """Bytes of a bf16 call's workspace: tiles of 128 rows have eight times the places of those of 16."""
    import ctypes

    from tjev_amd import _lib

    p = dict(tokens=64, requests=64, table_width=4096, pages=64, page_size=16, heads=16, kv_heads=4, dim=256, dtype=_lib.BF16, scale=1.0)
    return _lib.load().tjev_gdn_paged_workspace_bytes(ctypes.byref(_lib.PagedParams(**{**p, **kw})))


def test_unused_requests_do_not_count():
    """More rows per token than a streamed tile holds: no batch is of streamed tiles, whatever places its table has."""
    kw = dict(tokens=40, heads=20, kv_heads=1, dim=128)
    assert _workspace(**kw, requests=64) == _workspace(**kw, requests=40) > _workspace(**{**kw, "heads": 8}, requests=40)


@pytest.mark.parametrize("dim,heads,kv_heads", [(256, 16, 4), (128, 32, 4), (64, 16, 4)])
def test_the_most_new_tokens_choose(dim, heads, kv_heads):
    kw = dict(dim=dim, heads=heads, kv_heads=kv_heads)
    wide = _workspace(**kw, requests=1)
    for requests in (2, 64, 256):
        assert _workspace(**kw, requests=requests, max_new=64) == _workspace(**kw, requests=requests, max_new=10 ** 6) == wide
        assert _workspace(**kw, requests=requests, max_new=1) < wide
    assert _workspace(**kw, max_new=-1) == 0


@pytest.mark.parametrize("max_new", [0, -1, 2 ** 31])
def test_the_most_new_tokens_are_a_number_of_tokens(library, max_new):
    with pytest.raises(ValueError, match="max_new"):
        _attend(q=torch.zeros(1, 4, 64), max_new=max_new)
