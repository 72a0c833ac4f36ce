"""The drafted step's operators on the host (CPU only): refusals come before a launch, nothing falls back to the CPU, derivatives and
recorded calls raise, views are copied where they have to be; and the plain forms that the GPU tests compare with, checked against
mistakes planted in them."""

from __future__ import annotations

import contextlib
import ctypes
import os
import random
import shutil
import subprocess
from pathlib import Path

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from draft_cases import bits_of, fork_walk, random_tree, tree_attention64, tree_walk, verify_walk
from paged_cases import attention64, batch
from test_attention_calls_host import _Library

BF = torch.bfloat16


@pytest.fixture
def library(monkeypatch):
    from tjev_amd import _lib, drafts, paged

    lib = _Library()
    lib.addresses = []

    def compact(p, stream, ks, vs, *rest):
        lib.calls.append(("tjev_gdn_paged_compact", (p, stream, ks, vs, *rest)))
        lib.addresses = [list((ctypes.c_uint64 * p._obj.layers).from_address(a)) for a in (ks, vs)]
        return 0

    lib.tjev_gdn_paged_compact = compact
    lib.tjev_gdn_verify_workspace_bytes = lambda p: 256
    lib.tjev_gdn_fork_workspace_bytes = lambda p: 256
    lib.tjev_gdn_paged_tree_workspace_bytes = lambda p: 256
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(_lib, "one_gpu", lambda what, devices: None)
    monkeypatch.setattr(_lib, "current_stream", lambda device: 0)
    monkeypatch.setattr(_lib, "on_device", lambda device: contextlib.nullcontext())
    yield lib
    for kept in (paged._attention_params, paged._compact_params, paged._fork_params, drafts._tree_params,
                 drafts._verify_params):
        kept.cache_clear()  # checks that passed here alone


def _i(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _args(what, **kw):
    cache = torch.zeros(4, 16, 2, 64)
    a = {"draft_tree": dict(parents=_i(5), starts=_i(3), lengths=_i(2), max_new=4),
         "verify_drafts": dict(tokens=_i(5), target_probs=torch.zeros(5, 11), starts=_i(3), uniforms=torch.zeros(5), parents=None, draft_probs=None,
                               max_new=4),
         "paged_tree_attention": dict(q=torch.zeros(3, 4, 64), k_cache=cache, v_cache=cache.clone(), block_table=_i(2, 3), starts=_i(3), lengths=_i(2),
                                      ancestors=torch.zeros(3, 1, dtype=torch.int64)),
         "paged_compact": dict(caches=[(cache, cache.clone())], block_table=_i(2, 3), starts=_i(3), lengths=_i(2), path=_i(2, 4), kept=_i(2)),
         "paged_fork": dict(caches=[(cache, cache.clone())], block_table=_i(2, 3), lengths=_i(2), sources=_i(3), keep=_i(3), free_pages=_i(5), taken=_i(1),
                            shared=_i(4), page_size=16)}[what]
    a.update(kw)
    return a


def _call(what, **kw):
    import tjev_amd

    return getattr(tjev_amd, what)(**_args(what, **kw))


OPERATORS = ("draft_tree", "verify_drafts", "paged_tree_attention", "paged_compact", "paged_fork")


@pytest.mark.parametrize("what", OPERATORS)
def test_no_cpu_fallback(what):
    with pytest.raises(RuntimeError, match=f"{what} runs on the GPU"):
        _call(what)


CACHE = torch.zeros(4, 16, 2, 64)
FAR = 2 ** 32 + 16


@pytest.mark.parametrize("what,bad,match", [
    ("draft_tree", dict(parents=_i(5, 1)), "parents"), ("draft_tree", dict(parents=torch.zeros(5)), "int32 or int64"),
    ("draft_tree", dict(starts=_i(1)), "starts"), ("draft_tree", dict(lengths=_i(3)), "lengths"), ("draft_tree", dict(max_new=0), "max_new"),
    ("draft_tree", dict(max_new=1 << 31), "max_new"), ("draft_tree", dict(lengths=torch.zeros(2)), "int32 or int64"),
    ("verify_drafts", dict(target_probs=torch.zeros(5, 11, dtype=torch.float16)), "float32 or bfloat16"),
    ("verify_drafts", dict(target_probs=torch.zeros(5)), "target_probs"), ("verify_drafts", dict(target_probs=torch.zeros(5, 0)), "target_probs"),
    ("verify_drafts", dict(tokens=_i(4)), "tokens"), ("verify_drafts", dict(tokens=torch.zeros(5)), "tokens"),
    ("verify_drafts", dict(uniforms=torch.zeros(5, dtype=torch.float64)), "uniforms"), ("verify_drafts", dict(uniforms=torch.zeros(4)), "uniforms"),
    ("verify_drafts", dict(starts=_i(1)), "starts"), ("verify_drafts", dict(starts=torch.zeros(3)), "starts"),
    ("verify_drafts", dict(parents=_i(4)), "parents"), ("verify_drafts", dict(parents=torch.zeros(5)), "parents"),
    ("verify_drafts", dict(draft_probs=torch.zeros(5, 12)), "draft_probs"), ("verify_drafts", dict(draft_probs=torch.zeros(5, 11, dtype=BF)), "draft_probs"),
    ("verify_drafts", dict(draft_probs=torch.zeros(5, 11), parents=_i(5)), "chains"), ("verify_drafts", dict(max_new=0), "max_new"),
    ("verify_drafts", dict(max_new=1 << 31), "max_new"),
    ("paged_tree_attention", dict(ancestors=torch.zeros(3, 1, dtype=torch.int32)), "ancestors"),
    ("paged_tree_attention", dict(ancestors=torch.zeros(4, 1, dtype=torch.int64)), "ancestors"),
    ("paged_tree_attention", dict(ancestors=torch.zeros(3, 0, dtype=torch.int64)), "ancestors"),
    ("paged_tree_attention", dict(ancestors=torch.zeros(3, dtype=torch.int64)), "ancestors"),
    ("paged_tree_attention", dict(ancestors=torch.zeros(3, 1, dtype=torch.int64).expand(3, FAR)), "2\\^31"),
    ("paged_tree_attention", dict(q=torch.zeros(3, 3, 64)), "groups"), ("paged_tree_attention", dict(starts=_i(2)), "starts"),
    ("paged_tree_attention", dict(gate=torch.zeros(3, 4, 32)), "gate"), ("paged_tree_attention", dict(max_new=0), "max_new"),
    ("paged_compact", dict(caches=[(CACHE,)]), "pairs"), ("paged_compact", dict(caches=[(CACHE, CACHE[:3])]), "caches"),
    ("paged_compact", dict(caches=[(CACHE, CACHE), (CACHE, CACHE.transpose(0, 1).contiguous().transpose(0, 1))]), "alike"),
    ("paged_compact", dict(caches=[(CACHE.half(), CACHE.half())]), "float32 or bfloat16"),
    ("paged_compact", dict(caches=[(CACHE[0], CACHE[0])]), "caches"), ("paged_compact", dict(caches=[(CACHE[:0], CACHE[:0])]), "without"),
    ("paged_compact", dict(caches=[(CACHE[:, :1].expand(4, 16, 2, 64),) * 2]), "expanded"),
    ("paged_compact", dict(caches=[(CACHE.transpose(2, 3), CACHE.transpose(2, 3))]), "contiguous"),
    ("paged_compact", dict(block_table=_i(2, 0)), "block_table"), ("paged_compact", dict(block_table=torch.zeros(2, 3, dtype=torch.int64)), "int32"),
    ("paged_compact", dict(block_table=_i(8193, 1)), "requests"), ("paged_compact", dict(starts=_i(2)), "starts"),
    ("paged_compact", dict(kept=_i(3)), "kept"), ("paged_compact", dict(path=_i(3, 4)), "path"), ("paged_compact", dict(path=_i(2, 0)), "path"),
    ("paged_compact", dict(path=torch.zeros(2, 4)), "int32 or int64"),
    ("paged_compact", dict(block_table=torch.zeros(1, 1, dtype=torch.int32).expand(2, FAR)), "2\\^31"),
    ("paged_fork", dict(page_size=8), "pages of 8"), ("paged_fork", dict(shared=_i(5)), "5 pages"), ("paged_fork", dict(page_size=0, caches=[]), "one token"),
    ("paged_fork", dict(block_table=_i(0, 3)), "block_table"), ("paged_fork", dict(lengths=_i(3)), "lengths"), ("paged_fork", dict(keep=_i(2)), "keep"),
    ("paged_fork", dict(sources=_i(0)), "sources"), ("paged_fork", dict(sources=_i(8193), keep=None), "sources"), ("paged_fork", dict(taken=_i(2)), "taken"),
    ("paged_fork", dict(free_pages=_i(5, 1)), "free_pages"), ("paged_fork", dict(shared=_i(4, 1)), "shared"), ("paged_fork", dict(keep=torch.zeros(3)), "int32 or int64"),
    ("paged_fork", dict(caches=[], shared=_i(0)), "shared"),
])
def test_refusals(library, what, bad, match):
    with pytest.raises(ValueError, match=match):
        _call(what, **bad)
    assert not [c for c in library.calls if not c[0].endswith("bytes")]


@pytest.mark.parametrize("what", ["paged_compact", "paged_fork"])
def test_a_cache_given_twice(library, what):
    """Its tokens would be moved twice. Keys and values in one tensor are two caches."""
    joint, other = torch.zeros(4, 16, 2, 2, 64), torch.zeros(4, 16, 2, 64)
    k, v = joint[..., 0, :], joint[..., 1, :]
    for caches in ([(k, k)], [(k, v), (k, v)], [(k, v), (v, k)]):
        with pytest.raises(ValueError, match="twice"):
            _call(what, caches=caches)
    assert not [c for c in library.calls if not c[0].endswith("bytes")]
    _call(what, caches=[(k, v)])
    _call(what, caches=[(other, other + 1)])


def test_products_past_32_bits(library):
    """A table of 2^31 entries: its rows are counted in 32 bits."""
    table = torch.zeros(1, 1, dtype=torch.int32).expand(2048, 1 << 20)
    with pytest.raises(ValueError, match="2\\^31"):
        _call("paged_fork", block_table=table, lengths=_i(2048))
    assert not library.calls


@pytest.mark.parametrize("what,which", [("verify_drafts", "target_probs"), ("verify_drafts", "draft_probs"), ("verify_drafts", "uniforms"),
                                        ("paged_tree_attention", "q"), ("paged_tree_attention", "k_cache"), ("paged_tree_attention", "gate"),
                                        ("paged_tree_attention", "out"), ("paged_compact", "caches"), ("paged_fork", "caches")])
def test_gradients_are_not_lost(library, what, which):
    x = {"target_probs": torch.zeros(5, 11), "draft_probs": torch.zeros(5, 11), "uniforms": torch.zeros(5), "q": torch.zeros(3, 4, 64), "k_cache": CACHE.clone(),
         "gate": torch.zeros(3, 4, 64), "out": torch.zeros(3, 4, 64), "caches": CACHE.clone()}[which]
    give = (lambda t: dict(caches=[(CACHE, CACHE + 1), (CACHE + 2, t)])) if which == "caches" else (lambda t: {which: t})
    with forward_ad.dual_level(), torch.no_grad():
        with pytest.raises(RuntimeError, match=f"{what} has no gradient"):
            _call(what, **give(forward_ad.make_dual(x, torch.ones_like(x))))
    x.requires_grad_(True)
    with pytest.raises(RuntimeError, match=f"{what} has no gradient"):
        _call(what, **give(x))
    assert not [c for c in library.calls if not c[0].endswith("bytes")]
    with torch.no_grad():
        _call(what, **give(x))
    assert len(library.calls) == 1


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("what", OPERATORS)
@pytest.mark.parametrize("record", ["jit", "make_fx", "pre_dispatch"])
def test_recorded_calls_are_refused(library, what, record):
    from torch.fx.experimental.proxy_tensor import make_fx

    def f(lengths):
        name = "starts" if what == "verify_drafts" else "lengths"
        r = _call(what, **{name: lengths})
        return r if isinstance(r, torch.Tensor) else r[0]

    x = _i(3) if what == "verify_drafts" else _i(2)
    with pytest.raises(RuntimeError, match=f"{what}.*recorded"):
        torch.jit.trace(f, (x,), check_trace=False) if record == "jit" else make_fx(f, pre_dispatch=record == "pre_dispatch")(x)
    assert not library.calls


@pytest.mark.parametrize("what", OPERATORS)
def test_modes_that_only_look_on(library, what):
    from torch.utils.flop_counter import FlopCounterMode

    with FlopCounterMode(display=False):
        _call(what)
    assert len(library.calls) == 1


def test_strides_reach_the_library(library):
    """Rows of a wider tensor as they are; a last dim that is not contiguous copied; one row's stride 0."""
    wide = torch.zeros(5, 30)
    _call("verify_drafts", target_probs=wide[:, 3:14], draft_probs=torch.zeros(11, 5).t())
    (_, args), = library.calls
    p = args[0]._obj
    assert args[6] == wide.data_ptr() + 12 and p.target_stride == 30 and p.draft_stride == 11 and p.vocab == 11
    library.calls.clear()
    _call("verify_drafts", tokens=_i(1), uniforms=torch.zeros(1), target_probs=torch.zeros(1, 11).as_strided((1, 11), (-3 % 7, 1)))
    assert library.calls[0][1][0]._obj.target_stride == 0


def test_layers_reach_the_library(library):
    """Every layer's addresses in order, the strides once; no layers at all."""
    pairs = [tuple(torch.zeros(4, 2, 16, 64).transpose(1, 2) for _ in range(2)) for _ in range(20)]
    _call("paged_compact", caches=pairs)
    (_, args), = library.calls
    p = args[0]._obj
    assert p.layers == 20 and list(p.k_stride) == [2048, 64, 1024] and (p.pages, p.page_size, p.kv_heads, p.dim) == (4, 16, 2, 64)
    assert library.addresses == [[k.data_ptr() for k, _ in pairs], [v.data_ptr() for _, v in pairs]]
    library.calls.clear()
    _call("paged_fork", caches=[])
    p = library.calls[0][1][0]._obj
    assert p.layers == 0 and p.pages == 4 and p.page_size == 16 and p.n_free == 5 and p.new_requests == 3


# ---------------------------------------------------------------- the C ABI, with made-up addresses never launched on
def _fake(n):
    if torch.cuda.is_available():
        pytest.skip("host-side refusals with made-up device addresses: CPU only")
    return [ctypes.c_void_p(4096 * (i + 1)) for i in range(n)]


def _draft(**kw):
    from tjev_amd import _lib

    return ctypes.byref(_lib.DraftParams(**{**dict(tokens=5, max_new=4, requests=2, vocab=11, target_stride=11, draft_stride=11), **kw}))


def _pages(**kw):
    from tjev_amd import _lib

    return ctypes.byref(_lib.PagesParams(**{**dict(max_new=4, n_free=5, requests=2, new_requests=3, table_width=3, pages=4, page_size=16, kv_heads=2, dim=64,
                                                   dtype=1, layers=2, k_stride=(2048, 128, 64), v_stride=(2048, 128, 64)), **kw}))


def test_drafts_c_abi():
    from tjev_amd import _lib

    lib, f = _lib.load(), _fake(12)
    said = lambda: lib.tjev_gdn_last_error().decode()  # noqa: E731
    for bad, status in ((dict(requests=0), 1), (dict(tokens=-1), 1), (dict(max_new=0), 1), (dict(tokens=1 << 31), 1), (dict(requests=1 << 25), 2),
                        (dict(max_new=1 << 31), 1)):
        assert lib.tjev_gdn_draft_tree(_draft(**bad), None, *f[:5]) == status, (bad, said())
    assert lib.tjev_gdn_draft_tree(None, None, *f[:5]) == 1 and lib.tjev_gdn_draft_tree(_draft(tokens=0), None, *[None] * 5) == 0
    for i in range(5):
        a = list(f[:5])
        a[i] = None
        assert lib.tjev_gdn_draft_tree(_draft(), None, *a) == 1 and "null" in said()
    need = lib.tjev_gdn_verify_workspace_bytes(_draft())
    assert need > 0
    for bad, status in ((dict(requests=65536), 2), (dict(vocab=0), 1), (dict(dtype=2), 1), (dict(max_new=0), 1)):
        assert lib.tjev_gdn_verify_workspace_bytes(_draft(**bad)) == 0
        assert lib.tjev_gdn_verify_drafts(_draft(**bad), None, f[0], None, *f[2:10], 1 << 40) == status, (bad, said())
    call = lambda a, n=need: lib.tjev_gdn_verify_drafts(_draft(), None, *a, n)  # noqa: E731
    a = [f[0], None, *f[2:10]]
    assert call(a, need - 1) == 3
    for i in (0, 2, 3, 4, 6, 7, 8):
        b = list(a)
        b[i] = None
        assert call(b) == 1 and "null" in said(), i
    b = list(a)
    b[1] = f[10]
    assert call(b) == 1 and "chains" in said()
    b = list(a)
    b[9] = ctypes.c_void_p(4096 + 128)
    assert call(b) == 1 and "256" in said()
    b = list(a)
    b[4] = ctypes.c_void_p(4096 + 2)
    assert call(b) == 1 and "aligned" in said()


def test_pages_c_abi():
    from tjev_amd import _lib

    lib, f = _lib.load(), _fake(20)
    said = lambda: lib.tjev_gdn_last_error().decode()  # noqa: E731
    ks, vs = ((ctypes.c_void_p * 2)(1 << 20, 1 << 21) for _ in range(2))
    compact = lambda p, a=None, k=ks, v=vs: lib.tjev_gdn_paged_compact(p, None, k, v, *(a or f[:6]))  # noqa: E731
    need = lib.tjev_gdn_fork_workspace_bytes(_pages())
    assert need > 0
    fork = lambda p, a=None, k=ks, v=vs, n=need: lib.tjev_gdn_paged_fork(p, None, k, v, *(a or f[:13]), n)  # noqa: E731
    for bad, status in ((dict(requests=0), 1), (dict(table_width=0), 1), (dict(page_size=0), 1), (dict(pages=0), 1), (dict(layers=-1), 1),
                        (dict(requests=8193), 2), (dict(dtype=2), 1), (dict(kv_heads=0), 1), (dict(dim=0), 1), (dict(kv_heads=1 << 20), 2)):
        assert compact(_pages(**bad)) == status, (bad, said())
        assert fork(_pages(**bad)) == status, (bad, said())
    assert compact(_pages(max_new=0)) == 1 and compact(None) == 1 and fork(None) == 1
    for bad, status in ((dict(new_requests=0), 1), (dict(new_requests=8193), 2), (dict(n_free=-1), 1), (dict(n_free=1 << 31), 1),
                        (dict(table_width=1 << 30, requests=2), 1), (dict(table_width=1 << 30, requests=1), 1)):
        assert fork(_pages(**bad)) == status, (bad, said())
    odd, none = (ctypes.c_void_p * 2)(1 << 20, (1 << 21) + 1), (ctypes.c_void_p * 2)(1 << 20, None)
    for k in (odd, none, None):
        assert compact(_pages(), k=k) == 1 and compact(_pages(), v=k) == 1
    assert fork(_pages(), k=none) == 1 and fork(_pages(), v=None) == 1
    assert fork(_pages(), k=odd) == 1 and fork(_pages(), v=odd) == 1 and "aligned" in said()  # (before anything is launched)
    assert fork(_pages(page_size=1 << 20)) == 2 and "2^20" in said()
    for i in range(6):
        a = list(f[:6])
        a[i] = None
        assert compact(_pages(), a) == 1 and "null" in said()
    a = list(f[:6])
    a[5] = a[2]
    assert compact(_pages(), a) == 1 and "alias" in said()
    for i in (0, 1, 2, 4, 5, 6, 7, 8, 9, 10, 11):  # (keep may be null)
        a = list(f[:13])
        a[i] = None
        assert fork(_pages(), a) == 1 and "null" in said(), i
    for i, j in ((7, 0), (8, 1), (9, 4), (10, 5), (11, 6)):
        a = list(f[:13])
        a[i] = a[j]
        assert fork(_pages(), a) == 1 and "alias" in said(), i
    assert fork(_pages(), n=need - 1) == 3
    a = list(f[:13])
    a[12] = ctypes.c_void_p(4096 + 64)
    assert fork(_pages(), a) == 1


def test_tree_attention_c_abi():
    from tjev_amd import _lib

    lib, f = _lib.load(), _fake(12)
    p = _lib.PagedParams(tokens=3, requests=2, table_width=3, pages=4, page_size=16, heads=4, kv_heads=2, dim=64, dtype=1, scale=0.125, q_stride=(256, 64),
                         out_stride=(256, 64), k_stride=(2048, 128, 64), v_stride=(2048, 128, 64))
    need = lib.tjev_gdn_paged_tree_workspace_bytes(ctypes.byref(p))
    assert need > 0 and lib.tjev_gdn_paged_tree_workspace_bytes(None) == 0
    call = lambda a, words, n=need: lib.tjev_gdn_paged_tree_attention(ctypes.byref(p), None, *a[:7], words, None, a[8], a[9], n)  # noqa: E731
    assert call(f, 0) == 1 and "word" in lib.tjev_gdn_last_error().decode()
    assert call(f, 1, need - 1) == 3
    for i in (0, 1, 2, 3, 4, 5, 6, 8):
        a = list(f)
        a[i] = None
        assert call(a, 1) == 1 and "null" in lib.tjev_gdn_last_error().decode(), i


def test_the_keys_of_a_tree_under_asan(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(hipcc).exists():
        pytest.skip("hipcc not available")
    exe = tmp_path / "tree_asan"
    build = subprocess.run([hipcc, "--offload-arch=gfx950", "-O1", "-g", "-std=c++17", "-Xarch_host", "-fsanitize=address",
                            "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                            str(Path(__file__).parent / "asan" / "tree_driver.hip"), "-o", str(exe)], capture_output=True, text=True)
    assert build.returncode == 0, build.stderr[-3000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:halt_on_error=1:exitcode=86")
    run = subprocess.run([str(exe)], capture_output=True, text=True, env=env, timeout=300)
    assert run.returncode == 0 and "0 wrong" in run.stdout, (run.stdout + run.stderr)[-3000:]


def _tree_workspace(**kw):
    from tjev_amd import _lib

    p = dict(tokens=12, requests=1, table_width=254, pages=64, page_size=16, heads=16, kv_heads=4, dim=256, dtype=_lib.BF16, scale=1.0)
    p = _lib.PagedParams(**{**p, **kw})
    return _lib.load().tjev_gdn_paged_tree_workspace_bytes(ctypes.byref(p)), _lib.load().tjev_gdn_paged_workspace_bytes(ctypes.byref(p))


def test_small_batches_of_trees_are_streamed():
    """Places of 16 rows, not of 128: within a few units to a workgroup; beyond that, in fp32 and in few rows as causal rows are."""
    place = lambda rows: 2 * rows * (256 + 2) * 4 + 32  # noqa: E731
    tree, causal = _tree_workspace()
    assert tree % place(16) == 0 and causal % place(128) == 0
    for kw in (dict(table_width=4000), dict(tokens=400), dict(tokens=4), dict(dtype=0)):
        tree, causal = _tree_workspace(**kw)
        assert tree == causal > 0


# ---------------------------------------------------------------- the plain forms
def test_the_plain_trees_agree():
    """A chain's rows are the causal ones; a mask of one row moved to the next is told apart."""
    case = batch(torch.Generator().manual_seed(1), [(9, 5), (0, 3)], heads=2, kv_heads=1, dim=8, page=4, dtype=torch.float32)
    sets, positions = tree_walk([-1, 0, 1, 2, 3, -1, 0, 1], [0, 5, 8], [14, 3], 5)
    assert positions == [9, 10, 11, 12, 13, 0, 1, 2]
    names = ("q", "k_cache", "v_cache", "block_table", "starts", "lengths")
    want, room = attention64(*(case[n] for n in names))
    got, _ = tree_attention64(*(case[n] for n in names), bits_of(sets, 1))
    assert torch.allclose(got, want, rtol=0, atol=1e-12)
    wrong, _ = tree_attention64(*(case[n] for n in names), bits_of(sets, 1).roll(1, 0))
    assert bool(((wrong - want).abs() > room).any())


@pytest.mark.parametrize("drawn", [False, True])
def test_the_plain_walk_keeps_the_targets_distribution(drawn):
    """The first emitted token over a grid of numbers; a walk that forgets what was rejected is told apart."""
    gen = torch.Generator().manual_seed(2)
    p, q = (torch.softmax(1.5 * torch.randn(4, generator=gen), -1) for _ in range(2))
    m = 40
    grid = [(i + 0.5) / m for i in range(m)]
    got, wrong = torch.zeros(4, dtype=torch.float64), torch.zeros(4, dtype=torch.float64)
    for x in range(4) if drawn else [2]:
        weight = float(q[x]) if drawn else 1.0
        for u1 in grid:
            for u0 in grid:
                a = (torch.tensor([0, x]), p.repeat(2, 1), [0, 2], [u0, u1], None if drawn else [-1, 0], q.repeat(2, 1) if drawn else None, 2)
                says = verify_walk(*a)[0][0][0]
                got[says] += weight / m ** 2
                accepted = u1 * (float(q[x]) if drawn else 1.0) < float(p[x])
                wrong[x if accepted else verify_walk(torch.tensor([0]), p[None], [0, 1], [u0], None, None, 1)[0][0][0]] += weight / m ** 2
    assert float((got - p.double()).abs().max()) < 3 / m < float((wrong - p.double()).abs().max())


def test_the_plain_fork_counts_every_page():
    """After forks at random every page is held or on the list; the holders are `shared` + 1."""
    rng, page, width = random.Random(3), 4, 6
    table, lengths, free, taken, shared = [[-1] * width for _ in range(3)], [0] * 3, list(range(40)), 0, [0] * 40
    for _ in range(60):
        for b in range(3):  # growth
            n = min(lengths[b] + rng.randint(0, 7), width * page)
            for j in range(-(-lengths[b] // page), -(-n // page)):
                table[b][j] = free[taken]
                taken += 1
            lengths[b] = n
        sources = [rng.choice([b, rng.randrange(3), -1]) for b in range(3)]
        keep = [rng.randint(0, width * page) for _ in range(3)]
        table, lengths, free, taken, shared = fork_walk([], table, lengths, sources, keep, free, taken, shared, page)
        held = [p for row in table for p in row if p >= 0]
        assert sorted({*held, *free[taken:]}) == list(range(40)) and len(set(held)) + 40 - taken == 40
        assert [max(1, held.count(p)) - 1 for p in range(40)] == shared


def test_random_trees_are_trees():
    rng = random.Random(4)
    for kind in ("tree", "chain", "star", "any"):
        for n in (1, 2, 9, 70):
            p = random_tree(rng, n, kind)
            assert len(p) == n and p[0] == -1 and all(0 <= x < i for i, x in enumerate(p) if i)
