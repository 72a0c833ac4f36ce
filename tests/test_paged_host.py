"""Host-side checks of the attention layers' operators (CPU only): every refusal comes before a launch, with
the framework's errors; nothing falls back to a CPU path; the kernels' index arithmetic stays in bounds
over batches that hold anything (under AddressSanitizer)."""

import ctypes
import os
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]
BF = torch.bfloat16


def test_indexes_stay_in_bounds_under_asan(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(hipcc).exists():
        pytest.skip("hipcc not available")
    exe = tmp_path / "paged_asan"
    build = subprocess.run([hipcc, "--offload-arch=gfx950", "-O1", "-g", "-std=c++17", "-Xarch_host", "-fsanitize=address",
                            "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                            str(ROOT / "tests" / "asan" / "paged_driver.hip"), "-o", str(exe)], capture_output=True, text=True)
    assert build.returncode == 0, build.stderr[-3000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:halt_on_error=1:exitcode=86")
    run = subprocess.run([str(exe)], capture_output=True, text=True, env=env, timeout=300)
    assert run.returncode == 0 and "0 out of bounds" in run.stdout, (run.stdout + run.stderr)[-3000:]


def _rotary_args(**kw):
    a = dict(q=torch.zeros(2, 5, 4, 64), k=torch.zeros(2, 5, 2, 64), positions=torch.zeros(3, 2, 5, dtype=torch.int64),
             inv_freq=torch.ones(16, dtype=torch.float64), sections=(6, 5, 5))
    a.update(kw)
    return a


@pytest.mark.parametrize("bad,match", [
    (dict(q=torch.zeros(2, 5, 4, 64, dtype=torch.float16)), "float32 or bfloat16"),
    (dict(q=torch.zeros(5, 64)), "q is"),
    (dict(k=torch.zeros(2, 6, 2, 64)), "does not go with"),
    (dict(k=torch.zeros(2, 5, 2, 64, dtype=BF)), "does not go with"),
    (dict(positions=torch.zeros(2, 5, dtype=torch.int64)), "positions"),
    (dict(positions=torch.zeros(3, 2, 5)), "int32 or int64"),
    (dict(positions=torch.zeros(2, 2, 5, dtype=torch.int64)), "2 axes for 3"),
    (dict(sections=(6, 5, 4)), "do not add up"),
    (dict(sections=(18, 5, -7)), "do not add up"),
    (dict(sections=(2, 7, 7), interleaved=True), "runs out"),
    (dict(sections=(6, 4, 2, 2, 2), positions=torch.zeros(5, 2, 5, dtype=torch.int64)), "position axes"),
    (dict(inv_freq=torch.ones(33)), "frequencies turn"),
    (dict(inv_freq=torch.ones(16, dtype=torch.int32)), "frequencies"),
    (dict(inv_freq=torch.ones(0), sections=None, positions=torch.zeros(1, 2, 5, dtype=torch.int64)), "frequencies turn"),
])
def test_rotary_refusals(bad, match):
    from tjev_amd import rotary_axes

    a = _rotary_args(**bad)
    with pytest.raises(ValueError, match=match):
        rotary_axes(a.pop("q"), a.pop("k"), a.pop("positions"), a.pop("inv_freq"), **a)


def test_no_cpu_fallback():
    from tjev_amd import paged_append, paged_attention, paged_tables, rotary_axes

    a = _rotary_args()
    with pytest.raises(RuntimeError, match="GPU"):
        rotary_axes(a["q"], a["k"], a["positions"], a["inv_freq"], sections=a["sections"])
    i = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        paged_tables(i, i, table, i, page_size=16, tokens=4)
    cache = torch.zeros(4, 16, 2, 64)
    with pytest.raises(RuntimeError, match="GPU"):
        paged_append(torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), cache, cache, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="GPU"):
        paged_attention(torch.zeros(3, 4, 64), cache, cache, table, torch.zeros(3, dtype=torch.int32), i)


@pytest.mark.parametrize("bad,match", [
    (dict(block_table=torch.zeros(2, 3, dtype=torch.int64)), "int32"),
    (dict(block_table=torch.zeros(0, 3, dtype=torch.int32)), "requests"),
    (dict(block_table=torch.zeros(8193, 1, dtype=torch.int32)), "requests"),
    (dict(cached=torch.zeros(3, dtype=torch.int32)), "lengths"),
    (dict(new=torch.zeros(2)), "int32 or int64"),
    (dict(taken=torch.zeros(2, dtype=torch.int32)), "one number"),
    (dict(page_size=0), "requests of pages"),
    (dict(tokens=-1), "tokens"),
])
def test_tables_refusals(bad, match):
    from tjev_amd import paged_tables

    i = torch.zeros(2, dtype=torch.int32)
    a = dict(cached=i, new=i, block_table=torch.zeros(2, 3, dtype=torch.int32), free_pages=i, taken=None, page_size=16, tokens=4)
    a.update(bad)
    with pytest.raises(ValueError, match=match):
        paged_tables(**a)


@pytest.mark.parametrize("table", [torch.zeros(2, 6, dtype=torch.int32)[:, ::2], torch.zeros(3, 2, dtype=torch.int32).t(),
                                   torch.zeros(2, 3, dtype=torch.int32)[:, :1], torch.zeros(2, 5, dtype=torch.int32)[:, :3]])
def test_tables_refuse_to_copy_a_table_changed_in_place(monkeypatch, table):
    from tjev_amd import _lib, paged_tables

    monkeypatch.setattr(_lib, "one_gpu", lambda what, devices: None)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="contiguous"):
        paged_tables(i, i, table, i, page_size=16, tokens=4, inplace=True)


@pytest.mark.parametrize("bad,match", [
    (dict(v=torch.zeros(3, 2, 32)), "alike"),
    (dict(k=torch.zeros(3, 2, 64, dtype=BF), v=torch.zeros(3, 2, 64, dtype=BF)), "cache's type"),
    (dict(k_cache=torch.zeros(4, 16, 3, 64)), "caches"),
    (dict(v_cache=torch.zeros(5, 16, 2, 64)), "caches"),
    (dict(k_cache=torch.zeros(4, 16, 64, 2).transpose(2, 3)), "contiguous"),
    (dict(k_cache=torch.zeros(4, 1, 2, 64).expand(4, 16, 2, 64)), "expanded"),
    (dict(slots=torch.zeros(4, dtype=torch.int64)), "slots"),
    (dict(slots=torch.zeros(3)), "slots"),
])
def test_append_refusals(bad, match):
    from tjev_amd import paged_append

    a = dict(k=torch.zeros(3, 2, 64), v=torch.zeros(3, 2, 64), k_cache=torch.zeros(4, 16, 2, 64), v_cache=torch.zeros(4, 16, 2, 64),
             slots=torch.zeros(3, dtype=torch.int64))
    a.update(bad)
    with pytest.raises(ValueError, match=match):
        paged_append(**a)


@pytest.mark.parametrize("bad,match", [
    (dict(q=torch.zeros(3, 4, 64, dtype=torch.float16)), "float32 or bfloat16"),
    (dict(q=torch.zeros(3, 4, 64, dtype=BF)), "as the cache is"),
    (dict(q=torch.zeros(3, 3, 64)), "groups"),
    (dict(q=torch.zeros(3, 4, 60)), "caches"),
    (dict(k_cache=torch.zeros(64, 64)), "caches"),
    (dict(block_table=torch.zeros(2, 3)), "int32"),
    (dict(block_table=torch.zeros(2, 0, dtype=torch.int32)), "without pages"),
    (dict(starts=torch.zeros(2, dtype=torch.int32)), "starts"),
    (dict(lengths=torch.zeros(2)), "int32 or int64"),
    (dict(gate=torch.zeros(3, 4, 32)), "gate"),
    (dict(out=torch.zeros(3, 4, 64, dtype=BF)), "out"),
    (dict(out=torch.zeros(3, 1, 64).expand(3, 4, 64)), "expanded"),
])
def test_attention_refusals(bad, match):
    from tjev_amd import paged_attention

    i = torch.zeros(2, dtype=torch.int32)
    a = dict(q=torch.zeros(3, 4, 64), k_cache=torch.zeros(4, 16, 2, 64), v_cache=torch.zeros(4, 16, 2, 64),
             block_table=torch.zeros(2, 3, dtype=torch.int32), starts=torch.zeros(3, dtype=torch.int32), lengths=i)
    a.update(bad)
    with pytest.raises(ValueError, match=match):
        paged_attention(**a)


@pytest.mark.parametrize("dim", [4, 12, 264])
def test_attention_refuses_head_dims(dim):
    from tjev_amd import paged_attention

    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="multiples of 8"):
        paged_attention(torch.zeros(3, 4, dim), torch.zeros(4, 16, 2, dim), torch.zeros(4, 16, 2, dim),
                        torch.zeros(2, 3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), i)


# ---------------------------------------------------------------- the C ABI, with made-up addresses never launched on
def _fake(n):
    if torch.cuda.is_available():
        pytest.skip("host-side refusals with made-up device addresses: CPU only")
    return [ctypes.c_void_p(4096 * (i + 1)) for i in range(n)]


def _rotary_params(**kw):
    from tjev_amd import _lib

    p = _lib.RotaryParams(batch=2, length=5, q_heads=4, k_heads=2, dim=64, rotary=32, axes=3, sections=(6, 5, 5), dtype=1,
                          position_bits=64, freq_bits=64, q_stride=(1280, 256, 64), k_stride=(640, 128, 64))
    for n, v in kw.items():
        setattr(p, n, (ctypes.c_int32 * 4)(*v) if n == "sections" else v)
    return p


@pytest.mark.parametrize("bad,status,msg", [
    (dict(batch=-1), 1, "negative"), (dict(dim=2048), 2, "head dims"), (dict(rotary=31), 1, "rotated lanes"),
    (dict(rotary=66), 1, "rotated lanes"), (dict(axes=5), 1, "axes"), (dict(sections=(6, 5, 4)), 1, "add up"),
    (dict(sections=(2, 7, 7), interleaved=1), 1, "runs out"), (dict(dtype=2), 1, "dtype"), (dict(freq_bits=16), 1, "32 or 64"),
    (dict(length=1 << 40), 1, "too large"),
])
def test_rotary_c_abi(bad, status, msg):
    from tjev_amd import _lib

    lib = _lib.load()
    got = lib.tjev_gdn_rotary(ctypes.byref(_rotary_params(**bad)), None, *_fake(6))
    assert got == status and msg in lib.tjev_gdn_last_error().decode()


def test_rotary_c_abi_nulls():
    from tjev_amd import _lib

    lib = _lib.load()
    assert lib.tjev_gdn_rotary(None, None, *_fake(6)) == 1
    f = _fake(6)
    f[4] = None
    assert lib.tjev_gdn_rotary(ctypes.byref(_rotary_params()), None, *f) == 1 and "null" in lib.tjev_gdn_last_error().decode()
    f = _fake(6)
    f[0] = ctypes.c_void_p(4097)
    assert lib.tjev_gdn_rotary(ctypes.byref(_rotary_params()), None, *f) == 1 and "aligned" in lib.tjev_gdn_last_error().decode()
    assert lib.tjev_gdn_rotary(ctypes.byref(_rotary_params(length=0)), None, *[None] * 6) == 0  # nothing to do


def _paged_params(**kw):
    from tjev_amd import _lib

    p = dict(tokens=3, requests=2, table_width=3, pages=4, page_size=16, heads=4, kv_heads=2, dim=64, dtype=1, scale=0.125,
             q_stride=(256, 64), out_stride=(256, 64), gate_stride=(256, 64), k_stride=(2048, 128, 64), v_stride=(2048, 128, 64),
             k_new_stride=(128, 64), v_new_stride=(128, 64))
    p.update(kw)
    return _lib.PagedParams(**p)


@pytest.mark.parametrize("bad,status,msg", [
    (dict(requests=0), 1, "positive"), (dict(page_size=0), 1, "positive"), (dict(pages=0), 1, "positive"), (dict(tokens=-1), 1, "negative"),
    (dict(heads=3), 1, "groups"), (dict(dtype=3), 1, "dtype"), (dict(dim=12), 2, "multiples of 8"), (dict(dim=264), 2, "multiples of 8"),
    (dict(scale=float("nan")), 1, "finite"), (dict(scale=float("inf")), 1, "finite"), (dict(table_width=1 << 28), 1, "too large"),
    (dict(table_width=(1 << 20) - 1, page_size=2048), 1, "too large"),  # keys whose tiles end past the 32-bit numbers
    (dict(tokens=1 << 30), 1, "too large"), (dict(q_stride=(256, 60)), 1, "16-byte"), (dict(k_stride=(2044, 128, 64)), 1, "16-byte"),
])
def test_attention_c_abi(bad, status, msg):
    from tjev_amd import _lib

    lib = _lib.load()
    p = _paged_params(**bad)
    got = lib.tjev_gdn_paged_attention(ctypes.byref(p), None, *_fake(9), 1 << 40)
    assert got == status and msg in lib.tjev_gdn_last_error().decode()


def test_attention_c_abi_workspace_and_nulls():
    from tjev_amd import _lib

    lib = _lib.load()
    p = _paged_params()
    need = lib.tjev_gdn_paged_workspace_bytes(ctypes.byref(p))
    assert need > 0 and lib.tjev_gdn_paged_workspace_bytes(ctypes.byref(_paged_params(dim=12))) == 0
    f = _fake(9)
    assert lib.tjev_gdn_paged_attention(ctypes.byref(p), None, *f, need - 1) == 3
    f[8] = ctypes.c_void_p(4096 + 64)
    assert lib.tjev_gdn_paged_attention(ctypes.byref(p), None, *f, need) == 1
    for i in (0, 1, 2, 3, 4, 5, 7):
        f = _fake(9)
        f[i] = None
        assert lib.tjev_gdn_paged_attention(ctypes.byref(p), None, *f, need) == 1
    f = _fake(9)
    f[0] = ctypes.c_void_p(4096 + 8)
    assert lib.tjev_gdn_paged_attention(ctypes.byref(p), None, *f, need) == 1
    assert lib.tjev_gdn_paged_attention(None, None, *f, need) == 1
    assert lib.tjev_gdn_paged_attention(ctypes.byref(_paged_params(tokens=0)), None, *[None] * 9, 0) == 0


def test_tables_and_append_c_abi():
    from tjev_amd import _lib

    lib = _lib.load()
    f = _fake(12)
    tables = lambda p, a: lib.tjev_gdn_paged_tables(ctypes.byref(p), None, *a[:4], 5, *a[4:10])  # noqa: E731
    for bad, status in ((dict(requests=0), 1), (dict(requests=8193), 2), (dict(table_width=0), 1), (dict(page_size=0), 1),
                        (dict(tokens=1 << 31), 1)):
        assert tables(_paged_params(**bad), f) == status, bad
    for i in (0, 1, 2, 3, 5, 6, 7, 8, 9):
        a = list(f)
        a[i] = None
        assert tables(_paged_params(), a) == 1, i
    a = list(f)
    a[9] = a[4]  # taken_out over taken
    assert tables(_paged_params(), a) == 1 and "alias" in lib.tjev_gdn_last_error().decode()
    append = lambda p, a: lib.tjev_gdn_paged_append(ctypes.byref(p), None, *a[:5])  # noqa: E731
    for bad, status in ((dict(pages=0), 1), (dict(kv_heads=0), 1), (dict(dim=0), 1), (dict(dtype=2), 1), (dict(tokens=-1), 1),
                        (dict(kv_heads=1 << 14), 2)):
        assert append(_paged_params(**bad), f) == status, bad
    for i in range(5):
        a = list(f)
        a[i] = None
        assert append(_paged_params(), a) == 1
    a = list(f)
    a[0] = ctypes.c_void_p(4097)
    assert append(_paged_params(), a) == 1
    assert append(_paged_params(tokens=0), [None] * 5) == 0
