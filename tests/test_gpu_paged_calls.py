"""The paged cache's operators (tjev_amd.paged) called in ways that a served batch comes to: views off 16 bytes, against their
plain 64-bit forms (tests/paged_cases.py)."""

from __future__ import annotations

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
