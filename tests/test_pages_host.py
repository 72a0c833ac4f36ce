"""Forks' last check before a launch (CPU only): the grid that copies a page's tokens."""

from __future__ import annotations

import ctypes

import pytest
import torch


@pytest.mark.parametrize("dtype,kv_heads,dim,page_size", [(1, 8, 256, (1 << 20) - 15), (0, 8, 256, (1 << 20) - 1), (1, 9, 256, (1 << 20) - 1),
                                                          (1, 129, 1, (1 << 20) - 15)])
def test_pages_of_more_parts_than_a_grid_has(dtype, kv_heads, dim, page_size):
    """A workgroup takes 16 tokens of more than 128 vectors: 65536 of them are one more than a grid's third dimension holds. Made-up
    addresses that are never launched on."""
    from tjev_amd import _lib

    if torch.cuda.is_available():
        pytest.skip("host-side refusals with made-up device addresses: CPU only")
    lib = _lib.load()
    slot = kv_heads * dim
    p = _lib.PagesParams(n_free=5, requests=2, new_requests=3, table_width=3, pages=4, page_size=page_size, kv_heads=kv_heads, dim=dim, dtype=dtype,
                         layers=1, k_stride=(page_size * slot, slot, dim), v_stride=(page_size * slot, slot, dim))
    caches = (ctypes.c_void_p * 1)(1 << 40)
    given = [ctypes.c_void_p(4096 * (i + 1)) for i in range(13)]
    need = lib.tjev_gdn_fork_workspace_bytes(ctypes.byref(p))
    assert lib.tjev_gdn_paged_fork(ctypes.byref(p), None, caches, caches, *given, need) == 2
    assert "2^20 - 16" in lib.tjev_gdn_last_error().decode()
