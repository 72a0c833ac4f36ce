"""The room that tests/test_gpu_paged_pages.py leaves streamed rows is too small for weights of one bf16 term (CPU only: the mistake
is planted in the plain form)."""

from __future__ import annotations

import pytest
import torch

from test_gpu_paged_pages import SHAPES, cancelling, weighted


@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
def test_weights_of_one_term_are_told_apart(heads, kv_heads, dim, page):
    q, k, v = cancelling(torch.Generator().manual_seed(33), 1, 12, heads, kv_heads, dim)
    want, room = weighted(q, k, v)
    upper = lambda w: (w.float().view(torch.int32) & ~0xFFFF).view(torch.float32).double()  # noqa: E731
    for one in (upper, lambda w: w.to(torch.bfloat16).double()):
        bad, _ = weighted(q, k, v, one)
        assert float(((bad - want).abs() > room).double().mean()) > 0.02  # (one lane would fail the test)
    two = lambda w: upper(w) + (w - upper(w)).to(torch.bfloat16).double()  # noqa: E731
    kept, _ = weighted(q, k, v, two)
    assert bool(((kept - want).abs() <= room).all())
