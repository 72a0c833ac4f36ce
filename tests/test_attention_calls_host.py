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
    from tjev_amd import _lib

    lib = _Library()
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(_lib, "one_gpu", lambda what, devices: None)
    monkeypatch.setattr(_lib, "current_stream", lambda device: 0)
    monkeypatch.setattr(_lib, "on_device", lambda device: contextlib.nullcontext())
    return lib


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
