"""Slopes that need a gradient, through the public calls: refused where gradients are recorded, whatever else needs one,
taken where they are not. The launches are stubbed, so no GPU is needed."""

from __future__ import annotations

import sys

import pytest
import torch

from rfdetr_jax_amd import _native, packed_attention, packed_attention_forward

_module = sys.modules[packed_attention.__module__]  # (the package's name for it is the function's)
OFFSETS = torch.tensor([0, 4], dtype=torch.int32)


@pytest.fixture
def stubbed(monkeypatch):
    """The Python path with a forward that launches nothing, on CPU tensors."""
    monkeypatch.setattr(_native, "binding", lambda: _native._NoBinding)
    monkeypatch.setattr(_module, "_check", lambda q, k, v: None)
    monkeypatch.setattr(_module, "_forward", lambda q, *args: (q.clone(), None, torch.zeros(q.shape[0], q.shape[1], 4)))


@pytest.mark.parametrize("leaves", [(), (0,), (0, 1, 2)], ids=["none", "queries", "all"])
def test_learned_slopes_are_refused(stubbed, leaves):
    q, k, v = (torch.zeros(4, 2, 32, requires_grad=i in leaves) for i in range(3))
    slopes = torch.zeros(2, requires_grad=True)
    for given in (slopes, slopes * 2):
        with pytest.raises(ValueError, match="slopes get no gradient"):
            packed_attention(q, k, v, OFFSETS, slopes=given)
        with pytest.raises(ValueError, match="slopes get no gradient"):
            packed_attention_forward(q, k, v, OFFSETS, slopes=given)


def test_slopes_without_a_gradient_are_taken(stubbed):
    q, k, v = (torch.zeros(4, 2, 32, requires_grad=True) for _ in range(3))
    slopes = torch.zeros(2, requires_grad=True)
    assert packed_attention(q, k, v, OFFSETS, slopes=slopes.detach()).requires_grad
    assert packed_attention(q, k, v, OFFSETS, slopes=None).requires_grad
    with torch.no_grad():
        assert not packed_attention(q, k, v, OFFSETS, slopes=slopes).requires_grad
