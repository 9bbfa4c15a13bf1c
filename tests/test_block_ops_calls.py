"""CPU checks of what the feed-forward half's operators hand to the C entries and to
autograd.  The launches are recorded, not made: no kernel runs here."""

from __future__ import annotations

import importlib

import pytest
import torch


@pytest.fixture
def launches(monkeypatch):
    """Lets the operators take CPU tensors; every launch is recorded as (entry, parameters)."""
    from dsalt.kernels import _ext
    gated_ffn, residual_norm = (importlib.import_module(f"dsalt.kernels.{m}") for m in ("gated_ffn", "residual_norm"))
    calls = []
    monkeypatch.setattr(_ext, "require_cuda", lambda t, what="input": None)
    monkeypatch.setattr(_ext, "call_on", lambda device, name, p: calls.append((name, p)))
    monkeypatch.setattr(gated_ffn, "device_status_ptr", lambda device: 0)
    monkeypatch.setattr(residual_norm, "_parts", lambda T, d, device: 1)
    return calls


def ffn_leaves(T, d, F, d_out):
    """Operands in every layout that is read in place, or copied to rows of eights."""
    stacked = torch.randn(2, F, d + (-d) % 8).bfloat16()
    wide = torch.randn(T, d + 16 + (-d) % 8).bfloat16()
    return [t.requires_grad_(True) for t in (wide[:, :d], stacked[0][:, :d], stacked[1][:, :d], torch.randn(d_out, F).bfloat16())]


@pytest.mark.parametrize("sizes", [(5, 64, 96, 40), (5, 710, 769, 710), (1, 17, 5, 9)])
def test_saved_operands_may_come_back_in_another_layout(launches, sizes):
    """Saved tensors that a hook moved (to the host and back, say) are dense: their strides
    are read from what came back, not kept from the forward."""
    from dsalt.kernels.gated_ffn import gated_ffn
    T, d, F, d_out = sizes
    back = {}

    def unpack(t):
        dense = torch.empty(t.shape, dtype=t.dtype).copy_(t)
        back[dense.data_ptr()] = dense
        return dense

    leaves = ffn_leaves(*sizes)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), unpack):
        y = gated_ffn(*leaves, dtype=torch.bfloat16)
        torch.autograd.grad(y, leaves, torch.randn(T, d_out).bfloat16())
    (name, p), = launches[1:]
    assert name == "dsalt_gated_ffn_bwd"
    for ptr, ld, rows in ((p.x, p.ld_x, T), (p.w_gate, p.ld_wg, F), (p.w_up, p.ld_wu, F), (p.w_down, p.ld_wd, d_out)):
        assert ld % 8 == 0
        if ptr in back and rows > 1:
            assert ld == back[ptr].stride(0)
