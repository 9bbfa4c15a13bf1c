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


def dual_calls():
    from dsalt import counter_dropout, gated_ffn, residual_norm
    half, seed = torch.bfloat16, torch.tensor([1])
    x, w, v, d = (torch.randn(*s).to(half) for s in ((4, 8), (16, 8), (8, 16), (8,)))
    gate = torch.rand(4).to(half)
    return {"gated_ffn": (lambda *t: gated_ffn(*t, dtype=half), (x, w, w.clone(), v)),
            "residual_norm": (lambda a, f, n, p, s, g: residual_norm(a, f, n, post_weight=p, scale=s, gate=g)[0],
                              (x, x.clone(), d, d.clone(), d.clone(), gate)),
            "counter_dropout": (lambda t: counter_dropout(t, 0.5, seed), (x,))}


@pytest.mark.parametrize("no_grad", [False, True])
@pytest.mark.parametrize("name", ["gated_ffn", "residual_norm", "counter_dropout"])
def test_forward_mode_is_refused(launches, name, no_grad):
    """A tangent on any input raises: without a rule for it the result would silently carry
    none, a derivative of 0."""
    import torch.autograd.forward_ad as fw
    fn, args = dual_calls()[name]
    with torch.set_grad_enabled(not no_grad):
        for i in range(len(args)):
            with fw.dual_level():
                dual = [fw.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
                with pytest.raises(NotImplementedError, match="jvp"):
                    fn(*dual)
                assert fw.unpack_dual(torch.as_tensor(fn(*args))).tangent is None  # no tangent: no refusal
        del launches[:]
        fn(*args)
        assert len(launches) == 1


def test_one_status_word_however_many_threads_make_it(monkeypatch):
    """A thread that finds no status word may make one while another does: both get the word
    that is kept, so that no launch holds the address of one that was freed."""
    from dsalt.kernels import dsalt_cuda
    monkeypatch.setattr(dsalt_cuda, "_STATUS", {})
    zeros, other = torch.zeros, torch.zeros(1, dtype=torch.int32)

    def zeros_while_another_thread_is_first(*args, device, **kw):
        dsalt_cuda._STATUS[("cuda", 0)] = other
        return zeros(*args, **kw)

    monkeypatch.setattr(torch, "zeros", zeros_while_another_thread_is_first)
    assert dsalt_cuda.device_status(torch.device("cuda:0")) is other
    assert dsalt_cuda._STATUS == {("cuda", 0): other}


def test_products_too_long_for_the_kernels_waits_are_refused():
    """A tile's products all end before its epilogue starts, within the limit of the kernels'
    waits (about 2 s): past 2^27 tokens a weight gradient is refused instead of given up on the
    device.  (Widths are held far below by the number of tiles.)"""
    import ctypes
    from dsalt.kernels import _ext
    align, large, lib = 6, 7, _ext.load()  # DSALT_ERR_*

    def rc(name, **kw):
        base = dict(x=16, w_gate=16, w_up=16, w_down=16, h=16, h_lo=16, y=16, dy=16, a=16, b=16, ab=16, dg=16, du=16,
                    T=4, ld_x=64, ld_wg=64, ld_wu=64, ld_wd=96, ld_f=96, ld_dy=64, d=64, F=96, d_out=64, dtype=_ext.BF16)
        return getattr(lib, name)(ctypes.byref(_ext.GatedFfnParams(**{**base, **kw})), ctypes.c_void_p(0))

    for grad in ("dw_gate", "dw_up", "dw_down"):
        assert rc("dsalt_gated_ffn_bwd", T=(1 << 27) + 1, **{grad: 16}) == large, grad
        # refused for its pointers, not for its size (and so before any launch)
        assert rc("dsalt_gated_ffn_bwd", T=1 << 27, dy=24, **{grad: 16}) == align, grad
    assert rc("dsalt_gated_ffn_bwd", T=1 << 29, dy=24, dx=16) == align
    assert rc("dsalt_gated_ffn_fwd", T=1 << 29, x=24) == align
    n = (1 << 22) + 8
    for wide in (dict(d=n, ld_x=n, ld_wg=n, ld_wu=n), dict(F=n, ld_wd=n, ld_f=n), dict(d_out=n, ld_dy=n)):
        assert rc("dsalt_gated_ffn_fwd", **wide) == rc("dsalt_gated_ffn_bwd", dx=16, **wide) == large, wide
