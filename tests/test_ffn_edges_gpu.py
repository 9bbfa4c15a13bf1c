"""GPU tests of the gated feed-forward block at its edges, against the bounds of
``test_gated_ffn_gpu``."""

from __future__ import annotations

import pytest
import torch

from test_gated_ffn_gpu import NAMES, check, inputs, reference

pytestmark = pytest.mark.gpu


# K of 2048 and more splits over the eight CTAs of a cluster (16 tokens at most), from 1024
# on over eight (17 to 384): the last CTA with tokens then has results for half a warp
@pytest.mark.parametrize("size", [(1, 2056, 520, 40), (3, 2048, 2056, 24), (9, 2056, 2048, 40), (1, 2048, 72, 8),
                                  (17, 1032, 72, 40), (33, 1032, 1096, 24), (65, 1096, 72, 8), (321, 1032, 1032, 8)])
def test_results_of_part_of_a_warp(size):
    """The loop over a CTA's results ends lane by lane: the cluster's barrier after it (and the
    release of TMEM) waits for whole warps.  Ten calls in a row, all with the same bits."""
    from dsalt.kernels.gated_ffn import gated_ffn
    *leaves, dy = inputs(*size, torch.bfloat16)
    y = gated_ffn(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    ref = reference(*leaves, dy, "silu")
    for name, g in zip(("y",) + NAMES, (y, *grads)):
        check(g, ref[name], name)
    with torch.no_grad():
        assert all(torch.equal(gated_ffn(*leaves), y) for _ in range(10))


@pytest.mark.parametrize("size", [(37, 64, 96, 40), (140, 710, 769, 710), (1, 17, 5, 9)])
def test_gradients_of_operands_saved_on_the_host(size):
    """torch's save_on_cpu brings slices and padded copies back as dense tensors: the same bits."""
    from dsalt.kernels.gated_ffn import gated_ffn
    T, d, F, _ = size
    x, wg, wu, wd, dy = inputs(*size, torch.bfloat16, grad=False)
    pad = (-d) % 8 + 16
    xs = torch.nn.functional.pad(x, (0, pad))[:, :d].requires_grad_(True)
    stacked = torch.nn.functional.pad(torch.stack([wg, wu]), (0, pad))
    leaves = [xs, *(w[:, :d].requires_grad_(True) for w in stacked), wd.requires_grad_(True)]
    ref = torch.autograd.grad(gated_ffn(*leaves), leaves, dy)
    with torch.autograd.graph.save_on_cpu():
        y = gated_ffn(*leaves)
    got = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_residual_step_and_dropout_saved_on_the_host():
    from dsalt import counter_dropout, residual_norm
    seed = torch.tensor([3], dtype=torch.int64, device="cuda")
    x, f = (torch.randn(60, 264, device="cuda").bfloat16().requires_grad_(True) for _ in range(2))
    w = torch.rand(264, device="cuda").requires_grad_(True)
    gate = torch.rand(60, 528, device="cuda").bfloat16()[:, ::2].requires_grad_(True)
    leaves = (x, f, w, gate)

    def step():
        x_new, h = residual_norm(x, counter_dropout(f, 0.25, seed, 1), w, post_weight=w, gate=gate, dropout_p=0.25, seed=seed)
        return x_new.float().sum() + h.float().square().sum()

    ref = torch.autograd.grad(step(), leaves)
    with torch.autograd.graph.save_on_cpu():
        y = step()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves), ref))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 4, 16, 24, 40, 64, 70, 400])
def test_hidden_values_past_the_type(T, dtype):
    """A hidden value that the type holds only as an infinity makes the outputs that use it
    infinite, or NaN where infinities of both signs or a weight of 0 meet, at any number of
    tokens: only the sum's infinities, none that the split into two words brings in."""
    from dsalt.kernels.gated_ffn import gated_ffn
    d, F, d_out = 32, 48, 24
    x, wg, wu, wd, _ = inputs(T, d, F, d_out, dtype, grad=False)
    big = 300.0 if dtype == torch.float16 else 2.0 ** 65  # its square is past the type
    x[:, 0] = 0
    x[::2, 0] = 1.0                                # every other token
    wg[:, 0], wu[:, 0] = 0, 0
    wg[5, 0] = wu[5, 0] = wg[20, 0] = big          # h[5] past the type, h[20] not
    wg[5, 1:], wu[5, 1:], wg[20, 1:] = 0, 0, 0
    wd[:4, 5], wd[4:8, 5], wd[8:12, 5] = 0.5, -0.5, 0
    wg[30, 0], wu[30, 0], wg[30, 1:], wu[30, 1:] = big, -big, 0, 0   # h[30] past it with the other sign
    wd[:, 30] = 0.0
    wd[12:, 30], wd[12:, 5] = 0.25, 0.25           # inf - inf
    y = gated_ffn(x, wg, wu, wd)
    on, off = y[::2], y[1::2]
    assert torch.isfinite(off).all()
    # weights of 0 times an infinity are NaN: columns 0 to 11 have h[30] · 0
    assert torch.isnan(on).all()
    wd[:, 30] = 1e-3
    wu[30] = 0                                     # h[30] = 0: one infinity alone
    y = gated_ffn(x, wg, wu, wd)
    on = y[::2]
    assert (on[:, :4] == float("inf")).all() and (on[:, 4:8] == -float("inf")).all()
    assert torch.isnan(on[:, 8:12]).all() and (on[:, 12:] == float("inf")).all()
    assert torch.isfinite(y[1::2]).all()


def test_calls_from_many_threads_at_once():
    """Every variant and both directions from four threads on streams of their own: the bits of
    one thread's calls."""
    import threading
    from dsalt import counter_dropout, residual_norm
    from dsalt.kernels.gated_ffn import gated_ffn
    seed = torch.tensor([3], dtype=torch.int64, device="cuda")
    ffn = [inputs(T, 264, 520, 264, torch.bfloat16) for T in (4, 30, 200, 700)]
    x, f, w = (torch.randn(s, device="cuda").requires_grad_(True) for s in ((300, 777), (300, 777), (777,)))

    def work():
        out = []
        for *leaves, dy in ffn:
            y = gated_ffn(*leaves)
            out += [y, *torch.autograd.grad(y, leaves, dy)]
        x_new, h = residual_norm(counter_dropout(x, 0.25, seed, 1), f, w, post_weight=w, dropout_p=0.1, seed=seed)
        return out + [x_new, h, *torch.autograd.grad((x_new.sum() + h.square().sum()), (x, f, w))]

    ref = work()
    torch.cuda.synchronize()
    got = [None] * 4

    def thread(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[i] = work()
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for out in got:
        assert all(torch.equal(a, b) for a, b in zip(out, ref))


@pytest.mark.parametrize("n", [8, 4099, 3_000_008])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_dropout_in_place(n, dtype):
    """The C entry may write where it reads."""
    from dsalt import counter_dropout
    from dsalt.kernels import _ext
    x, seed = torch.randn(n, device="cuda").to(dtype), torch.tensor([3], dtype=torch.int64, device="cuda")
    ref = counter_dropout(x, 0.25, seed, 2)
    _ext.call("dsalt_dropout", _ext.DropoutParams(_ext.ptr(x), _ext.ptr(x), _ext.ptr(seed), n, 2, 16384, _ext.dtype_code(dtype)))
    assert torch.equal(x, ref)
