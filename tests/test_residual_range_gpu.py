"""GPU tests of the residual step's gradients over the range of row sizes that its
forward holds, against 64 bits (the bounds of ``test_residual_norm_gpu``)."""

from __future__ import annotations

import pytest
import torch

from test_residual_norm_gpu import check, make, reference, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [72, 1024, 4099])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gate", ["token", "full", "none"])
@pytest.mark.parametrize("size,eps", [(1e15, 1e-6), (1e13, 1e-6), (1e-14, 0.0), (1e-12, 1e-30)])
def test_large_and_small_rows(size, eps, gate, dtype, d):
    """The cube of an inverse root mean square leaves fp32's range long before the row does."""
    t, dx_new, dh = make(9, d, dtype, torch.float32, True, True, gate, True)
    with torch.no_grad():
        t["x"].mul_(size)
        t["f"].mul_(size)
        t["post"].mul_(size)   # the branch is of the stream's size
        dx_new /= size         # and both parts of dx of one size
    outs = run(t, eps=eps)
    names = list(t) if gate != "none" else [k for k in t if k != "gate"]
    grads = torch.autograd.grad(outs, [t[k] for k in names], [dx_new, dh])
    ref = reference(t, outs[0], dx_new, dh, 1.0, eps)
    check(outs[0], ref["x_new"], "x_new", 9)
    check(outs[1], ref["h"], "h", 9)
    for k, g in zip(names, grads):
        check(g, ref[k], k, 9)
