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
