"""GPU tests of dropout masks at element indices past 32 bits, and past the 35 bits from
which on the generator's counter (index / 8) has a high word."""

from __future__ import annotations

import pytest
import torch

from test_counter_dropout_gpu import philox_draws, seed_of

pytestmark = pytest.mark.gpu


def test_counter_has_a_high_word():
    """2^35 elements and some, in place (69 GB of f16), on both sides of the border."""
    from dsalt.kernels import _ext
    n, around = (1 << 35) + 4099, 2048
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 90e9:
        pytest.skip("needs 90 GB of free device memory")
    x = torch.empty(n, device="cuda", dtype=torch.float16)
    first = (1 << 35) - around
    x[first:] = 1
    s = seed_of(41)
    _ext.call("dsalt_dropout", _ext.DropoutParams(_ext.ptr(x), _ext.ptr(x), _ext.ptr(s), n, 9, 32768, _ext.F16))
    keep = (philox_draws(n - first, 41, 9, first=first) >= 32768).cuda()
    assert torch.equal(x[first:] != 0, keep)
    # the high word matters: the draws of the low words alone are others
    low = (philox_draws(n - (1 << 35), 41, 9, first=0) >= 32768).cuda()
    assert not torch.equal(keep[around:], low)
    del x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("d", [1024, 1001])
def test_residual_masks_past_32_bits(d):
    """The residual step's masks of the last rows of more than 2^32 elements, forward and
    backward, with rows that start on a block of draws and rows that do not."""
    from dsalt import residual_norm
    T, rows, p = (1 << 32) // d + 9, 5, 0.25
    x = torch.zeros(T, d, device="cuda", dtype=torch.bfloat16)
    f = torch.ones(T, d, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    x_new, _ = residual_norm(x, f, dropout_p=p, seed=seed_of(6), site=2)
    (df,) = torch.autograd.grad(x_new, f, f.detach())
    keep = (philox_draws(rows * d, 6, 2, first=(T - rows) * d) >= round(p * 65536)).cuda().view(rows, d)
    assert torch.equal(x_new[-rows:] != 0, keep) and torch.equal(df[-rows:] != 0, keep)
