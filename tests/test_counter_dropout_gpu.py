"""GPU tests of the counter-based dropout against Philox4x32-10 in numpy."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def philox_draws(n, seed, site, first=0):
    """16-bit draws of elements first … first + n − 1 (numpy, 64-bit products)."""
    u, low = np.uint64, np.uint64(0xFFFFFFFF)
    blocks = np.arange(first // 8, (first + n + 7) // 8, dtype=np.uint64)
    c = [blocks & low, blocks >> u(32), np.full_like(blocks, site), np.zeros_like(blocks)]
    k = [seed % 2 ** 32, (seed >> 32) % 2 ** 32]
    for _ in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> u(32)) ^ c[1] ^ u(k[0]), b & low, (a >> u(32)) ^ c[3] ^ u(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    d = np.stack(c, axis=1).astype(np.uint32).view(np.uint16).reshape(-1)
    return torch.from_numpy(d[first % 8:first % 8 + n].astype(np.int64))


def seed_of(v):
    return torch.tensor([v], dtype=torch.int64, device="cuda")


def test_generator_known_answer():
    """The published test vector of Philox4x32-10: counter 0, key 0."""
    d = philox_draws(8, 0, 0).numpy().astype(np.uint16).view(np.uint32)
    assert [hex(v) for v in d] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,offset", [(1, 0), (7, 0), (8, 0), (4099, 0), (4099, 1), (100_000, 3)])
def test_mask_values_and_gradient(n, offset, dtype):
    from dsalt.kernels.counter_dropout import counter_dropout
    p, site, sd = 0.3, 0xFFFF0001, -5 if offset else 2 ** 61 + 12345
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(n + offset, generator=g, device="cuda").to(dtype)[offset:].requires_grad_(True)  # unaligned too
    dy = torch.randn(n, generator=g, device="cuda").to(dtype)
    y = counter_dropout(x, p, seed_of(sd), site)
    (dx,) = torch.autograd.grad(y, x, dy)
    t = round(p * 65536)
    keep = (philox_draws(n, sd % 2 ** 64, site) >= t).cuda()
    # one fp32 product and one rounding to the type; the factor itself is rounded to fp32
    e = torch.finfo(dtype).eps / 2 + 2 * 2.0 ** -24
    for got, src in ((y, x), (dx, dy)):
        assert got.dtype == dtype
        assert not got[~keep].any()
        ref = src.detach().double() * 65536 / (65536 - t)
        assert ((got.double() - ref).abs()[keep] <= e * ref.abs()[keep] + 2.0 ** -25).all()


def test_share_dropped_and_sites_differ():
    """The shares over n draws are within 5 standard deviations; two sites agree by chance only."""
    from dsalt.kernels.counter_dropout import counter_dropout
    n = 1 << 20
    x = torch.ones(n, device="cuda")
    for p in (0.05, 0.5, 0.9):
        kept = [counter_dropout(x, p, seed_of(s), site) != 0 for s, site in ((1, 0), (1, 1), (2, 0))]
        for k in kept:
            assert abs(k.double().mean().item() - (1 - p)) < 5 * (p * (1 - p) / n) ** 0.5 + 2.0 ** -17
        both = (1 - p) ** 2
        for a, b in ((0, 1), (0, 2), (1, 2)):
            share = (kept[a] & kept[b]).double().mean().item()
            assert abs(share - both) < 5 * (both * (1 - both) / n) ** 0.5 + 2.0 ** -15


def test_ends_of_the_range():
    from dsalt.kernels.counter_dropout import counter_dropout
    x = torch.tensor([float("nan"), float("inf"), 1.0, -2.0] * 8, device="cuda")
    assert counter_dropout(x, 0.0, seed_of(1)) is x
    assert counter_dropout(x, 2.0 ** -18, seed_of(1)) is x
    assert counter_dropout(x, 0.7, None, training=False) is x
    assert not counter_dropout(x, 1.0, seed_of(1)).any()         # NaN and infinity are dropped too
    assert counter_dropout(x[:0], 0.5, seed_of(1)).shape == (0,)
    y = counter_dropout(x, 0.5, seed_of(3))
    keep = (philox_draws(32, 3, 0) >= 32768).cuda()
    assert torch.equal(torch.nan_to_num(y, 9.0, 8.0, 7.0), torch.nan_to_num(torch.where(keep, 2 * x, 0 * torch.ones_like(x)), 9.0, 8.0, 7.0))


def test_strided_input_counts_row_major():
    from dsalt.kernels.counter_dropout import counter_dropout
    x = torch.randn(40, 24, device="cuda")
    assert torch.equal(counter_dropout(x.t(), 0.4, seed_of(5)), counter_dropout(x.t().contiguous(), 0.4, seed_of(5)))


def test_positions_past_32_bits():
    """Element indices of a tensor beyond 2^32 elements draw from the counter's high word."""
    from dsalt.kernels.counter_dropout import counter_dropout
    n, tail = (1 << 35) // 8 + 40, 40     # f16 so that the tensor is 8.6 GB
    x = torch.empty(n, device="cuda", dtype=torch.float16)
    x[-64:] = 1
    y = counter_dropout(x, 0.5, seed_of(77))
    keep = (philox_draws(tail, 77, 0, first=n - tail) >= 32768).cuda()
    assert torch.equal(y[-tail:] != 0, keep)


def test_seed_change_before_backward_raises_and_replay_takes_the_new_seed():
    from dsalt.kernels.counter_dropout import counter_dropout
    x = torch.ones(4096, device="cuda", requires_grad=True)
    s = seed_of(10)
    y = counter_dropout(x, 0.5, s)
    s.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    del y
    s.fill_(20)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = counter_dropout(x, 0.5, s)
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    for v in (20, 21):
        s.fill_(v)
        graph.replay()
        keep = (philox_draws(4096, v, 0) >= 32768).cuda()
        assert torch.equal(y != 0, keep) and torch.equal(dx != 0, keep)
