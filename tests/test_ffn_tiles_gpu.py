"""GPU tests of the gated feed-forward block on the tiles that large calls take, and of what
its forward keeps.  Bounds as in ``test_gated_ffn_gpu``."""

from __future__ import annotations

import importlib
import math

import pytest
import torch

from test_gated_ffn_gpu import ACTS, NAMES, check, inputs, reference

pytestmark = pytest.mark.gpu

# T, d, F, d_out; on 148 SMs the tiles' columns are, for (hidden, out, dh, dx, weights):
SIZES = [(3379, 1299, 1290, 281),     # 256,  64, 128, 512, 512; no side a multiple of 8
         (2019, 1204, 1593, 70),      # 256,  64, 128, 256, 512
         (6326, 673, 969, 76),        # 256,  64, 128, 512, 128
         (6791, 92, 294, 597),        # 128, 128, 256, 128, 128
         (2112, 66, 620, 1049),       #  64, 256, 128, 128, 128
         (3106, 91, 69, 1121),        #  64, 128, 128, 128, 128
         (580, 302, 2358, 79),        # 128,  64, 128, 128, 256
         (3218, 656, 258, 90),        # 128,  64, 128, 256, 128
         (579, 598, 1602, 106),       # 256,  64, 128, 128, 256
         (8200, 1032, 1400, 1032),    # 256, 256, 256, 256, 512; ragged multiples of 8
         (16384, 1024, 2816, 1024)]   # 256, 256, 256, 512, 512


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", SIZES)
def test_values_and_gradients(size, dtype):
    from dsalt.kernels.gated_ffn import gated_ffn
    *leaves, dy = inputs(*size, dtype)
    act = ACTS[(size[0] + (dtype == torch.float16)) % 3]
    y = gated_ffn(*leaves, activation=act)
    grads = torch.autograd.grad(y, leaves, dy)
    ref = reference(*leaves, dy, act)
    for name, g in zip(("y",) + NAMES, (y, *grads)):
        check(g, ref[name], name)
    del ref
    with torch.no_grad():
        assert torch.equal(gated_ffn(*leaves, activation=act), y)
    # the fp32 sums of fp32 weights' gradients, rounded, are the 16-bit gradients
    full = [leaves[0], *(t.detach().float().requires_grad_(True) for t in leaves[1:])]
    again = torch.autograd.grad(gated_ffn(*full, activation=act, dtype=dtype), full, dy)
    for name, a, b in zip(NAMES, grads, again):
        assert torch.equal(a, b.to(dtype)), name
    assert all(g.dtype == torch.float32 and not torch.equal(g, g.to(dtype).float()) for g in again[1:])
    # other tiles, the same bits: fewer products in a launch, fewer tokens
    for i in (1, 3):
        alone = [t.detach().requires_grad_(j == i) for j, t in enumerate(leaves)]
        (g,) = torch.autograd.grad(gated_ffn(*alone, activation=act), (alone[i],), dy)
        assert torch.equal(g, grads[i])
    part = [leaves[0].detach()[-437:].requires_grad_(True), *leaves[1:]]
    yp = gated_ffn(*part, activation=act)
    (gp,) = torch.autograd.grad(yp, (part[0],), dy[-437:])
    assert torch.equal(yp, y[-437:]) and torch.equal(gp, grads[0][-437:])


def gates(act):
    """bf16 gates over the range where the activation is not 0 in bf16, as exact values."""
    low = {"silu": -87.0, "gelu": -13.0, "gelu_tanh": -9.0}[act]
    g = torch.cat([torch.linspace(low, -low, 1536, device="cuda"), torch.linspace(-4, 4, 512, device="cuda")])
    return g.bfloat16()


def act_tails64(name, g):
    """The activations in forms whose 64-bit values hold in the tails (1 + tanh and 1 + erf cancel)."""
    if name == "silu":
        return g * torch.sigmoid(g)
    if name == "gelu":
        return 0.5 * g * torch.special.erfc(-g * math.sqrt(0.5))
    return g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))


def act_bounds(act, g):
    """act(g), act'(g) and the error that the fast exponential brings to each, in 64 bits.  The
    exponent's argument is rounded in fp32 (one to five roundings of 2^-24), which is a relative
    error of the exponential of as much as its magnitude times that; the rest (the exponential's
    and the reciprocal's own, erfc's fit, the last products) is below 2^-19."""
    gl = g.double().requires_grad_(True)
    a = act_tails64(act, gl)
    (b,) = torch.autograd.grad(a.sum(), gl)
    gl, a = gl.detach(), a.detach()
    arg, roundings = {"silu": (gl.abs(), 2), "gelu": (gl * gl / 2, 3),
                      "gelu_tanh": (2 * math.sqrt(2 / math.pi) * (gl.abs() + 0.044715 * gl.abs() ** 3), 6)}[act]
    rel = roundings * 2.0 ** -24 * arg + 2.0 ** -19
    share = torch.where(gl == 0, 0.5, a / gl)            # σ(g) or Φ(g)
    rest = (b - share).abs()                             # the other term of the derivative
    # towards +∞ the share is 1 − tail: off by fp32's rounding and by the tail's error
    low = torch.minimum(share, 1 - share).clamp(min=0)
    err = torch.where(gl < 0, rel * share, rel * low + 2.0 ** -22)
    # the derivative's other term is σ(1 − σ)·slope for the two with a sigmoid: near σ = 1 the
    # difference 1 − σ of fp32 values is off by 2^-22 (of 1: the sum under the reciprocal 2^-24,
    # the reciprocal 2^-23, the difference 2^-24), which the slope carries into the term
    slope = {"silu": gl.abs(), "gelu": torch.zeros_like(gl),
             "gelu_tanh": 2 * math.sqrt(2 / math.pi) * gl.abs() * (1 + 3 * 0.044715 * gl * gl)}[act]
    eb = err + 2 * rel * rest + 2.0 ** -22 * rest + torch.where(gl > 0, 2.0 ** -22 * slope, 0.0)
    return a, b, err * gl.abs(), eb


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("T", [4, 40, 200, 500])
def test_kept_words_hold_24_bits_and_tails_hold_their_values(T, act):
    """One token's gates are a weight's entries, u is 1 and the second product copies h: a and b
    are cut to 24 bits (2^-15 of the value), y is rounded once, far into the tails."""
    mod = importlib.import_module("dsalt.kernels.gated_ffn")
    g = gates(act)
    F = g.numel()
    x = torch.zeros(T, 8, device="cuda", dtype=torch.bfloat16)
    x[:, 0] = 1
    wg, wu = torch.zeros(F, 8, device="cuda", dtype=torch.bfloat16), torch.zeros(F, 8, device="cuda", dtype=torch.bfloat16)
    wg[:, 0], wu[:, 0] = g, 1
    wd = torch.eye(F, device="cuda", dtype=torch.bfloat16)
    ops = [mod._operand(t, torch.bfloat16) for t in (x, wg, wu, wd)]
    y, kept = mod._forward(*ops, mod.ACTIVATIONS[act], torch.bfloat16, True)
    words = kept[:4, :, :F].contiguous().view(torch.int16).to(torch.int32) & 0xffff
    a, b, ea, eb = act_bounds(act, g)
    smallest = 2.0 ** -118  # where fp32 or the reciprocal goes to 0
    for word, low, val, err in ((words[1], words[3] & 0xff, a, ea), (words[2], words[3] >> 8, b, eb)):
        got = ((word << 16) | (low << 8)).view(torch.float32).double()
        assert ((got - val).abs() <= 2.0 ** -15 * val.abs() + (1 + 2.0 ** -15) * err + smallest).all()
    e = torch.finfo(torch.bfloat16).eps / 2
    assert ((y.double() - a).abs() <= e * a.abs() + (1 + e) * ea + smallest).all()
    tail = (g < -3) & (a.abs() > 2.0 ** -100)
    assert tail.sum() > 100 and (y[:, tail] != 0).all()
