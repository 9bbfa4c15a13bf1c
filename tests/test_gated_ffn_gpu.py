"""GPU tests of the gated feed-forward block against its formulas in 64 bits.

Every bound is a sum of the roundings that the kernels make, carried through the
formulas with absolute values (no cancellation assumed):
  * a rounding to the 16-bit type is off by e = finfo.eps / 2 of the value (or half
    the smallest subnormal, f16);
  * a product of length K accumulated in fp32 is off by K·2^-22 of the sum of its
    terms' magnitudes (2^-23 for an addition that truncates, twice that for the
    alignment of the terms of one instruction);
  * the activations' fast exponential and reciprocal are off by 2^-19 of the value.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

ACTS = ["silu", "gelu", "gelu_tanh"]
NAMES = ("x", "w_gate", "w_up", "w_down")


def act64(name, g):
    if name == "silu":
        return g * torch.sigmoid(g)
    if name == "gelu":
        return g * torch.special.ndtr(g)
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))


def reference(x, wg, wu, wd, dy, act):
    """{name: (value, bound)} of y and the gradients, float64."""
    e, tiny = torch.finfo(x.dtype).eps / 2, (2.0 ** -25 if x.dtype == torch.float16 else 0.0)
    x, wg, wu, wd = (t.detach().double() for t in (x, wg, wu, wd))

    def gamma(k):
        return k * 2.0 ** -22

    def mm(p, dp, q, k):  # p·q where p is off by dp and the sum is made in fp32
        return p @ q, dp @ q.abs() + gamma(k) * (p.abs() @ q.abs())

    def rounded(v, dv):
        return v, dv + e * (v.abs() + dv) + tiny

    d, F, T = x.shape[1], wg.shape[0], x.shape[0]
    g, dg_ = mm(x, torch.zeros_like(x), wg.t(), d)
    u, du_ = mm(x, torch.zeros_like(x), wu.t(), d)
    gl = g.clone().requires_grad_(True)
    a = act64(act, gl)
    (b,) = torch.autograd.grad(a.sum(), gl)
    a = a.detach()
    fast = 2.0 ** -19
    # |act'| <= 1.13 and |act''| <= 1.1 for the three activations
    ea, eb = 1.13 * dg_ + fast * (a.abs() + 1e-3 * g.abs()), 1.1 * dg_ + fast * (1 + b.abs())
    h, eh = a * u, a.abs() * du_ + (u.abs() + du_) * ea
    # up to 64 tokens the second product takes h to two 16-bit words
    eh1 = eh + e * e * h.abs() + tiny if T <= 64 else rounded(h, eh)[1]
    out = {"y": rounded(*mm(h, eh1, wd.t(), F))}
    h, eh = rounded(h, eh)
    if dy is None:
        return out
    dy = dy.double()
    av, ea = rounded(a, ea)
    bv, eb = rounded(u * b, b.abs() * du_ + (u.abs() + du_) * eb)
    dh, edh = mm(dy, torch.zeros_like(dy), wd, dy.shape[1])
    du, edu = rounded(dh * av, dh.abs() * ea + (av.abs() + ea) * edh)
    dg, edg = rounded(dh * bv, dh.abs() * eb + (bv.abs() + eb) * edh)
    p, q = mm(dg, edg, wg, 2 * F), mm(du, edu, wu, 2 * F)
    out["x"] = rounded(p[0] + q[0], p[1] + q[1])
    out["w_gate"] = rounded(*(t.t() for t in mm(x.t(), torch.zeros_like(x.t()), dg, T)))
    out["w_up"] = rounded(*(t.t() for t in mm(x.t(), torch.zeros_like(x.t()), du, T)))
    out["w_gate"] = (out["w_gate"][0], out["w_gate"][1] + edg.t() @ x.abs() * (1 + e))
    out["w_up"] = (out["w_up"][0], out["w_up"][1] + edu.t() @ x.abs() * (1 + e))
    p = mm(dy.t(), torch.zeros_like(dy.t()), h, T)
    out["w_down"] = rounded(p[0], p[1] + dy.t().abs() @ eh)
    return out


def check(got, ref, what):
    val, bound = ref
    err = (got.detach().double() - val).abs()
    bad = ~(err <= bound * 1.01 + 1e-30)  # 1 %: products of two errors
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {(err / (bound + 1e-30)).max():.3g} bounds"


def inputs(T, d, F, d_out, dtype, seed=0, grad=True):
    g = torch.Generator(device="cuda").manual_seed(seed + 7 * T + d)

    def n(*s, std=1.0):
        return (torch.randn(*s, generator=g, device="cuda") * std).to(dtype)

    s = 1.0 / math.sqrt(d)
    ts = [n(T, d), n(F, d, std=s), n(F, d, std=s), n(d_out, F, std=1.0 / math.sqrt(F))]
    return [t.requires_grad_(grad) for t in ts] + [n(T, d_out)]


SIZES = [(16, 264, 72, 1000), (17, 1024, 200, 8), (31, 65, 130, 67), (33, 520, 1368, 520), (64, 72, 40, 136), (65, 200, 264, 136),
         (128, 264, 520, 264), (200, 129, 63, 258), (256, 512, 1408, 512), (384, 72, 136, 24), (385, 63, 129, 65),
         (513, 200, 264, 136), (20, 264, 520, 2504), (130, 1032, 136, 2504), (4, 1032, 2056, 40), (700, 2056, 264, 520),
         (1, 8, 8, 8), (1, 64, 96, 64), (2, 1, 1, 1), (3, 17, 5, 9), (5, 40, 72, 40), (17, 72, 136, 24), (64, 256, 512, 256),
         (127, 64, 128, 64), (129, 200, 264, 136), (300, 96, 1000, 96), (257, 63, 129, 65), (640, 512, 1408, 512)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", SIZES)
def test_values_and_gradients(size, dtype):
    from dsalt.kernels.gated_ffn import gated_ffn
    *leaves, dy = inputs(*size, dtype)
    act = ACTS[size[0] % 3]
    y = gated_ffn(*leaves, activation=act)
    grads = torch.autograd.grad(y, leaves, dy)
    ref = reference(*leaves, dy, act)
    assert y.dtype == dtype and y.shape == dy.shape
    check(y, ref["y"], "y")
    for name, g, t in zip(NAMES, grads, leaves):
        assert g.dtype == dtype and g.shape == t.shape
        check(g, ref[name], name)
    with torch.no_grad():  # the inference forward keeps nothing, and rounds the same
        check(gated_ffn(*leaves, activation=act), ref["y"], "y, inference")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_activations_far_out(act, dtype):
    """Gates from -60 to 60: the tails go to 0 and to the identity, nothing overflows."""
    from dsalt.kernels.gated_ffn import gated_ffn
    T, d, F = 160, 16, 64
    *leaves, dy = inputs(T, d, F, 16, dtype, seed=3)
    with torch.no_grad():
        leaves[0][:, 0] = torch.linspace(-60, 60, T, device="cuda").to(dtype)
        leaves[1][:, 0] = 1.0
        leaves[1][:, 1:] *= 0.01
    y = gated_ffn(*leaves, activation=act)
    grads = torch.autograd.grad(y, leaves, dy)
    ref = reference(*leaves, dy, act)
    for name, g in zip(("y",) + NAMES, (y, *grads)):
        check(g, ref[name], name)


def test_gradient_against_differences():
    """<grad, v> against the 64-bit definition's central difference along v."""
    from dsalt.kernels.gated_ffn import gated_ffn
    *leaves, dy = inputs(70, 48, 104, 56, torch.float16, seed=11)
    for act in ACTS:
        grads = torch.autograd.grad(gated_ffn(*leaves, activation=act), leaves, dy)
        ref = reference(*leaves, dy, act)

        def loss(ts):
            x, wg, wu, wd = ts
            return float((((act64(act, x @ wg.t()) * (x @ wu.t())) @ wd.t()) * dy.double()).sum())

        base = [t.detach().double() for t in leaves]
        for i, name in enumerate(NAMES):
            v = torch.randn_like(base[i])
            eps = 1e-4
            up, dn = ([t + s * eps * v if j == i else t for j, t in enumerate(base)] for s in (1, -1))
            diff = (loss(up) - loss(dn)) / (2 * eps)
            dot = float((grads[i].double() * v).sum())
            bound = float((ref[name][1] * v.abs()).sum()) * 1.01 + 1e-5 * abs(diff) + 1e-6
            assert abs(dot - diff) <= bound, f"{act} {name}: {dot} vs {diff}, bound {bound}"


def test_strides_and_shapes():
    """Stacked weights, column slices, transposed and expanded tensors give the results of
    their contiguous copies bit for bit."""
    from dsalt.kernels.gated_ffn import gated_ffn
    dt = torch.bfloat16
    x, wg, wu, wd, dy = inputs(4 * 37, 64, 96, 64, dt, grad=False)
    stacked = torch.cat([wg, wu])                                        # [2F, d]
    wide = torch.cat([x, torch.full_like(x, float("nan"))], dim=1)       # x as a column slice
    odd = torch.cat([torch.zeros(148, 3, device="cuda", dtype=dt), x], dim=1)[:, 3:]   # unaligned rows
    col = wd.t().contiguous().t()                                        # column-major weight
    ref = gated_ffn(x, wg, wu, wd)
    assert torch.equal(ref, gated_ffn(wide[:, :64], stacked[:96], stacked[96:], wd))
    assert torch.equal(ref, gated_ffn(odd, wg, wu, col))
    assert torch.equal(ref.view(4, 37, 64), gated_ffn(x.view(4, 37, 64), wg, wu, wd))
    assert gated_ffn(x[5], wg, wu, wd).shape == (64,)
    one = x[5:6].expand(148, 64)
    assert torch.equal(gated_ffn(one, wg, wu, wd), gated_ffn(one.contiguous(), wg, wu, wd))

    def grads(t):
        leaves = [t.requires_grad_(True), *(w.detach().requires_grad_(True) for w in (wg, wu, wd))]
        return torch.autograd.grad(gated_ffn(*leaves).sum(), leaves)     # dy is an expanded scalar

    a, b = grads(x.clone()), grads(wide[:, :64].detach())
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_no_tokens_and_no_gradient_needed():
    from dsalt.kernels.gated_ffn import gated_ffn
    x, wg, wu, wd, _ = inputs(1, 64, 96, 40, torch.bfloat16)
    y = gated_ffn(x[:0], wg, wu, wd)
    assert y.shape == (0, 40)
    gx, *gw = torch.autograd.grad(y.sum(), (x, wg, wu, wd))
    assert gx.shape == x.shape and all(not g.any() for g in (gx, *gw))
    x, wg, wu, wd, dy = inputs(50, 64, 96, 40, torch.bfloat16)
    full = torch.autograd.grad(gated_ffn(x, wg, wu, wd), (x, wg, wu, wd), dy)
    for i in range(4):  # one leaf at a time: the same gradient
        leaves = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, wg, wu, wd))]
        (g,) = torch.autograd.grad(gated_ffn(*leaves), (leaves[i],), dy)
        assert torch.equal(g, full[i])


def test_other_weight_types_and_autocast():
    """fp32 weights: cast for the products, their gradients the fp32 sums (no second rounding)."""
    from dsalt.kernels.gated_ffn import gated_ffn
    x, wg, wu, wd, dy = inputs(200, 64, 96, 64, torch.bfloat16, grad=False)
    half = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    full = [t.float().requires_grad_(True) for t in (x, wg, wu, wd)]
    ga = torch.autograd.grad(gated_ffn(*half), half, dy)
    y = gated_ffn(*full, dtype=torch.bfloat16)
    assert y.dtype == torch.bfloat16
    gb = torch.autograd.grad(y, full, dy)
    for a, b in zip(ga, gb):
        assert b.dtype == torch.float32
        assert torch.equal(a, b.to(torch.bfloat16))
    assert not torch.equal(gb[1], gb[1].to(torch.bfloat16).float())
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(gated_ffn(*full), y)


def test_repeats_streams_and_graph_replay():
    """The same bits twice, on another stream, and from a replayed graph with new inputs."""
    from dsalt.kernels.gated_ffn import gated_ffn
    *leaves, dy = inputs(333, 96, 264, 96, torch.bfloat16)

    def step():
        y = gated_ffn(*leaves)
        return [y, *torch.autograd.grad(y, leaves, dy)]

    a, b = step(), step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(a, c))
    del a, b, c
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    *other, dy2 = inputs(333, 96, 264, 96, torch.bfloat16, seed=9, grad=False)
    with torch.no_grad():
        for t, s in zip(leaves, other):
            t.copy_(s)
        dy.copy_(dy2)
    graph.replay()
    ref = step()
    assert all(torch.equal(p, q) for p, q in zip(out, ref))


@pytest.mark.parametrize("T", [130, 50])
def test_results_end_where_the_tensors_end(T):
    """The C entries write exactly [T, ·]: rows and columns behind stay as they were."""
    from dsalt.kernels import _ext
    d, F = 40, 72
    x, wg, wu, wd, dy = inputs(T, d, F, d, torch.bfloat16, grad=False)
    mark = 7.0
    f = [torch.full((T + 4, 80), mark, device="cuda", dtype=torch.bfloat16) for _ in range(7)]
    y, dx = (torch.full((T + 4, d), mark, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    dws = [torch.full((n + 2, m), mark, device="cuda") for n, m in ((F, d), (F, d), (d, F))]
    P = _ext.ptr
    p = _ext.GatedFfnParams(x=P(x), w_gate=P(wg), w_up=P(wu), w_down=P(wd), h=P(f[0]), a=P(f[1]), b=P(f[2]), ab=P(f[5]), h_lo=P(f[6]),
                            y=P(y), dy=P(dy), dg=P(f[3]), du=P(f[4]), dx=P(dx), dw_gate=P(dws[0]), dw_up=P(dws[1]),
                            dw_down=P(dws[2]), T=T, ld_x=d, ld_wg=d, ld_wu=d, ld_wd=F, ld_f=80, ld_dy=d, d=d, F=F,
                            d_out=d, dtype=_ext.BF16, w_grad_f32=1)
    for name in ("dsalt_gated_ffn_fwd", "dsalt_gated_ffn_bwd"):
        _ext.call(name, p)
    for t, n in [(t, T) for t in (*f[:6], y, dx)] + list(zip(dws, (F, F, d))):
        assert (t[n:] == mark).all()
        assert not (t[:n, :min(F, t.shape[1])] == mark).all()
    for t in f:
        assert (t[:, F:] == mark).all() and (t[T:] == mark).all()
    assert (f[6] == mark).all() == (T > 64)  # h_lo is the scratch of few tokens
