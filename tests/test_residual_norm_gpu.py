"""GPU tests of the fused residual step against its formulas in 64 bits.

The 64-bit formulas take the kernel's own rounded ``x_new`` where the definition does
(the backward; ``h`` is the norm of the sum before its rounding).  Bounds: each result is rounded once to its type (e of the
value) from fp32 sums and products; those are off by c = 2^-18 of the sum of the
terms' magnitudes (row sums of up to 2^6·8 terms a thread and a tree, a reciprocal
square root of 2 ulp, fewer than 20 products).  Sums over T rows: T·2^-24 more.
"""

from __future__ import annotations

import pytest
import torch

from test_counter_dropout_gpu import philox_draws, seed_of

pytestmark = pytest.mark.gpu
C = 2.0 ** -18


def norm64(t, w, eps):
    return t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps) * w


def make(T, d, dtype, wdtype, post, scale, gate, norm, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 13 * T + d)

    def n(*s, std=1.0, mean=0.0, dt=dtype):
        return (torch.randn(*s, generator=g, device="cuda") * std + mean).to(dt).requires_grad_(True)

    t = {"x": n(T, d, std=2.0), "f": n(T, d),
         "post": n(d, std=0.3, mean=1.0, dt=wdtype) if post else None,
         "scale": n(d, std=0.3, mean=0.5, dt=wdtype) if scale else None,
         "gate": {"none": None, "token": n(T, 1), "flat": n(T), "full": n(T, d)}[gate],
         "norm": n(d, std=0.3, mean=1.0, dt=wdtype) if norm else None}
    return t, n(T, d).detach(), n(T, d).detach()


def run(t, p=0.0, seed=None, site=0, eps=1e-6):
    from dsalt.kernels.residual_norm import residual_norm
    return residual_norm(t["x"], t["f"], t["norm"], post_weight=t["post"], scale=t["scale"], gate=t["gate"],
                         dropout_p=p, seed=seed, site=site, eps=eps)


def reference(t, x_new, dx_new, dh, mask, eps=1e-6):
    """{name: (value, magnitude of the terms)} in 64 bits."""
    v = {k: None if s is None else s.detach().double() for k, s in t.items()}
    T, d = v["x"].shape
    gate = 1.0 if v["gate"] is None else v["gate"].view(T, -1)
    scale = 1.0 if v["scale"] is None else v["scale"]
    f = v["f"]
    rf = 1 / torch.sqrt((f * f).mean(-1, keepdim=True) + eps) if v["post"] is not None else 1.0
    post = 1.0 if v["post"] is None else v["post"]
    n = f * rf * post
    branch = mask * scale * gate * n
    out = {"x_new": (v["x"] + branch, v["x"].abs() + branch.abs())}
    xn, s = x_new.detach().double(), out["x_new"][0]
    r = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    G = torch.zeros_like(xn) if dx_new is None else dx_new.double()
    mag = G.abs()
    if v["norm"] is not None:
        out["h"] = (s * r * v["norm"], (out["x_new"][1] + s.abs()) * r * v["norm"].abs())
        if dh is not None:
            q = dh.double() * v["norm"]
            G = G + r * (q - xn * r * r * (q * xn).mean(-1, keepdim=True))
            mag = mag + r * (q.abs() + xn.abs() * r * r * (q * xn).abs().mean(-1, keepdim=True))
            out["norm"] = ((dh.double() * xn * r).sum(0), (dh.double() * xn * r).abs().sum(0))
    out["x"] = (G, mag)
    dn, dn_mag = G * mask * scale * gate, mag * abs(mask * scale * gate)
    q, qm = dn * post, dn_mag * abs(post)
    if v["post"] is not None:
        out["f"] = (rf * (q - f * rf * rf * (q * f).mean(-1, keepdim=True)),
                    rf * (qm + f.abs() * rf * rf * (qm * f.abs()).mean(-1, keepdim=True)))
        out["post"] = ((dn * f * rf).sum(0), (dn_mag * (f * rf).abs()).sum(0))
    else:
        out["f"] = (dn, dn_mag)
    if v["scale"] is not None:
        out["scale"] = ((G * mask * gate * n).sum(0), (mag * (mask * gate * n).abs()).sum(0))
    if v["gate"] is not None:
        dg, dgm = G * mask * scale * n, mag * (mask * scale * n).abs()
        if t["gate"].numel() != T * d:
            dg, dgm = dg.sum(-1), dgm.sum(-1)
        out["gate"] = (dg.reshape(t["gate"].shape), dgm.reshape(t["gate"].shape))
    return out


def check(got, ref, name, T):
    val, mag = ref
    e = torch.finfo(got.dtype).eps / 2
    c = C + (T * 2.0 ** -24 if name in ("post", "scale", "norm") else 0.0)
    err = (got.detach().double() - val).abs()
    bad = ~(err <= e * val.abs() + 1.01 * c * mag + (2.0 ** -25 if got.dtype == torch.float16 else 1e-37))
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {err[bad].max().item():.3g}"


def check_all(t, p=0.0, sd=99, site=3, with_dx=True, with_dh=True, seed=5):
    T, d = t["x"].shape
    g = torch.Generator(device="cuda").manual_seed(seed)
    dx_new, dh = (torch.randn(T, d, generator=g, device="cuda").to(t["x"].dtype) for _ in range(2))
    x_new, h = run(t, p, seed_of(sd) if p else None, site)
    th = round(p * 65536)
    mask = 1.0
    if p:
        keep = (philox_draws(T * d, sd, site) >= th).cuda().view(T, d)
        mask = keep.double() * (65536 / (65536 - th))
    assert (h is None) == (t["norm"] is None)
    dx_new = dx_new if with_dx or h is None else None
    dh = dh if with_dh and h is not None else None
    outs = [(o, g_) for o, g_ in ((x_new, dx_new), (h, dh)) if g_ is not None]
    names = [k for k, s in t.items() if s is not None and (k != "norm" or dh is not None)]
    grads = torch.autograd.grad([o for o, _ in outs], [t[k] for k in names], [g_ for _, g_ in outs])
    ref = reference(t, x_new, dx_new, dh, mask)
    check(x_new, ref["x_new"], "x_new", T)
    if h is not None:
        check(h, ref["h"], "h", T)
    for k, g_ in zip(names, grads):
        assert g_.shape == t[k].shape and g_.dtype == t[k].dtype
        check(g_, ref[k], k, T)
    with torch.no_grad():
        again = run(t, p, seed_of(sd) if p else None, site)
    assert torch.equal(again[0], x_new) and (h is None or torch.equal(again[1], h))


SIZES = [(1, 1), (1, 8), (3, 5), (2, 64), (33, 72), (40, 120), (129, 256), (65, 257), (300, 777), (513, 1024), (37, 2560),
         (9, 4099), (5, 8192), (4, 10000), (3, 16384)]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_everything_on(size, dtype):
    gate = ("token", "full", "flat")[size[0] % 3]
    t, _, _ = make(*size, dtype, dtype, True, True, gate, True)
    check_all(t, p=0.25)


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("scale", [False, True])
@pytest.mark.parametrize("gate", ["none", "token", "full"])
@pytest.mark.parametrize("norm", [False, True])
def test_parts_left_out(post, scale, gate, norm):
    t, _, _ = make(130, 264, torch.bfloat16, torch.float32, post, scale, gate, norm)
    check_all(t, p=0.0)
    check_all(t, p=0.5)


@pytest.mark.parametrize("with_dx,with_dh", [(True, False), (False, True)])
def test_one_output_unused(with_dx, with_dh):
    t, _, _ = make(70, 512, torch.bfloat16, torch.bfloat16, True, True, "token", True)
    check_all(t, p=0.1, with_dx=with_dx, with_dh=with_dh)


def test_mixed_weight_types():
    t, _, _ = make(70, 256, torch.float16, torch.float16, True, True, "none", True)
    t["scale"] = t["scale"].detach().float().requires_grad_(True)
    check_all(t)


def test_same_draws_as_counter_dropout_and_same_sum_as_add_rms_norm():
    from dsalt.kernels.counter_dropout import counter_dropout
    from dsalt.kernels.residual_norm import residual_norm
    from dsalt.kernels.rmsnorm_cuda import add_rms_norm
    x, f = (torch.randn(100, 512, device="cuda") for _ in range(2))
    w = torch.randn(512, device="cuda")
    s = seed_of(4)
    a, _ = residual_norm(x, f, dropout_p=0.5, seed=s, site=7)   # 1 / 0.5 is exact: the same bits
    assert torch.equal(a, x + counter_dropout(f, 0.5, s, 7))
    xb, fb = x.bfloat16(), f.bfloat16()
    got, ref = residual_norm(xb, fb, w, eps=1e-6), add_rms_norm(xb, fb, w, 1e-6)
    assert torch.equal(got[0], ref[0])
    # the norm of the sum before and after its rounding, each rounded: 3 · 2^-9
    assert ((got[1].float() - ref[1].float()).abs() <= 2.0 ** -7 * ref[1].float().abs()).all()


def test_gradient_against_differences():
    """<grad, v> in fp32 against the 64-bit definition's central difference along v."""
    t, dx_new, dh = make(20, 96, torch.float32, torch.float32, True, True, "token", True)
    p, sd = 0.25, 8
    th = round(p * 65536)
    mask = (philox_draws(20 * 96, sd, 0) >= th).cuda().view(20, 96).double() * (65536 / (65536 - th))
    outs = run(t, p, seed_of(sd))
    names = list(t)
    grads = torch.autograd.grad(outs, [t[k] for k in names], [dx_new, dh])

    def loss(v):
        xn = v["x"] + mask * v["scale"] * v["gate"] * norm64(v["f"], v["post"], 1e-6)
        return float((xn * dx_new.double()).sum() + (norm64(xn, v["norm"], 1e-6) * dh.double()).sum())

    base = {k: s.detach().double() for k, s in t.items()}
    for k, g in zip(names, grads):
        v = torch.randn_like(base[k])
        step = 1e-5
        diff = (loss({**base, k: base[k] + step * v}) - loss({**base, k: base[k] - step * v})) / (2 * step)
        mag = float((g.double() * v).abs().sum())  # the terms of the scalar product, each off by C
        assert abs(float((g.double() * v).sum()) - diff) <= 8 * C * mag + 1e-6 * abs(diff) + 1e-6, k


def test_dropped_elements_ignore_what_f_holds():
    """Infinity and NaN in dropped places reach neither the sum nor a gradient (no norm of f there)."""
    t, _, _ = make(16, 64, torch.float32, torch.float32, False, True, "full", True)
    keep = (philox_draws(16 * 64, 1, 0) >= 32768).cuda().view(16, 64)
    clean = {k: s if s is None else s.detach().clone().requires_grad_(True) for k, s in t.items()}
    with torch.no_grad():
        t["f"][~keep] = float("nan")
        clean["f"][~keep] = 0.0
    for a, b in ((t, clean),):
        oa, ob = run(a, 0.5, seed_of(1)), run(b, 0.5, seed_of(1))
        names = [k for k in a if a[k] is not None]
        ga, gb = (torch.autograd.grad(o, [s[k] for k in names], [torch.ones_like(o[0]), torch.ones_like(o[1])])
                  for o, s in ((oa, a), (ob, b)))
        for p, q in zip((*oa, *ga), (*ob, *gb)):
            assert torch.equal(p, q)


def test_all_dropped_zero_rows_and_no_rows():
    t, _, _ = make(30, 128, torch.bfloat16, torch.bfloat16, True, True, "token", True)
    x_new, _ = run(t, 1.0, seed_of(1))
    assert torch.equal(x_new, t["x"])
    (df,) = torch.autograd.grad(x_new.sum(), t["f"])
    assert not df.any()
    with torch.no_grad():
        t["f"].zero_()
        t["x"].zero_()
    outs = run(t)
    grads = torch.autograd.grad([o.sum() for o in outs], [t[k] for k in t])
    assert all(torch.isfinite(o).all() for o in (*outs, *grads)) and not outs[0].any() and not outs[1].any()
    t, _, _ = make(0, 128, torch.bfloat16, torch.bfloat16, True, True, "token", True)
    outs = run(t, 0.5, seed_of(1))
    grads = torch.autograd.grad([o.sum() for o in outs], [t[k] for k in t])
    assert all(g.shape == t[k].shape and not g.any() for g, k in zip(grads, t))


def test_strides_leading_dims_and_unaligned_rows():
    from dsalt.kernels.residual_norm import residual_norm
    x, f = torch.randn(6, 10, 64, device="cuda"), torch.randn(6, 10, 64, device="cuda")
    w, g = torch.randn(64, device="cuda"), torch.rand(6, 10, device="cuda")
    ref = residual_norm(x, f, w, post_weight=w, gate=g)
    assert ref[0].shape == x.shape
    xt = x.transpose(0, 1).contiguous().transpose(0, 1)
    buf = torch.zeros(3841, device="cuda")
    fu = buf[1:].view(6, 10, 64)
    fu.copy_(f)
    wide = torch.stack([w, w], dim=1)[:, 0]
    got = residual_norm(xt, fu, wide, post_weight=wide, gate=g.t().contiguous().t())
    for a, b in zip(ref, got):  # the unaligned pass sums in the same order
        assert torch.equal(a, b)


def test_repeats_streams_and_graph_replay():
    t, dx_new, dh = make(1000, 1024, torch.bfloat16, torch.bfloat16, True, True, "token", True)
    s = seed_of(1)

    def step():
        outs = run(t, 0.1, s)
        return [*outs, *torch.autograd.grad(outs, [t[k] for k in t], [dx_new, dh])]

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
    s.fill_(2)
    graph.replay()
    ref = step()
    assert all(torch.equal(p, q) for p, q in zip(out, ref))


def test_results_end_where_the_tensors_end():
    from dsalt.kernels import _ext
    T, d = 21, 200
    t, dx_new, dh = make(T, d, torch.bfloat16, torch.bfloat16, False, False, "none", True)
    mark = 7.0
    x_new, h, dx, df = (torch.full((T + 3, d), mark, device="cuda", dtype=torch.bfloat16) for _ in range(4))
    r = torch.full((T + 3,), mark, device="cuda")
    parts = torch.empty(_ext.load().dsalt_residual_norm_parts(T, d), 2, d, device="cuda")
    P = _ext.ptr
    p = _ext.ResidualNormParams(x=P(t["x"]), f=P(t["f"]), norm=P(t["norm"]), x_new=P(x_new), h=P(h), r=P(r), dx=P(dx),
                                df=P(df), dx_new=P(dx_new), dh=P(dh), parts=P(parts), T=T, d=d, eps=1e-6,
                                dtype=_ext.BF16)
    _ext.call("dsalt_residual_norm_fwd", p)
    _ext.call("dsalt_residual_norm_bwd", p)
    for buf in (x_new, h, dx, df, r):
        assert (buf[T:] == mark).all() and not (buf[:T] == mark).all()
