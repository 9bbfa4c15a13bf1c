"""Cases and plain forms of the feed-forward half of a transformer block.

Three operators that a block runs next to one another:

``ffn``       the gated feed-forward block ``(act(x Wgᵀ) ⊙ (x Wuᵀ)) Wdᵀ`` with its gradients;
``residual``  ``x' = x + drop(scale ⊙ gate ⊙ norm(f))`` and ``h = norm(x')``: the norm after a
              block, its gate, residual scale and dropout, the residual add and the norm before
              the next block, with their gradients;
``dropout``   dropout whose mask comes from a counter-based generator and is never stored.

``run`` computes them in elementary torch operations in 32 bits, or, with ``own``, through the
framework's entry points.
"""

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-6

# the most that one case may ask for: the listed training steps
_MOST_FFN = 18 * 16384 * 1024 * 2816
_MOST_ROWS = 2 * 16384 * 1024


# ------------------------------------------------------------------ cases
def listed():
    def ffn(name, T, d, F, dtype, act, train):
        return {"name": name, "op": "ffn", "T": T, "d": d, "F": F, "dtype": dtype, "act": act, "train": train}

    def residual(name, T, d, dtype, post, scale, gate, p, pre, train):
        return {"name": name, "op": "residual", "T": T, "d": d, "dtype": dtype, "post": post, "scale": scale,
                "gate": gate, "p": p, "pre": pre, "train": train}

    def dropout(name, T, d, dtype, p, train):
        return {"name": name, "op": "dropout", "T": T, "d": d, "dtype": dtype, "p": p, "train": train}

    return [
        # one token of one sequence: the call whose latency a reader waits for
        ffn("ffn one token", 1, 1024, 2816, "bf16", "silu", False),
        # a step of 24 sequences that are answered at the same time
        ffn("ffn 24 tokens", 24, 1024, 2816, "fp16", "gelu", False),
        # a ragged prompt through the small model (d_model 512, 8 heads)
        ffn("ffn prompt", 1531, 512, 1408, "bf16", "silu", False),
        # the training step of the 24-layer model: 8 sequences of 2048
        ffn("ffn training", 16384, 1024, 2816, "bf16", "silu", True),
        # a packed batch whose sizes no tile divides
        ffn("ffn odd training", 1999, 520, 1368, "fp16", "gelu_tanh", True),
        # between two blocks of one token's answer
        residual("residual one token", 1, 1024, "bf16", True, True, "token", 0.0, True, False),
        # the training step of the 24-layer model, everything switched on
        residual("residual training", 16384, 1024, "bf16", True, True, "token", 0.1, True, True),
        # a pre-norm model without gates: the add, the dropout and the next norm
        residual("residual pre-norm", 8192, 512, "fp16", False, False, "none", 0.1, True, True),
        # 32-bit training at a width that no vector divides, a gate for each element
        residual("residual odd", 3001, 777, "fp32", True, True, "full", 0.25, True, True),
        # the embeddings' dropout of the training step
        dropout("dropout training", 16384, 1024, "bf16", 0.1, True),
        # a small odd 32-bit tensor
        dropout("dropout odd", 613, 1001, "fp32", 0.25, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ffn", "ffn", "residual", "residual", "dropout"])
    if op == "ffn":
        step = rng.choice([8, 8, 8, 1])  # widths are multiples of 8 as a rule, not always
        d = max(64 // step, round(_log(rng, 64, 2048) / step)) * step
        F = max(d // step, round(d * rng.uniform(1.0, 4.0) / step)) * step
        train = rng.random() < 0.5
        T = _log(rng, 1, max(1, min(16384, _MOST_FFN // ((18 if train else 6) * d * F))))
        return {"op": op, "T": T, "d": d, "F": F, "dtype": rng.choice(["bf16", "fp16"]),
                "act": rng.choice(["silu", "gelu", "gelu_tanh"]), "train": train}
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    d = _log(rng, 64, 8192)
    if rng.random() < 0.7:
        d = max(8, d // 8 * 8)
    T = _log(rng, 1, max(1, min(32768, _MOST_ROWS // _SIZE[dtype] // d)))
    p = rng.choice([0.0, 0.05, 0.1, 0.25, 0.5])
    if op == "dropout":
        return {"op": op, "T": T, "d": d, "dtype": dtype, "p": p or 0.1, "train": rng.random() < 0.7}
    return {"op": op, "T": T, "d": d, "dtype": dtype, "post": rng.random() < 0.6, "scale": rng.random() < 0.6,
            "gate": rng.choice(["none", "token", "full"]), "p": p, "pre": rng.random() < 0.8,
            "train": rng.random() < 0.6}


def work(case):
    T, d, b = case["T"], case["d"], _SIZE[case["dtype"]]
    n = T * d
    if case["op"] == "ffn":
        w = 3 * d * case["F"]
        if case["train"]:  # x, dy, the weights in; y, dx and the weights' gradients out
            return {"bytes": b * (4 * n + 2 * w), "flops": 18.0 * T * d * case["F"]}
        return {"bytes": b * (2 * n + w), "flops": 6.0 * T * d * case["F"]}
    if case["op"] == "dropout":
        return {"bytes": b * n * (4 if case["train"] else 2), "flops": 0}
    full, token = case["gate"] == "full", case["gate"] == "token"
    vectors = d * (case["post"] + case["scale"] + case["pre"])
    fwd = 3 * n + n * case["pre"] + n * full + T * token + vectors  # x, f, gate in; x', h out
    bwd = 3 * n + n * case["pre"] + n * full + T * token + vectors  # dx', dh in; dx, df, dgate out
    return {"bytes": b * (fwd + (bwd if case["train"] else 0)), "flops": 0}


# ----------------------------------------------------------------- inputs
def prepare(case, seed):
    dt, T, d, train = _DTYPES[case["dtype"]], case["T"], case["d"], case["train"]
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, std=1.0, mean=0.0, grad=True):
        t = (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dt)
        return t.requires_grad_(train and grad)

    s = {"case": case}
    if case["op"] == "ffn":
        F = case["F"]
        # a normalised stream and weights of the size that the models start from
        s.update(x=normal(T, d), w_gate=normal(F, d, std=0.02 * 32 / math.sqrt(d)),
                 w_up=normal(F, d, std=0.02 * 32 / math.sqrt(d)), w_down=normal(d, F, std=0.02))
        if train:
            s["dy"] = normal(T, d, std=0.1, grad=False)
        return s
    if case["p"] > 0:
        s["seed"] = torch.randint(0, 2 ** 62, (1,), generator=g, device="cuda")
    if case["op"] == "dropout":
        s["x"] = normal(T, d)
        if train:
            s["dy"] = normal(T, d, std=0.1, grad=False)
        return s
    s.update(x=normal(T, d, std=2.0), f=normal(T, d))
    s["post"] = normal(d, std=0.2, mean=1.0) if case["post"] else None
    s["scale"] = normal(d, std=0.05, mean=0.3) if case["scale"] else None
    s["pre"] = normal(d, std=0.2, mean=1.0) if case["pre"] else None
    s["gate"] = None
    if case["gate"] != "none":  # a sigmoid's values
        shape = (T, d) if case["gate"] == "full" else (T, 1)
        s["gate"] = torch.sigmoid(torch.randn(*shape, generator=g, device="cuda")).to(dt).requires_grad_(train)
    if train:
        s["dx_new"] = normal(T, d, std=0.1, grad=False)
        s["dh"] = normal(T, d, std=0.1, grad=False) if case["pre"] else None
    return s


# ------------------------------------------------------------ plain forms
def _mulhilo(a, m):
    """High and low 32 bits of a·m for 32-bit values held in int64."""
    lo16, hi16 = (a & 0xFFFF) * m, (a >> 16) * m
    mid = (lo16 >> 16) + (hi16 & 0xFFFFFFFF)
    lo = ((mid & 0xFFFF) << 16) | (lo16 & 0xFFFF)
    return ((hi16 >> 32) << 16) + (mid >> 16), lo


def _keep(n, p, seed, site):
    """The kept elements of a tensor of n: 16-bit draws of Philox4x32-10 that are not below p·2^16.
    Eight consecutive elements share the counter (index / 8, site)."""
    block = torch.arange((n + 7) // 8, device=seed.device)
    c0, c1 = block & 0xFFFFFFFF, block >> 32
    c2, c3 = torch.full_like(block, site), torch.zeros_like(block)
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(10):
        h0, l0 = _mulhilo(c0, 0xD2511F53)
        h1, l1 = _mulhilo(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = torch.stack([c0, c1, c2, c3], dim=1)
    draws = torch.stack([words & 0xFFFF, words >> 16], dim=2).reshape(-1)[:n]
    return draws >= round(p * 65536)


def _mask(case, s, shape):
    """0 where dropped, 1 / (share kept) elsewhere; a number where nothing is dropped."""
    if case["p"] == 0:
        return 1.0
    n = shape[0] * shape[1]
    keep = _keep(n, case["p"], s["seed"], 0).view(shape)
    return keep.float() * (65536.0 / (65536 - round(case["p"] * 65536)))


def _act(name, g):
    """The activation of the gate and its derivative."""
    if name == "silu":
        sig = 1 / (1 + torch.exp(-g))
        return g * sig, sig * (1 + g * (1 - sig))
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    c, k = math.sqrt(2 / math.pi), 0.044715
    t = torch.tanh(c * (g + k * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * k * g * g)


def _plain_ffn(case, s):
    dt = s["x"].dtype
    x, wg, wu, wd = (s[k].float() for k in ("x", "w_gate", "w_up", "w_down"))
    g, u = x @ wg.t(), x @ wu.t()
    a, da = _act(case["act"], g)
    h = a * u
    y = h @ wd.t()
    if not case["train"]:
        return y.to(dt)
    dy = s["dy"].float()
    dh = dy @ wd
    dg, du = dh * u * da, dh * a
    grads = [dg @ wg + du @ wu, dg.t() @ x, du.t() @ x, dy.t() @ h]
    return [y.to(dt)] + [t.to(dt) for t in grads]


def _plain_residual(case, s):
    dt = s["x"].dtype

    def f32(k):
        return None if s[k] is None else s[k].float()

    x, f, post, scale, pre, gate = (f32(k) for k in ("x", "f", "post", "scale", "pre", "gate"))
    m = _mask(case, s, x.shape)
    rf = torch.rsqrt((f * f).mean(-1, keepdim=True) + _EPS)
    n = f * rf * post if post is not None else f
    sc, ga = (1.0 if t is None else t for t in (scale, gate))
    x_new = x + m * sc * ga * n
    r = torch.rsqrt((x_new * x_new).mean(-1, keepdim=True) + _EPS)
    out = [x_new] + ([x_new * r * pre] if pre is not None else [])
    if not case["train"]:
        return [t.to(dt) for t in out]
    dx = s["dx_new"].float()
    if pre is not None:
        dh = s["dh"].float()
        t = dh * pre
        dx = dx + r * (t - x_new * r * r * (t * x_new).mean(-1, keepdim=True))
    dn = dx * m * sc * ga
    df = dn
    if post is not None:
        t = dn * post
        df = rf * (t - f * rf * rf * (t * f).mean(-1, keepdim=True))
    out += [dx, df]
    if post is not None:
        out.append((dn * f * rf).sum(0))
    if scale is not None:
        out.append((dx * m * ga * n).sum(0))
    if gate is not None:
        dgate = dx * m * sc * n
        out.append(dgate if case["gate"] == "full" else dgate.sum(-1, keepdim=True))
    if pre is not None:
        out.append((dh * x_new * r).sum(0))
    return [t.to(dt) for t in out]


def _plain_dropout(case, s):
    m = _mask(case, s, s["x"].shape)
    out = [(s["x"].float() * m).to(s["x"].dtype)]
    if case["train"]:
        out.append((s["dy"].float() * m).to(s["x"].dtype))
    return out


# ------------------------------------------------------- the framework's calls
def _package():
    if "dsalt" not in sys.modules:  # once: a user's program has imported the package
        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "dsalt-library_b200"))


def _own_ffn(case, s):
    from dsalt.kernels.gated_ffn import gated_ffn
    leaves = [s["x"], s["w_gate"], s["w_up"], s["w_down"]]
    if not case["train"]:
        with torch.no_grad():
            return gated_ffn(*leaves, activation=case["act"])
    y = gated_ffn(*leaves, activation=case["act"])
    return [y, *torch.autograd.grad(y, leaves, s["dy"])]


def _own_residual(case, s):
    from dsalt.kernels.residual_norm import residual_norm
    args = dict(post_weight=s["post"], scale=s["scale"], gate=s["gate"], dropout_p=case["p"], seed=s.get("seed"),
                eps=_EPS)
    if not case["train"]:
        with torch.no_grad():
            x_new, h = residual_norm(s["x"], s["f"], s["pre"], **args)
        return [x_new] if h is None else [x_new, h]
    x_new, h = residual_norm(s["x"], s["f"], s["pre"], **args)
    outs, grads = ([x_new], [s["dx_new"]]) if h is None else ([x_new, h], [s["dx_new"], s["dh"]])
    leaves = [s[k] for k in ("x", "f", "post", "scale", "gate", "pre") if s[k] is not None]
    return [*outs, *torch.autograd.grad(outs, leaves, grads)]


def _own_dropout(case, s):
    from dsalt.kernels.counter_dropout import counter_dropout
    if not case["train"]:
        with torch.no_grad():
            return [counter_dropout(s["x"], case["p"], s["seed"])]
    y = counter_dropout(s["x"], case["p"], s["seed"])
    return [y, *torch.autograd.grad(y, [s["x"]], s["dy"])]


def run(state):
    op = state["case"]["op"]
    if own:
        _package()
        return {"ffn": _own_ffn, "residual": _own_residual, "dropout": _own_dropout}[op](state["case"], state)
    with torch.no_grad():
        return {"ffn": _plain_ffn, "residual": _plain_residual, "dropout": _plain_dropout}[op](state["case"], state)


# --------------------------------------------------------------- 64 bits
def _draws64(n, seed, site):
    """The 16-bit draws of a tensor of n, by numpy's 64-bit unsigned products."""
    u = np.uint64
    low = u(0xFFFFFFFF)
    index = np.arange(-(-n // 8), dtype=np.uint64)
    ctr = [index & low, index >> u(32), np.full_like(index, site), np.zeros_like(index)]
    key = [u(seed % 2 ** 32), u(seed >> 32)]
    for i in range(10):
        pa, pb = ctr[0] * u(0xD2511F53), ctr[2] * u(0xCD9E8D57)
        ka = u((int(key[0]) + i * 0x9E3779B9) % 2 ** 32)
        kb = u((int(key[1]) + i * 0xBB67AE85) % 2 ** 32)
        ctr = [(pb >> u(32)) ^ ctr[1] ^ ka, pb & low, (pa >> u(32)) ^ ctr[3] ^ kb, pa & low]
    words = np.stack(ctr, axis=1).astype(np.uint32)
    return words.view(np.uint16).reshape(-1)[:n]


def _drop64(case, s, t):
    if case["p"] == 0:
        return t
    limit = round(case["p"] * 65536)
    draws = torch.from_numpy(_draws64(t.numel(), int(s["seed"]), 0).astype(np.int32)).to(t.device).view(t.shape)
    return torch.where(draws < limit, torch.zeros((), dtype=t.dtype, device=t.device), t / (1 - limit / 65536))


def _norm64(t, w):
    return t / torch.sqrt(torch.mean(t ** 2, dim=-1, keepdim=True) + _EPS) * w


def exact(case, seed):
    """The operator's definition in float64, its gradients by differentiating that definition."""
    s = prepare(case, seed)
    s.pop("case")
    v = {k: t.detach().double().requires_grad_(t.requires_grad) if t is not None and t.is_floating_point() else t
         for k, t in s.items()}
    if case["op"] == "ffn":
        g = torch.nn.functional.linear(v["x"], v["w_gate"])
        act = {"silu": lambda t: t * torch.sigmoid(t),
               "gelu": lambda t: t * torch.special.ndtr(t),
               "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[case["act"]]
        y = torch.nn.functional.linear(act(g) * torch.nn.functional.linear(v["x"], v["w_up"]), v["w_down"])
        if not case["train"]:
            return y
        return [y.detach(), *torch.autograd.grad(y, [v[k] for k in ("x", "w_gate", "w_up", "w_down")], v["dy"])]
    if case["op"] == "dropout":
        out = [_drop64(case, v, v["x"])]
        if case["train"]:
            out += torch.autograd.grad(out[0], [v["x"]], v["dy"])
        return [t.detach() for t in out]
    branch = v["f"] if v["post"] is None else _norm64(v["f"], v["post"])
    for k in ("gate", "scale"):
        branch = branch if v[k] is None else branch * v[k]
    out = [v["x"] + _drop64(case, v, branch)]
    if v["pre"] is not None:
        out.append(_norm64(out[0], v["pre"]))
    if case["train"]:
        grads = [v["dx_new"], v["dh"]][:len(out)]
        leaves = [v[k] for k in ("x", "f", "post", "scale", "gate", "pre") if v[k] is not None]
        out = [*out, *torch.autograd.grad(out, leaves, grads)]
    return [t.detach() for t in out]
