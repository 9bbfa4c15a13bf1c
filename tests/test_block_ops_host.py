"""CPU checks of the feed-forward half's operators: what they refuse, before any launch,
and how the model is configured with them.  No kernel runs here."""

from __future__ import annotations

import ctypes

import pytest
import torch

ARG, DT, HD, ALIGN, LARGE = 1, 2, 3, 6, 7  # DSALT_ERR_* of include/dsalt_b200.h


def rc(name, p):
    from dsalt.kernels import _ext
    return getattr(_ext.load(), name)(ctypes.byref(p), ctypes.c_void_p(0))


class OnGpu:
    """A stand-in whose checks must fail before anything touches a device."""

    def __init__(self, *shape, dtype=torch.bfloat16, device="cuda:0", requires_grad=False):
        self.shape, self.dtype, self.device = torch.Size(shape), dtype, torch.device(device)
        self.is_cuda, self.requires_grad = self.device.type == "cuda", requires_grad

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def is_floating_point(self):
        return self.dtype.is_floating_point


def test_gated_ffn_entry_points_reject_bad_arguments():
    from dsalt.kernels import _ext

    def params(**kw):
        base = dict(x=16, w_gate=16, w_up=16, w_down=16, h=16, h_lo=16, y=16, dy=16, T=4, ld_x=64, ld_wg=64, ld_wu=64, ld_wd=96,
                    ld_f=96, ld_dy=64, d=64, F=96, d_out=64, dtype=_ext.BF16)
        return _ext.GatedFfnParams(**{**base, **kw})

    fwd, bwd = "dsalt_gated_ffn_fwd", "dsalt_gated_ffn_bwd"
    assert rc(fwd, params(dtype=_ext.F32)) == DT
    for bad in (dict(T=-1), dict(d=0), dict(F=0), dict(d_out=-8), dict(activation=3), dict(ld_x=56), dict(ld_x=68),
                dict(ld_f=88), dict(ld_wd=90), dict(x=0), dict(w_up=0), dict(h=0), dict(h_lo=0), dict(y=0), dict(a=16), dict(a=16, b=16)):
        assert rc(fwd, params(**bad)) == ARG, bad
    assert rc(fwd, params(x=24)) == ALIGN
    assert rc(fwd, params(T=(1 << 30) + 1)) == LARGE
    assert rc(fwd, params(T=1 << 30, F=1 << 20, ld_wd=1 << 20, ld_f=1 << 20)) == LARGE
    assert rc(fwd, params(T=0, x=0, y=0, h_lo=0)) == 0
    kept = dict(a=16, b=16, ab=16, dg=16, du=16)
    assert rc(bwd, params(dx=16)) == ARG                       # nothing kept by the forward
    assert rc(bwd, params(dx=16, **{**kept, "du": 0})) == ARG
    assert rc(bwd, params(dx=16, **{**kept, "ab": 24})) == ALIGN
    assert rc(bwd, params(dw_down=16, dy=0)) == ARG
    assert rc(bwd, params(dx=16, **{**kept, "dy": 0})) == ARG
    assert rc(bwd, params(T=0)) == 0                           # no gradient asked for


def test_dropout_and_residual_entry_points_reject_bad_arguments():
    from dsalt.kernels import _ext
    d = lambda **kw: _ext.DropoutParams(**{**dict(x=16, y=16, seed=16, n=8, threshold=100, dtype=_ext.BF16), **kw})  # noqa: E731
    assert rc("dsalt_dropout", d(dtype=5)) == DT
    for bad in (dict(n=-1), dict(threshold=-1), dict(threshold=65537), dict(x=0), dict(y=0), dict(seed=0)):
        assert rc("dsalt_dropout", d(**bad)) == ARG, bad
    assert rc("dsalt_dropout", d(n=1 << 42)) == LARGE
    assert rc("dsalt_dropout", d(n=0, x=0)) == 0

    def r(**kw):
        base = dict(x=16, f=16, x_new=16, h=16, norm=16, dx=16, df=16, parts=16, T=4, d=64, eps=1e-6, dtype=_ext.BF16)
        return _ext.ResidualNormParams(**{**base, **kw})

    fwd, bwd = "dsalt_residual_norm_fwd", "dsalt_residual_norm_bwd"
    assert rc(fwd, r(dtype=9)) == DT
    for bad in (dict(T=-1), dict(d=0), dict(eps=-1.0), dict(eps=float("nan")), dict(threshold=70000), dict(threshold=9),
                dict(gate_mode=3), dict(gate_mode=1), dict(x=0), dict(f=0), dict(x_new=0), dict(h=0)):
        assert rc(fwd, r(**bad)) == ARG, bad
    for bad in (dict(dx=0), dict(df=0), dict(parts=0), dict(gate_mode=2, gate=16), dict(post=16), dict(dh=16)):
        assert rc(bwd, r(**bad)) == ARG, bad
    for name in (fwd, bwd):
        assert rc(name, r(d=_ext.RESIDUAL_MAX_D + 8)) == LARGE
        assert rc(name, r(T=1 << 50)) == LARGE
    assert rc(fwd, r(T=0, f=0)) == 0
    lib = _ext.load()
    assert lib.dsalt_residual_norm_parts(-1, 64) == -ARG and lib.dsalt_residual_norm_parts(4, 1 << 20) == -LARGE


def test_operators_refuse_cpu_tensors():
    from dsalt import counter_dropout, gated_ffn, residual_norm
    x, w, v = torch.zeros(4, 8).bfloat16(), torch.zeros(16, 8).bfloat16(), torch.zeros(8, 16).bfloat16()
    for call in (lambda: gated_ffn(x, w, w, v), lambda: residual_norm(x, x), lambda: counter_dropout(x, 0.5, None)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_gated_ffn_refusals():
    from dsalt import gated_ffn
    x, w, v = OnGpu(4, 8), OnGpu(16, 8), OnGpu(8, 16)
    for args in ((OnGpu(4, 9), w, w, v), (x, OnGpu(15, 8), w, v), (x, w, w, OnGpu(8, 15)), (x, OnGpu(16, 8, 1), w, v),
                 (OnGpu(), w, w, v), (OnGpu(4, 0), OnGpu(16, 0), OnGpu(16, 0), v), (x, w, w, OnGpu(0, 16))):
        with pytest.raises(ValueError):
            gated_ffn(*args)
    with pytest.raises(ValueError, match="activation"):
        gated_ffn(x, w, w, v, activation="tanh")
    with pytest.raises(ValueError, match="w_up is on"):
        gated_ffn(x, w, OnGpu(16, 8, device="cuda:1"), v)
    with pytest.raises(TypeError, match="float16 or bfloat16"):  # fp32 without autocast or a dtype
        gated_ffn(*(OnGpu(*t.shape, dtype=torch.float32) for t in (x, w, w, v)))
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        gated_ffn(x, w, w, v, dtype=torch.float32)
    with pytest.raises(TypeError, match="float16 or bfloat16"):  # two 16-bit types
        gated_ffn(x, OnGpu(16, 8, dtype=torch.float16), w, v)


def test_counter_dropout_refusals():
    from dsalt import counter_dropout
    x, seed = OnGpu(4, 8), OnGpu(1, dtype=torch.int64)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="probability"):
            counter_dropout(x, p, seed)
    with pytest.raises(TypeError, match="unsupported dtype"):
        counter_dropout(OnGpu(4, 8, dtype=torch.float64), 0.5, seed)
    for bad in (None, 3, torch.zeros(1), torch.zeros(2, dtype=torch.int64)):
        with pytest.raises(TypeError, match="seed"):
            counter_dropout(x, 0.5, bad)
    with pytest.raises(ValueError, match="site"):
        counter_dropout(x, 0.5, torch.zeros(1, dtype=torch.int64), site=2 ** 32)
    with pytest.raises(ValueError, match="seed is on cpu"):
        counter_dropout(x, 0.5, torch.zeros(1, dtype=torch.int64))


def test_residual_norm_refusals():
    from dsalt import residual_norm
    x, f, w = OnGpu(4, 8), OnGpu(4, 8), OnGpu(8)
    with pytest.raises(ValueError, match="one shape"):
        residual_norm(x, OnGpu(4, 9))
    with pytest.raises(ValueError, match="one shape"):
        residual_norm(x, OnGpu(4, 8, dtype=torch.float32))
    with pytest.raises(ValueError, match="d must be"):
        residual_norm(OnGpu(4, 16385), OnGpu(4, 16385))
    with pytest.raises(ValueError, match="norm_weight must be"):
        residual_norm(x, f, OnGpu(7))
    with pytest.raises(ValueError, match="scale must be"):
        residual_norm(x, f, w, scale=OnGpu(8, dtype=torch.int64))
    with pytest.raises(ValueError, match="gate must have x's dtype"):
        residual_norm(x, f, gate=OnGpu(4, dtype=torch.float32))
    with pytest.raises(ValueError, match="one value per token"):
        residual_norm(x, f, gate=OnGpu(8))
    with pytest.raises(ValueError, match="eps"):
        residual_norm(x, f, eps=-1.0)
    with pytest.raises(TypeError, match="seed"):
        residual_norm(x, f, dropout_p=0.1)
    with pytest.raises(ValueError, match="post_weight is on"):
        residual_norm(x, f, post_weight=OnGpu(8, device="cuda:1"))


def test_config_and_parameters():
    """The reference's model is untouched unless an option is set; the options add parameters only."""
    from dsalt.model import DSALTConfig, DSALTLMHeadModel
    base = dict(vocab_size=64, d_model=32, n_layers=2, n_heads=4, n_min=4, n_max=8, k_lmk=2, max_seq_len=64, d_ff=48,
                dropout=0.1)
    cfg = DSALTConfig(**base)
    assert DSALTConfig.from_dict(cfg.to_dict()) == cfg
    torch.manual_seed(3)
    plain = DSALTLMHeadModel.from_config(cfg)
    keys = set(plain.state_dict())
    assert not any("step" in k for k in keys)
    assert isinstance(plain.layers[0].ffn.drop, torch.nn.Dropout) and plain.layers[0].ffn.drop.p == 0.1
    torch.manual_seed(3)
    again = DSALTLMHeadModel.from_config(DSALTConfig(**base, ffn_impl="fused"))
    assert all(torch.equal(a, b) for a, b in zip(plain.state_dict().values(), again.state_dict().values()))
    full = DSALTLMHeadModel.from_config(DSALTConfig(**base, ffn_impl="fused", ffn_activation="gelu", post_norm=True,
                                                    residual_scale=0.1, residual_gate=True, counter_dropout=True))
    extra = set(full.state_dict()) - keys
    assert keys <= set(full.state_dict())
    assert extra == {f"layers.{i}.{b}_step.{n}" for i in range(2) for b in ("attn", "ffn")
                     for n in ("post_weight", "scale", "gate.weight", "gate.bias")}
    assert full.layers[1].ffn.drop.p == 0.0 and full.layers[1].ffn_step.dropout == 0.1
    assert (full.layers[0].attn_step.scale == 0.1).all()
    for bad in (dict(ffn_impl="other"), dict(ffn_activation="relu")):
        with pytest.raises(ValueError):
            DSALTConfig(**base, **bad)


def test_torch_path_of_the_feed_forward_module():
    """On the CPU the module computes its activation with torch's ops, fused or not."""
    import torch.nn.functional as F
    from dsalt.modules.dsalt_transformer import SwiGLUFFN
    x = torch.randn(5, 16)
    for act, fn in (("silu", F.silu), ("gelu", F.gelu)):
        m = SwiGLUFFN(16, 24, activation=act, impl="fused")
        assert torch.equal(m(x), m.down_proj(fn(m.gate_proj(x)) * m.up_proj(x)))
    with pytest.raises(ValueError):
        SwiGLUFFN(16, 24, activation="relu")
