"""Pre-norm transformer block with DSALT attention (reference dsalt/modules/dsalt_transformer.py)."""

from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F
import torch.utils.checkpoint

from ..kernels import _ext
from ..kernels import swiglu as swiglu_cuda
from ..kernels.RMSENorm import RMSENorm
from ..kernels.counter_dropout import new_dropout_seed
from ..kernels.gated_ffn import gated_ffn
from ..kernels.residual_norm import residual_norm
from .dsalt_attention import DSALTAttention


_ACTIVATIONS = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda x: F.gelu(x, approximate="tanh")}


class SwiGLUFFN(nn.Module):
    """``down(act(gate(x)) * up(x))``, ``act`` = silu in the reference (:10-21).

    On CUDA in 16-bit compute (autocast, or 16-bit input and weights) the block runs
    as one fused function: ``impl="gemm"`` (silu only) as ``kernels/swiglu.py``'s, one
    gate+up GEMM, the CUDA activation each way, one GEMM per gradient; ``impl="fused"``
    as ``kernels/gated_ffn.py``'s own kernels.  Elsewhere torch's ops.
    """

    def __init__(self, d_model: int, d_ff: int, dropout: float = 0.0, activation: str = "silu", impl: str = "gemm"):
        super().__init__()
        if activation not in _ACTIVATIONS or impl not in ("gemm", "fused"):
            raise ValueError(f"activation must be one of {list(_ACTIVATIONS)} and impl 'gemm' or 'fused', "
                             f"got {activation!r}, {impl!r}")
        self.gate_proj = nn.Linear(d_model, d_ff, bias=False)
        self.up_proj = nn.Linear(d_model, d_ff, bias=False)
        self.down_proj = nn.Linear(d_ff, d_model, bias=False)
        self.drop = nn.Dropout(dropout)
        self.activation = activation
        self.impl = impl

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        w_g, w_u, w_d = self.gate_proj.weight, self.up_proj.weight, self.down_proj.weight
        dt = _ext.half_compute_dtype(x, w_g, w_u, w_d)
        if dt is not None and self.impl == "fused":
            return self.drop(gated_ffn(x, w_g, w_u, w_d, self.activation, dt))
        if dt is not None and self.activation == "silu" and swiglu_cuda.supported(x, w_g):
            return self.drop(swiglu_cuda.swiglu_ffn(x, w_g, w_u, w_d, dt))
        return self.drop(self.down_proj(_ACTIVATIONS[self.activation](self.gate_proj(x)) * self.up_proj(x)))


class ResidualStep(nn.Module):
    """What lies between a branch's output and the residual stream in a block built with
    ``post_norm``, ``residual_scale``, ``residual_gate`` or counter-based dropout:
    ``x + drop(scale * gate * norm(f))``, fused with the norm after it
    (``kernels/residual_norm.py``).  ``gate`` = sigmoid of a linear map of the branch's
    input, one value a token.
    """

    def __init__(self, d_model: int, post_norm: bool, scale: float | None, gate: bool, dropout: float):
        super().__init__()
        self.post_weight = nn.Parameter(torch.ones(d_model)) if post_norm else None
        self.scale = nn.Parameter(torch.full((d_model,), float(scale))) if scale is not None else None
        self.gate = nn.Linear(d_model, 1) if gate else None
        self.dropout = dropout

    def branch(self, f: torch.Tensor, branch_input: torch.Tensor, seed, site: int):
        """The step for a branch's output ``f``, to be taken later: ``(x, norm) -> (x_new, norm(x_new))``,
        without a norm ``(x_new, None)``."""
        gate = torch.sigmoid(self.gate(branch_input)) if self.gate is not None else None
        p = self.dropout if self.training else 0.0

        def add(x: torch.Tensor, norm: RMSENorm | None):
            return residual_norm(x, f.to(x.dtype), None if norm is None else norm.weight, post_weight=self.post_weight,
                                 scale=self.scale, gate=None if gate is None else gate.to(x.dtype), dropout_p=p,
                                 seed=seed, site=site, eps=1e-6 if norm is None else norm.eps)
        return add


class DSALTTransformerBlock(nn.Module):
    """RMSNorm → DSALTAttention → residual, RMSNorm → SwiGLU → residual (reference :24-86).

    ``post_norm``, ``residual_scale``, ``residual_gate`` and ``counter_dropout`` put a
    ``ResidualStep`` on both residual adds (dropout on the feed-forward branch, as the
    reference has it).
    """

    def __init__(self, d_model, n_heads, n_min, n_max, k_lmk, max_seq_len, d_ff, dropout=0.0,
                 yarn_scale=1.0, layer_idx=0, n_kv_heads=None, qkv_bias=False, rope_base=10000.0,
                 ffn_impl="gemm", ffn_activation="silu", post_norm=False, residual_scale=None,
                 residual_gate=False, counter_dropout=False):
        super().__init__()
        self.layer_idx = layer_idx
        self.attn_norm = RMSENorm(d_model)
        self.ffn_norm = RMSENorm(d_model)
        self.attn = DSALTAttention(d_model=d_model, n_heads=n_heads, n_min=n_min, n_max=n_max, k_lmk=k_lmk,
                                   max_seq_len=max_seq_len, dropout=dropout, yarn_scale=yarn_scale,
                                   layer_idx=layer_idx, n_kv_heads=n_kv_heads, qkv_bias=qkv_bias,
                                   rope_base=rope_base)
        self.ffn = SwiGLUFFN(d_model=d_model, d_ff=d_ff, dropout=0.0 if counter_dropout else dropout,
                             activation=ffn_activation, impl=ffn_impl)
        self.attn_step = self.ffn_step = None
        if post_norm or residual_scale is not None or residual_gate or counter_dropout:
            self.attn_step = ResidualStep(d_model, post_norm, residual_scale, residual_gate, 0.0)
            self.ffn_step = ResidualStep(d_model, post_norm, residual_scale, residual_gate,
                                         dropout if counter_dropout else 0.0)

    def forward(self, x, cu_seqlens=None, max_seqlen=None, gradient_checkpointing=False, rope_cs=None,
                cu_list=None, pending=None, defer=False, dropout_seed=None):
        """``(x, aux)`` as the reference block.  ``pending`` / ``defer`` let the model
        fuse each residual add into the RMSNorm after it: with ``pending`` the block
        first forms ``x + pending``; with ``defer`` it returns ``(x, aux, ffn_out)``
        and leaves the final ``x + ffn_out`` to the caller.  In a block with residual
        steps ``pending`` and the deferred value are ``ResidualStep.branch``'s function;
        ``dropout_seed`` is the seed that its dropout takes (drawn here by default)."""
        if self.attn_step is not None:
            return self._forward_steps(x, cu_seqlens, max_seqlen, gradient_checkpointing and self.training, rope_cs,
                                       cu_list, pending, defer, dropout_seed)
        if not (gradient_checkpointing and self.training):
            if pending is not None:
                x, h = self.attn_norm.add_forward(x, pending)
            else:
                h = self.attn_norm(x)
            x_attn, aux = self.attn(h, cu_seqlens=cu_seqlens, max_seqlen=max_seqlen, rope_cs=rope_cs,
                                    cu_list=cu_list)
            x, h = self.ffn_norm.add_forward(x, x_attn)
            f = self.ffn(h)
            return (x, aux, f) if defer else (x + f, aux)
        if pending is not None:
            x = x + pending
        x, aux = self._forward_checkpointed(x, cu_seqlens, max_seqlen, rope_cs, cu_list)
        return (x, aux, None) if defer else (x, aux)

    def _forward_steps(self, x, cu_seqlens, max_seqlen, checkpointed, rope_cs, cu_list, pending, defer, seed):
        """The block with residual steps.  Checkpointing recomputes the branches, not the
        steps, so a dropped element is dropped once."""
        def run(fn, h):
            return torch.utils.checkpoint.checkpoint(fn, h, use_reentrant=False) if checkpointed else fn(h)

        if seed is None and self.training and self.ffn_step.dropout > 0:
            seed = new_dropout_seed(x.device)
        x, h = (x, self.attn_norm(x)) if pending is None else pending(x, self.attn_norm)
        a, aux = run(lambda t: self.attn(t, cu_seqlens=cu_seqlens, max_seqlen=max_seqlen, rope_cs=rope_cs,
                                         cu_list=cu_list), h)
        x, h = self.attn_step.branch(a, h, None, 0)(x, self.ffn_norm)
        add = self.ffn_step.branch(run(self.ffn, h), h, seed, 1 + self.layer_idx)
        # without a norm to come the add alone
        return (x, aux, add) if defer else (add(x, None)[0], aux)

    def _forward_checkpointed(self, x, cu_seqlens, max_seqlen, rope_cs, cu_list):
        """The reference's checkpointed path: attention and FFN recomputed in the backward."""
        aux_box = []

        def attn_fn(h):
            out, a = self.attn(h, cu_seqlens=cu_seqlens, max_seqlen=max_seqlen, rope_cs=rope_cs,
                               cu_list=cu_list)
            aux_box.append(a)
            return out
        x = x + torch.utils.checkpoint.checkpoint(attn_fn, self.attn_norm(x), use_reentrant=False)
        x = x + torch.utils.checkpoint.checkpoint(self.ffn, self.ffn_norm(x), use_reentrant=False)
        aux = aux_box[-1] if aux_box else torch.zeros((), device=x.device, dtype=x.dtype)
        return x, aux

