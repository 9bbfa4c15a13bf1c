"""Gated feed-forward block on the library's own tensor-core kernels.

``gated_ffn(x, w_gate, w_up, w_down)`` is ``down(act(gate(x)) * up(x))``, the block
of ``dsalt/modules/dsalt_transformer.py:10-21`` (``act`` = silu there), in f16 or
bf16 with fp32 accumulation.  Both projections, the activation and the product are
one kernel: neither ``gate(x)`` nor ``up(x)`` is written to memory.  A forward that
needs gradients also keeps ``a = act(g)`` and ``b = u·act'(g)``, from which the
backward forms ``du = dh·a`` and ``dg = dh·b`` in the epilogue of the product that
makes ``dh``.  Results are rounded once from the fp32 sums; on the way only the
operands of a further product are rounded to 16 bits, ``h``, ``dg`` and ``du``
(``a`` and ``b`` are cut to 24 bits, and ``h`` to two words in a forward of few tokens).

``swiglu_ffn`` computes the same block with library GEMMs around an activation
kernel, with torch's rounding at every step.
"""

from __future__ import annotations

import torch

from . import _ext
from .dsalt_cuda import device_status_ptr

ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}  # DSALT_ACT_*


def _operand(t: torch.Tensor, dtype: torch.dtype):
    """``(tensor, row stride)`` of a 2-D operand as the kernels read it: ``t`` itself when
    its rows are contiguous, 16-byte aligned and apart, else a copy that is."""
    rows, cols = t.shape
    ld, step = t.stride()
    if t.dtype == dtype and step == 1 and t.data_ptr() % 16 == 0:
        if ld % 8 == 0 and ld >= cols:
            return t, ld
        if rows == 1:
            return t, (cols + 7) // 8 * 8
    ld = (cols + 7) // 8 * 8
    return torch.empty_strided((rows, cols), (ld, 1), dtype=dtype, device=t.device).copy_(t), ld


def _params(x2, wg, wu, wd, activation: int, dtype: torch.dtype):
    (x_, ld_x), (wg_, ld_wg), (wu_, ld_wu), (wd_, ld_wd) = x2, wg, wu, wd
    F, d = wg_.shape
    p = _ext.GatedFfnParams(x_.data_ptr(), wg_.data_ptr(), wu_.data_ptr(), wd_.data_ptr())
    p.status = device_status_ptr(x_.device)
    p.T, p.d, p.F, p.d_out = x_.shape[0], d, F, wd_.shape[0]
    p.ld_x, p.ld_wg, p.ld_wu, p.ld_wd, p.ld_f = ld_x, ld_wg, ld_wu, ld_wd, (F + 7) // 8 * 8
    p.activation, p.dtype = activation, _ext.dtype_code(dtype)
    return p


def _set_kept(p, kept: torch.Tensor, keep: bool) -> None:
    """The pointers into ``kept``: h, then with ``keep`` a, b and ab, then h's low words."""
    step = 2 * p.T * p.ld_f
    base = kept.data_ptr()
    p.h, p.h_lo = base, base + (kept.shape[0] - 1) * step
    if keep:
        p.a, p.b, p.ab = base + step, base + 2 * step, base + 3 * step


def _forward(x2, wg, wu, wd, activation: int, dtype: torch.dtype, keep: bool):
    """``(y, kept)``: ``kept`` holds what a backward needs (with ``keep``) and scratch, in 16-bit words."""
    p = _params(x2, wg, wu, wd, activation, dtype)
    T, dev = p.T, x2[0].device
    kept = torch.empty((4 if keep else 1) + (T <= _ext.FFN_FEW_TOKENS), T, p.ld_f, dtype=dtype, device=dev)
    y = torch.empty(T, p.d_out, dtype=dtype, device=dev)
    _set_kept(p, kept, keep)
    p.y = y.data_ptr()
    _ext.call_on(dev, "dsalt_gated_ffn_fwd", p)
    return y, kept


class GatedFFNFunction(torch.autograd.Function):
    """``(x [T, d], w_gate [F, d], w_up [F, d], w_down [d_out, F], activation, dtype) -> [T, d_out]``."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation: int, dtype: torch.dtype):
        ops = [_operand(t, dtype) for t in (x, w_gate, w_up, w_down)]
        y, kept = _forward(*ops, activation, dtype, True)
        ctx.save_for_backward(*(t for t, _ in ops), kept)
        ctx.activation, ctx.dtype = activation, dtype
        ctx.dtypes = (x.dtype, w_gate.dtype, w_up.dtype, w_down.dtype)
        return y

    @staticmethod
    def backward(ctx, dy):
        _ext.first_derivative_only()
        *ops, kept = ctx.saved_tensors
        dtype, dev = ctx.dtype, kept.device
        # a saved tensor's layout is what came back: hooks (save_on_cpu) return dense copies
        ops = [_operand(t, dtype) for t in ops]
        p = _params(*ops, ctx.activation, dtype)
        _set_kept(p, kept, True)
        dy_, p.ld_dy = _operand(dy, dtype)
        p.dy = dy_.data_ptr()
        need_x, need_g, need_u, need_d = ctx.needs_input_grad[:4]
        if need_x or need_g or need_u:
            scratch = torch.empty(2, p.T, p.ld_f, dtype=dtype, device=dev)
            p.dg = scratch.data_ptr()
            p.du = p.dg and p.dg + 2 * p.T * p.ld_f
        dx = dw_gate = dw_up = dw_down = None
        if need_x:
            dx = torch.empty(p.T, p.d, dtype=dtype, device=dev)
            p.dx = dx.data_ptr()
        # fp32 sums where a weight is not of the compute dtype: its gradient is rounded once
        p.w_grad_f32 = any(dt != dtype for dt in ctx.dtypes[1:])
        out = torch.float32 if p.w_grad_f32 else dtype
        if need_g:
            dw_gate = torch.empty(p.F, p.d, dtype=out, device=dev)
            p.dw_gate = dw_gate.data_ptr()
        if need_u:
            dw_up = torch.empty(p.F, p.d, dtype=out, device=dev)
            p.dw_up = dw_up.data_ptr()
        if need_d:
            dw_down = torch.empty(p.d_out, p.F, dtype=out, device=dev)
            p.dw_down = dw_down.data_ptr()
        _ext.call_on(dev, "dsalt_gated_ffn_bwd", p)
        grads = (dx, dw_gate, dw_up, dw_down)
        return (*(t if t is None or t.dtype == dt else t.to(dt) for t, dt in zip(grads, ctx.dtypes)), None, None)


def _check(x, w_gate, w_up, w_down, activation):
    _ext.require_cuda(x, "x")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    xs, gs, us, ds = x.shape, w_gate.shape, w_up.shape, w_down.shape
    if not xs or len(gs) != 2 or len(ds) != 2:
        raise ValueError("gated_ffn takes x [..., d], w_gate and w_up [F, d], w_down [d_out, F]")
    if xs[-1] != gs[1] or us != gs or ds[1] != gs[0]:
        raise ValueError(f"shapes do not fit: x {tuple(xs)}, w_gate {tuple(gs)}, w_up {tuple(us)}, w_down {tuple(ds)}")
    if 0 in gs or ds[0] == 0:
        raise ValueError("gated_ffn needs widths of at least 1")
    dev = x.device
    if w_gate.device != dev or w_up.device != dev or w_down.device != dev:
        _ext.same_device(dev, w_gate=w_gate, w_up=w_up, w_down=w_down)


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
              activation: str = "silu", dtype: torch.dtype | None = None) -> torch.Tensor:
    """``(act(x w_gateᵀ) * (x w_upᵀ)) w_downᵀ``, ``[..., d] -> [..., d_out]``, in f16 or bf16.

    ``activation``: ``"silu"``, ``"gelu"`` (erf) or ``"gelu_tanh"``.  ``dtype`` is the
    compute dtype; by default autocast's, or the one 16-bit dtype of all four tensors.
    Tensors of other dtypes are cast to it and get gradients of their own dtype.
    Operands are read in place when their rows are contiguous and 16-byte aligned
    (a slice of a stacked weight is), else copied first.  First derivatives in reverse mode only.
    """
    _check(x, w_gate, w_up, w_down, activation)
    if dtype is None:
        dtype = _ext.half_compute_dtype(x, w_gate, w_up, w_down)
    if dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("gated_ffn computes in float16 or bfloat16: pass 16-bit tensors of one dtype, use autocast "
                        f"or give dtype (got x {x.dtype}, w_gate {w_gate.dtype}, dtype {dtype})")
    flat = x.dim() == 2
    x2 = x if flat else x.reshape(-1, x.shape[-1])
    act = ACTIVATIONS[activation]
    if _ext.differentiates(x, w_gate, w_up, w_down):
        y = GatedFFNFunction.apply(x2, w_gate, w_up, w_down, act, dtype)
    else:
        y = _forward(_operand(x2, dtype), _operand(w_gate, dtype), _operand(w_up, dtype), _operand(w_down, dtype), act,
                     dtype, False)[0]
    return y if flat else y.view(*x.shape[:-1], y.shape[1])
