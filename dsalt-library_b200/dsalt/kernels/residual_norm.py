"""From one block to the next in one kernel each way: the norm after a block, its
gate and residual scale, dropout, the residual add and the norm before the next
block (``dsalt_residual_norm_fwd`` / ``_bwd`` in ``csrc/residual_norm.cu``).

``rmsnorm_cuda.add_rms_norm`` is the add and the second norm alone, for four widths.
"""

from __future__ import annotations

from functools import lru_cache

import torch

from . import _ext
from .counter_dropout import check_seed, drop_threshold


def _vectors(dtype: torch.dtype, *vs):
    """The given weight vectors as the kernels read them (all of ``dtype``, or all fp32) and which."""
    f32 = any(v is not None and v.dtype != dtype for v in vs)
    want = torch.float32 if f32 else dtype
    return [v if v is None or (v.dtype == want and v.is_contiguous()) else v.detach().to(want).contiguous()
            for v in vs], f32


@lru_cache(maxsize=1024)
def _parts(T: int, d: int, device: int) -> int:
    """Partial rows of the backward's scratch."""
    with torch.cuda.device(device):
        n = _ext.load().dsalt_residual_norm_parts(T, d)
    if n < 0:
        raise RuntimeError(f"dsalt_residual_norm_parts failed: {_ext.status_string(-n)}")
    return n


def _params(x_new, f, gate, vectors, f32, seed, eps, site, threshold, gate_mode):
    p = _ext.ResidualNormParams(None, f.data_ptr())
    post, scale, norm = vectors
    if gate is not None:
        p.gate = gate.data_ptr()
    if post is not None:
        p.post = post.data_ptr()
    if scale is not None:
        p.scale = scale.data_ptr()
    if norm is not None:
        p.norm = norm.data_ptr()
    if seed is not None:
        p.seed = seed.data_ptr()
    p.x_new, (p.T, p.d), p.eps = x_new.data_ptr(), f.shape, eps
    p.site, p.threshold, p.gate_mode, p.dtype, p.w_f32 = site, threshold, gate_mode, _ext.dtype_code(f.dtype), f32
    return p


def _forward(x, f, gate, vectors, f32, seed, eps, site, threshold, gate_mode, keep: bool):
    """``(x_new, h, rf, r)``; the inverse root mean squares only with ``keep``."""
    x_new, h, rf, r = torch.empty_like(f), None, None, None
    p = _params(x_new, f, gate, vectors, f32, seed, eps, site, threshold, gate_mode)
    p.x = x.data_ptr()
    if vectors[2] is not None:
        h = torch.empty_like(f)
        p.h = h.data_ptr()
        if keep:
            r = torch.empty(p.T, dtype=torch.float32, device=f.device)
            p.r = r.data_ptr()
    if keep and vectors[0] is not None:
        rf = torch.empty(p.T, dtype=torch.float32, device=f.device)
        p.rf = rf.data_ptr()
    _ext.call_on(f.device, "dsalt_residual_norm_fwd", p)
    return x_new, h, rf, r


class ResidualNormFunction(torch.autograd.Function):
    """``(x, f, post, scale, gate, norm, seed, eps, site, threshold, gate_mode) -> (x_new, h)``
    on ``[T, d]``; without ``norm`` only ``x_new``."""

    @staticmethod
    def forward(ctx, x, f, post, scale, gate, norm, seed, eps, site, threshold, gate_mode):
        x, f = _ext.contiguous(x), _ext.contiguous(f)
        g = None if gate is None else _ext.contiguous(gate)
        vectors, f32 = _vectors(f.dtype, post, scale, norm)
        x_new, h, rf, r = _forward(x, f, g, vectors, f32, seed, eps, site, threshold, gate_mode, True)
        ctx.save_for_backward(x_new, f, g, *vectors, seed, rf, r)
        ctx.scalars = (eps, site, threshold, gate_mode)
        ctx.f32 = f32
        ctx.dtypes = [None if v is None else v.dtype for v in (post, scale, norm)]
        ctx.set_materialize_grads(False)
        return x_new if h is None else (x_new, h)

    @staticmethod
    def backward(ctx, dx_new, dh=None):
        _ext.first_derivative_only()
        x_new, f, gate, post, scale, norm, seed, rf, r = ctx.saved_tensors
        p = _params(x_new, f, gate, (post, scale, norm), ctx.f32, seed, *ctx.scalars)
        dx_new, dh = (None if t is None else _ext.contiguous(t) for t in (dx_new, dh))
        dx, df = torch.empty_like(f), torch.empty_like(f)
        dgate = None if gate is None else torch.empty_like(gate)
        need = ctx.needs_input_grad
        dpost = torch.empty_like(post) if post is not None and need[2] else None
        dscale = torch.empty_like(scale) if scale is not None and need[3] else None
        dnorm = torch.empty_like(norm) if norm is not None and need[5] else None
        parts = torch.empty(_parts(p.T, p.d, f.device.index), 2, p.d, dtype=torch.float32, device=f.device)
        p.rf, p.r, p.dx_new, p.dh = _ext.ptr(rf), _ext.ptr(r), _ext.ptr(dx_new), _ext.ptr(dh)
        p.dx, p.df, p.dgate, p.parts = dx.data_ptr(), df.data_ptr(), _ext.ptr(dgate), parts.data_ptr()
        p.dpost, p.dscale, p.dnorm = _ext.ptr(dpost), _ext.ptr(dscale), _ext.ptr(dnorm)
        _ext.call_on(f.device, "dsalt_residual_norm_bwd", p)
        if ctx.f32:
            dpost, dscale, dnorm = (t if t is None else t.to(dt) for t, dt in zip((dpost, dscale, dnorm), ctx.dtypes))
        return dx, df, dpost, dscale, dgate, dnorm, None, None, None, None, None


def residual_norm(x: torch.Tensor, f: torch.Tensor, norm_weight: torch.Tensor | None = None, *,
                  post_weight: torch.Tensor | None = None, scale: torch.Tensor | None = None,
                  gate: torch.Tensor | None = None, dropout_p: float = 0.0, seed: torch.Tensor | None = None,
                  site: int = 0, eps: float = 1e-6):
    """``(x_new, h)``: ``x_new = x + drop(scale * gate * norm(f))`` and ``h = norm(x_new)``.

    ``x`` (the residual stream) and ``f`` (a block's output): ``[..., d]`` of one dtype
    (f16, bf16, f32).  ``post_weight``, ``scale``, ``norm_weight``: ``[d]``, each may be left
    out: no norm of ``f``, no scale, no second norm (``h`` is then None).  ``gate``: x's
    dtype, one value per token (``[...]`` or ``[..., 1]``) or per element (``[..., d]``).
    Dropout draws as ``counter_dropout`` does for a tensor of x's shape.  ``h`` is the
    norm of the sum before it is rounded to ``x_new``.  All sums are fp32.  First derivatives in
    reverse mode only; the gradients of the vectors are summed in a fixed order.
    """
    _ext.require_cuda(x, "x")
    _ext.dtype_code(x.dtype)
    if x.dim() == 0 or f.shape != x.shape or f.dtype != x.dtype:
        raise ValueError(f"x and f must have one shape [..., d] and dtype, got {tuple(x.shape)} {x.dtype} and "
                         f"{tuple(f.shape)} {f.dtype}")
    d = x.shape[-1]
    if not 1 <= d <= _ext.RESIDUAL_MAX_D:
        raise ValueError(f"d must be in [1, {_ext.RESIDUAL_MAX_D}], got {d}")
    for name, v in (("post_weight", post_weight), ("scale", scale), ("norm_weight", norm_weight)):
        if v is not None and (v.shape != (d,) or not v.is_floating_point()):
            raise ValueError(f"{name} must be a floating vector of {d} elements, got {tuple(v.shape)} {v.dtype}")
    gate_mode = _ext.GATE_NONE
    if gate is not None:
        if gate.dtype != x.dtype:
            raise ValueError(f"gate must have x's dtype {x.dtype}, got {gate.dtype}")
        if gate.shape == x.shape:
            gate_mode = _ext.GATE_FULL
        elif gate.shape == x.shape[:-1] or gate.shape == (*x.shape[:-1], 1):
            gate_mode = _ext.GATE_TOKEN
        else:
            raise ValueError(f"gate must have one value per token or element of x {tuple(x.shape)}, "
                             f"got {tuple(gate.shape)}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    threshold = drop_threshold(dropout_p)
    if threshold > 0:
        check_seed(seed, site, x.device)
    else:
        seed, site = None, 0
    dev = x.device
    for t in (f, post_weight, scale, gate, norm_weight):
        if t is not None and t.device != dev:
            _ext.same_device(dev, f=f, post_weight=post_weight, scale=scale, gate=gate, norm_weight=norm_weight)
    x2, f2 = (x, f) if x.dim() == 2 else (x.reshape(-1, d), f.reshape(-1, d))
    if _ext.differentiates(x, f, post_weight, scale, gate, norm_weight):
        out = ResidualNormFunction.apply(x2, f2, post_weight, scale, gate, norm_weight, seed, float(eps), site,
                                         threshold, gate_mode)
        x_new, h = out if norm_weight is not None else (out, None)
    else:
        vectors, f32 = _vectors(x.dtype, post_weight, scale, norm_weight)
        g = None if gate is None else _ext.contiguous(gate)
        x_new, h, _, _ = _forward(_ext.contiguous(x2), _ext.contiguous(f2), g, vectors, f32, seed, float(eps), site, threshold,
                                  gate_mode, False)
    if x.dim() != 2:
        x_new, h = x_new.view(x.shape), None if h is None else h.view(x.shape)
    return x_new, h
