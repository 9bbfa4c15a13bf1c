"""Dropout from a counter-based generator, without a stored mask.

``counter_dropout(x, p, seed, site)`` drops element ``i`` (row-major index) when its
16-bit draw, a function of ``(seed, site, i)`` alone, is below ``round(p·65536)``.
The backward computes the same draws again, so nothing of the size of ``x`` is kept
for it (``torch.nn.functional.dropout`` keeps a mask).  ``seed`` is a tensor on the
device: a captured graph that writes a new seed into it drops other elements at
every replay.  ``site`` tells the places of one model apart that share a seed.
``residual_norm`` drops with the same draws.
"""

from __future__ import annotations

import torch

from . import _ext


def drop_threshold(p: float) -> int:
    """The 16-bit draws below this are dropped: ``p`` rounded to a multiple of 2^-16."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"the dropout probability must be in [0, 1], got {p}")
    return round(p * 65536)


def check_seed(seed, site: int, device: torch.device) -> None:
    if not isinstance(seed, torch.Tensor) or seed.dtype != torch.int64 or seed.numel() != 1:
        raise TypeError("seed must be an int64 tensor of one element")
    if not 0 <= site < 2 ** 32:
        raise ValueError(f"site must be in [0, 2^32), got {site}")
    if seed.device != device:
        _ext.same_device(device, seed=seed)


def new_dropout_seed(device: torch.device) -> torch.Tensor:
    """A fresh seed from torch's generator of ``device`` (``torch.manual_seed`` governs it;
    in a captured graph every replay draws another)."""
    return torch.randint(0, 2 ** 62, (1,), dtype=torch.int64, device=device)


def _launch(x: torch.Tensor, seed: torch.Tensor, site: int, threshold: int) -> torch.Tensor:
    x = _ext.contiguous(x)
    y = torch.empty_like(x)
    p = _ext.DropoutParams(x.data_ptr(), y.data_ptr(), seed.data_ptr(), x.numel(), site, threshold,
                           _ext.dtype_code(x.dtype))
    _ext.call_on(x.device, "dsalt_dropout", p)
    return y


class CounterDropoutFunction(torch.autograd.Function):
    """``(x, seed, site, threshold) -> y`` of x's shape and dtype."""

    @staticmethod
    def forward(ctx, x, seed, site: int, threshold: int):
        ctx.save_for_backward(seed)
        ctx.site, ctx.threshold = site, threshold
        return _launch(x, seed, site, threshold)

    @staticmethod
    def backward(ctx, dy):
        _ext.first_derivative_only()
        (seed,) = ctx.saved_tensors
        return _launch(dy, seed, ctx.site, ctx.threshold), None, None, None


def counter_dropout(x: torch.Tensor, p: float, seed: torch.Tensor, site: int = 0,
                    training: bool = True) -> torch.Tensor:
    """Dropout of ``x`` (f16, bf16 or f32) with probability ``p``, to the nearest 2^-16.

    Kept elements are divided by the share kept; dropped ones are 0 whatever ``x``
    holds there.  ``x`` itself comes back when nothing is dropped (``p`` rounds to 0, or
    not ``training``).  ``seed`` (int64, one element, on x's device) must not be
    changed before the backward has run: autograd then raises.  First derivatives in
    reverse mode only.
    """
    threshold = drop_threshold(p)
    _ext.require_cuda(x, "x")
    _ext.dtype_code(x.dtype)
    if not training or threshold == 0:
        return x
    check_seed(seed, site, x.device)
    if _ext.differentiates(x):
        return CounterDropoutFunction.apply(x, seed, site, threshold)
    return _launch(x, seed, site, threshold)
