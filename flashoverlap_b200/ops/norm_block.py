"""The norm behind a block, its gate, the scaled residual stream and the next block's norm as one call, with gradients."""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from .._build import load as _load


def _op():
    _load()
    return torch.ops.flashoverlap_op


class _NormBlock(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, t, post_weight, weight, gate, residual_scale, eps):
        h, y, stats = _op().rmsnorm_add_rmsnorm(x, t, post_weight, weight, gate, residual_scale, eps, True)
        ctx.save_for_backward(x, t, post_weight, weight, gate, stats)
        ctx.residual_scale = residual_scale
        ctx.set_materialize_grads(False)
        return h, y

    @staticmethod
    @once_differentiable
    def backward(ctx, gh, gy):
        if gh is None and gy is None:
            return (None,) * 7
        x, t, post_weight, weight, gate, stats = ctx.saved_tensors
        grads = _op().rmsnorm_add_rmsnorm_backward(gh, gy, x, t, post_weight, weight, gate, stats, ctx.residual_scale)
        return *(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None


def rmsnorm_add_rmsnorm(x: torch.Tensor, t: torch.Tensor, post_weight: torch.Tensor, weight: torch.Tensor,
                        gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0,
                        eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(h, y)`` with ``h = residual_scale * x + gate * (rmsnorm(t) * post_weight)``, ``y = rmsnorm(h) * weight``.

    ``x`` (the residual stream) and ``t`` (the block's output) are [rows, dim], bf16 or fp16, ``dim`` a multiple of 8 up to
    16384; the weights are [dim]; ``gate`` is None, [dim], or [lines, dim] with a line for every ``rows / lines`` consecutive
    rows (one for each sequence, or for each row).  All share one type.  Computed in fp32 and rounded once: ``y`` is the norm of
    ``h`` before its rounding.  ``residual_scale`` and ``eps`` are plain numbers without a gradient."""
    if torch.is_grad_enabled() and any(v is not None and v.requires_grad for v in (x, t, post_weight, weight, gate)):
        return _NormBlock.apply(x, t, post_weight, weight, gate, residual_scale, eps)
    h, y, _ = _op().rmsnorm_add_rmsnorm(x, t, post_weight, weight, gate, residual_scale, eps, False)
    return h, y
