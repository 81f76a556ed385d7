"""The norm behind a block, its gate, the scaled residual stream and the next block's norm as one call, with gradients."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ._native import native


def rmsnorm_add_rmsnorm(x: torch.Tensor, t: torch.Tensor, post_weight: torch.Tensor, weight: torch.Tensor,
                        gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0,
                        eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(h, y)`` with ``h = residual_scale * x + gate * (rmsnorm(t) * post_weight)``, ``y = rmsnorm(h) * weight``.

    ``x`` (the residual stream) and ``t`` (the block's output) are [rows, dim], bf16 or fp16, ``dim`` a multiple of 8 up to
    16384; the weights are [dim]; ``gate`` is None, [dim], or [lines, dim] with a line for every ``rows / lines`` consecutive
    rows (one for each sequence, or for each row).  All share one type.  Computed in fp32 and rounded once: ``y`` is the norm of
    ``h`` before its rounding.  ``residual_scale`` and ``eps`` are plain numbers without a gradient."""
    return native("rmsnorm_add_rmsnorm")(x, t, post_weight, weight, gate, residual_scale, eps, False)[:2]
