"""Linear layers in 8-bit integers: a scale for each token and one for each output channel."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ._native import native


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(q, scale)`` of ``x`` [rows, dim] in bf16 or fp16: with ``a = max(max|x[r]|, 2^-100)``, ``scale[r] = a / 127`` and
    ``q[r]`` the int8 nearest to ``x[r] * (127 / a)``, ties to even, every operation rounded in fp32.  (The quotient is one division;
    torch's ``127.0 / a`` on a GPU is a reciprocal and a product, another number for a quarter of the rows.)

    ``dim`` is a multiple of 8 up to 32768.  A row with a NaN or an infinity gets zeros and the scale NaN, so that
    what is computed from it is NaN."""
    return native("quantize_rows")(x)


def linear_i8(impl, x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
              offsets: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``quantize_rows(x)`` times 8-bit weights, in ``x``'s type: ``y[m, n] = scale[m] * weight_scale[n] * sum_k q[m, k] weight[n, k]``.

    ``impl`` is a single-rank ``OverlapImpl`` (its ``check_status()`` raises if a kernel gave up a wait or found offsets that are
    out of order or of range, whose rows it leaves unwritten); ``x`` is [..., K]
    in bf16 or fp16, ``weight`` int8 [N, K], ``weight_scale`` fp32 [N], K a multiple of 16 up to 32768, N of 8.  With
    ``offsets`` (``ExpertOrder.offsets``) ``weight`` is [experts, N, K] and ``weight_scale`` [experts, N]: rows
    ``offsets[e]`` to ``offsets[e + 1] - 1`` of ``x`` [rows, K] are multiplied by ``weight[e]``, other rows of the result are zero.
    The sums are exact; nothing here has a gradient."""
    return impl.linear_i8(x, weight, weight_scale, offsets)
