"""Rows sorted by expert and back, with gradients: what stands around the products of a mixture-of-experts block.

``moe_sort`` turns the router's choices into an order, ``moe_dispatch`` brings the tokens' rows into it (the form the
products by expert take; where a rank's experts follow one another it is also sorted by rank, as ``OverlapImpl.gemm_all2all``
takes its rows, which leaves out the rank's own), ``moe_combine`` sums the experts' rows back into their tokens with the
router's weights.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ._native import native


class ExpertOrder(NamedTuple):
    """Rows of ``tokens * top_k`` choices sorted by expert, an expert's in the order of their tokens.

    As ``moe_sort`` returns it.  To drop a choice (an expert's capacity, padding) set its id to -1 and sort: a -1 written into
    ``slot`` afterwards leaves its row among the expert's, as a row of zeros.  An order made by hand
    has no row twice among its slots and none from ``offsets[-1]`` on; its slots decide, and ``source`` may be None (a launch more)."""
    slot: torch.Tensor      # [tokens, top_k] int32: the row of every choice, -1 for one that is not served here
    source: torch.Tensor    # [tokens * top_k] int32: the choice (token * top_k + k) of every row, -1 behind the last
    offsets: torch.Tensor   # [experts + 1] int32: every expert's first row; the last entry is the number of rows


def moe_sort(ids: torch.Tensor, experts: int) -> ExpertOrder:
    """The order of the choices ``ids`` [tokens, top_k] (int32 or int64) by expert.

    An id outside ``[0, experts)`` is a choice that this GPU does not serve (another rank's expert, padding): it gets no
    row.  A token may choose an expert twice.  At most 1024 experts and 64 choices a token."""
    return ExpertOrder(*native("moe_sort")(ids, experts))


def moe_dispatch(x: torch.Tensor, order: ExpertOrder) -> torch.Tensor:
    """The rows of ``x`` [tokens, dim] in the order: [tokens * top_k, dim], rows that no choice has are zero.

    bf16 or fp16, ``dim`` a multiple of 8.  The gradient of a token is the fp32 sum of its rows', rounded once."""
    return native("moe_dispatch")(x, order[0], order[2], order[1])


def moe_combine(y: torch.Tensor, weights: Optional[torch.Tensor], order: ExpertOrder) -> torch.Tensor:
    """[tokens, dim]: for every token the sum of ``weights[t, k] * y[slot[t, k]]`` over its choices that have a row.

    ``y`` [tokens * top_k, dim] in bf16 or fp16, ``dim`` a multiple of 8; ``weights`` [tokens, top_k] in fp32 or ``y``'s
    type, or None for 1.  Sums are fp32, in the order of the choices, rounded once.  The gradient of a row without a choice
    and of a weight without a row is zero."""
    return native("moe_combine")(y, weights, order[0], order[2], order[1])
