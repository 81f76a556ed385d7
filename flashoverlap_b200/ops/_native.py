"""The overloads of ``torch.ops.flashoverlap_op``, looked up once: a call of few rows is bound by the host."""
import functools

import torch

from .._build import load


@functools.lru_cache(maxsize=None)
def native(name: str):
    load()
    return getattr(torch.ops.flashoverlap_op, name).default
