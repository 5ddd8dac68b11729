"""Rows in 8 bits (e4m3, a scale per row) and the linear layer on them (csrc/rmsnorm.cu, csrc/linear_e4m3.cu)."""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _ops


class Rows8(NamedTuple):
    """``values`` [.., N] float8_e4m3fn, rows on 16-byte boundaries, times ``scales`` [..] fp32, one per row."""
    values: torch.Tensor
    scales: torch.Tensor


def quantize_rows(x) -> Rows8:
    """Rows over the last dimension of x (fp32, bf16, fp16) as ``Rows8``: the largest magnitude of a row at 448, the others to the nearest e4m3."""
    return Rows8(*_ops.ops.quantize_rows(x))
