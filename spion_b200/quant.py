"""Rows in 8 bits (e4m3, a scale per row) and the linear layer on them (csrc/rmsnorm.cu, csrc/linear_e4m3.cu).

For calls without gradients: an encoder is trained with ``layernorm.BiasGradLinear`` and evaluated with its weights in 8 bits (``E4M3Linear``), whose input
rows come from ``rmsnorm.rms_norm_e4m3`` as they are needed, or are quantised by the call.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch import nn

from . import _ops


class Rows8(NamedTuple):
    """``values`` [.., N] float8_e4m3fn, rows on 16-byte boundaries, times ``scales`` [..] fp32, one per row."""
    values: torch.Tensor
    scales: torch.Tensor


def quantize_rows(x) -> Rows8:
    """Rows over the last dimension of x (fp32, bf16, fp16) as ``Rows8``: the largest magnitude of a row at 448, the others to the nearest e4m3.  No value of a
    row that holds a NaN or an infinity comes back finite."""
    return Rows8(*_ops.ops.quantize_rows(x))


def linear_e4m3(x, w: Rows8, bias=None, out_dtype=None):
    """``y[.., n] = (sum_k x[.., k] w[n, k]) + bias[n]`` with both operands in 8 bits, sums in fp32.  x: ``Rows8``, or fp32 / bf16 / fp16 rows, which the call
    quantises.  w: ``Rows8`` of [features out, features in].  out_dtype: fp32, bf16 or fp16; default x's type, bf16 for ``Rows8``.  It has no gradient: tensors
    that require one are refused in grad mode."""
    values, scales = x if isinstance(x, Rows8) else (x, None)
    return _ops.ops.linear_e4m3(values, scales, w.values, w.scales, bias, out_dtype)


class E4M3Linear(nn.Module):
    """An ``nn.Linear`` with its weight in 8 bits, for evaluation.  ``out_dtype``: of the result (default: bf16 under autocast to bf16 and for ``Rows8``, else the
    input's type)."""

    def __init__(self, linear: nn.Linear, out_dtype=None):
        super().__init__()
        q = quantize_rows(linear.weight.detach())
        self.register_buffer("values", q.values)
        self.register_buffer("scales", q.scales)
        self.register_buffer("bias", None if linear.bias is None else linear.bias.detach().clone())
        self.in_features, self.out_features, self.out_dtype = linear.in_features, linear.out_features, out_dtype

    def _apply(self, fn, recurse=True):
        """A change of type (``half()``, ``to(dtype)``) is not one of the codes and their scales: they go to the device that it names."""
        codes = {k: self._buffers[k] for k in ("values", "scales")}
        super()._apply(fn, recurse)
        for k, was in codes.items():
            if self._buffers[k].dtype != was.dtype:
                self._buffers[k] = was.to(self._buffers[k].device)
        return self

    def forward(self, x):
        dtype = self.out_dtype
        if dtype is None and torch.is_autocast_enabled() and torch.get_autocast_dtype("cuda") == torch.bfloat16:
            dtype = torch.bfloat16
        return linear_e4m3(x, Rows8(self.values, self.scales), self.bias, dtype)
