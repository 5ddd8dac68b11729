"""Root-mean-square norm of the encoder's token matrices through the library's kernels (csrc/rmsnorm.cu), with the residual's addition before it.

``s = x + res`` (rounded to the stream's type), ``y = s * weight / sqrt(mean(s^2) + eps)`` over the last dimension, of any width.  The stream is fp32,
bf16 or fp16; the residual and the output have its type, or 16 bits beside an fp32 stream.  The backward forms the gradients of both addends and of the
weight in one pass over the rows.  ``rms_norm_e4m3`` writes the rows in 8 bits with a scale each, for ``spion_b200.quant.linear_e4m3``.
"""
from __future__ import annotations

import torch
from torch import nn

from . import _ops
from .quant import Rows8


def rms_norm(x, weight, eps: float = 1e-6, res=None, out_dtype=None):
    """``y``, or with ``res`` the pair ``(s, y)``.  ``out_dtype``: the stream's type (default), or a 16-bit type beside an fp32 stream."""
    s, y = _ops.ops.rms_norm(x, weight, eps, res, out_dtype)
    return y if res is None else (s, y)


def rms_norm_e4m3(x, weight, eps: float = 1e-6, res=None):
    """The same with ``y`` as ``Rows8``.  It has no gradient: tensors that require one are refused in grad mode."""
    s, values, scales = _ops.ops.rms_norm_e4m3(x, weight, eps, res)
    rows = Rows8(values, scales)
    return rows if res is None else (s, rows)


class FusedRMSNorm(nn.Module):
    """Drop-in for ``nn.RMSNorm(dim)`` beside ``FusedLayerNorm``, with its ``add_norm``.

    ``bf16_out=True``: under ``torch.autocast`` to bf16 the output of an fp32 stream is bf16 (the dtype the next linear layer casts its input to anyway)."""

    def __init__(self, dim: int, eps: float = 1e-6, bf16_out: bool = False):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(dim))
        self.eps = eps
        self.bf16_out = bf16_out

    def _type(self, x):
        bf16 = self.bf16_out and x.dtype == torch.float32 and torch.is_autocast_enabled() and torch.get_autocast_dtype("cuda") == torch.bfloat16
        return torch.bfloat16 if bf16 else None

    def forward(self, x):
        return rms_norm(x, self.weight, self.eps, out_dtype=self._type(x))

    def add_norm(self, x, res):
        """``s = x + res`` and ``self(s)`` in one pass; returns ``(s, self(s))``."""
        if res.dtype != x.dtype and x.dtype != torch.float32:
            res = res.to(x.dtype)
        return rms_norm(x, self.weight, self.eps, res, self._type(x))
