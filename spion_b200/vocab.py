"""Losses over a vocabulary from the rows before the last layer, without the logits (csrc/vocab_loss.cu): cross entropy with labels, and distillation from a teacher's
largest logits.  Rows that do not count cost nothing.

x [.., features] and weight [vocabulary, features] have one type, fp32, bf16 or fp16; under ``torch.autocast`` both are converted to its type.  bias [vocabulary] is fp32 or
16 bits.  The products are exact to fp32's rounding for fp32 operands; for 16-bit ones the gradient of the logits is rounded to the operands' type before it is multiplied, to twice its bits
where rows or work are few (fp16: in units of 2^-13 of the largest |gradient| that arrives at a row, so probabilities below 2^-26 over a row's part of that lose bits in the row's dx, and below 2^-38 all of them).
Under autocast fp32 weights are converted by torch in each call, and their gradient back.
Losses are fp32.  ``reduction``: "mean" over the rows that count (NaN, with gradients of zero, where none does), "sum", or "none" (0 where a row does not count).
"""
from __future__ import annotations

import torch
from torch import nn

from . import _ops
from ._lib import SpionError
from .attention import untouched


def _operands(x, weight):
    if torch.is_autocast_enabled() and x.is_cuda:
        dtype = torch.get_autocast_dtype("cuda")
        return x.to(dtype), weight.to(dtype)
    return x, weight


def linear_cross_entropy(x, weight, labels, bias=None, ignore_index: int = -100, reduction: str = "mean"):
    """``torch.nn.functional.cross_entropy(x @ weight.T + bias, labels, ignore_index=.., reduction=..)``.  labels: int64 or int32, of x's shape without the features.
    A label that is neither ``ignore_index`` nor in the vocabulary makes its row's loss NaN, and with it the gradients."""
    return _ops.ops.linear_cross_entropy(*_operands(x, weight), labels, bias, ignore_index, reduction)


def distill_top_logits(x, weight, indices, teacher_logits, bias=None, temperature: float = 1.0, reduction: str = "mean"):
    """The divergence of ``p = softmax((x @ weight.T + bias) / temperature)``, over the whole vocabulary, from the teacher's ``q = softmax(teacher_logits /
    temperature)`` over the entries that are given: ``sum_j q_j (log q_j - log p[indices_j])`` a row.  indices (int64 or int32) and teacher_logits: [.., k], k up to 128.
    Entries with index -1 or a logit of -inf are left out; a row with no entry left does not count.  An entry that is given twice counts twice.  Other indices outside of the
    vocabulary make the row's loss NaN.  No gradient reaches the teacher."""
    return _ops.ops.distill_top_logits(*_operands(x, weight), indices, teacher_logits, bias, temperature, reduction)


class VocabHead(nn.Linear):
    """``nn.Linear(features, vocabulary)`` whose losses are formed without its logits.  ``tied``: an embedding whose weight is this layer's too.  Losses call no forward of the
    layer: they are refused where it has hooks (those of older weight normalisations and of pruning form the weight) or a forward of its own."""

    def __init__(self, features: int, vocabulary: int, bias: bool = True, tied=None):
        super().__init__(features, vocabulary, bias=bias)
        if tied is not None:
            if tuple(tied.weight.shape) != (vocabulary, features):
                raise ValueError(f"VocabHead: the tied table has shape {tuple(tied.weight.shape)}, the layer {(vocabulary, features)}")
            self.weight = tied.weight

    def _weights(self):
        if not untouched(self, (type(self),)) or type(self).forward is not nn.Linear.forward:
            raise SpionError("VocabHead: a loss calls no forward of the layer, whose hooks or own forward would be passed over")
        return self.weight, self.bias

    def loss(self, x, labels, ignore_index: int = -100, reduction: str = "mean"):
        weight, bias = self._weights()
        return linear_cross_entropy(x, weight, labels, bias, ignore_index, reduction)

    def distill(self, x, indices, teacher_logits, temperature: float = 1.0, reduction: str = "mean"):
        weight, bias = self._weights()
        return distill_top_logits(x, weight, indices, teacher_logits, bias, temperature, reduction)
