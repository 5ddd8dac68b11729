"""Rows of a token table of any size, with a scale, and the table's gradient by sorted tokens (csrc/token_rows.cu).

``layernorm.TokenEmbedding`` serves tables that fit in shared memory; here the table has any number of rows and any width, in fp32, bf16 or fp16.
"""
from __future__ import annotations

import torch
from torch import nn

from . import _ops


def embed_tokens(ids, weight, scale: float = 1.0, padding_idx=None, out_dtype=None):
    """``weight[ids] * scale`` with one rounding, [.., features].  ids: int64 or int32, any shape; one outside of the table gives a row of NaN and has no gradient.
    padding_idx: a row that gets no gradient (negative ones count from the end).  out_dtype: fp32, bf16 or fp16; default the table's type.  The gradient is summed
    in fp32 in the order of the tokens, the same bits on every run."""
    return _ops.ops.token_rows(ids, weight, scale, padding_idx, out_dtype)


class ScaledEmbedding(nn.Embedding):
    """``nn.Embedding`` (same parameter) times ``scale``, on ``embed_tokens``.  ``bf16_out=True``: under ``torch.autocast`` to bf16 the rows are bf16."""

    def __init__(self, num_embeddings: int, embedding_dim: int, padding_idx=None, scale: float = 1.0, bf16_out: bool = False, **kw):
        refused = [k for k in ("max_norm", "scale_grad_by_freq", "sparse") if kw.pop(k, None)]
        if refused:
            raise ValueError(f"ScaledEmbedding: {', '.join(refused)} not served")
        super().__init__(num_embeddings, embedding_dim, padding_idx, **kw)
        self.scale, self.bf16_out = scale, bf16_out

    def forward(self, ids):
        bf16 = self.bf16_out and torch.is_autocast_enabled() and torch.get_autocast_dtype("cuda") == torch.bfloat16
        return embed_tokens(ids, self.weight, self.scale, self.padding_idx, torch.bfloat16 if bf16 else None)
