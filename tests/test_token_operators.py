"""What the operators at a model's two ends refuse, without a GPU: arguments are checked before anything is launched."""
import ctypes

import pytest
import torch

from spion_b200 import _lib
from spion_b200._lib import SpionError


def test_tensors_on_the_cpu_are_refused():
    from spion_b200.tokens import ScaledEmbedding, embed_tokens
    from spion_b200.vocab import VocabHead, distill_top_logits, linear_cross_entropy
    w, ids, x = torch.randn(10, 8), torch.zeros(3, dtype=torch.long), torch.randn(3, 8)
    for call in (lambda: embed_tokens(ids, w), lambda: linear_cross_entropy(x, w, ids), lambda: distill_top_logits(x, w, ids[:, None], torch.zeros(3, 1)),
                 lambda: ScaledEmbedding(10, 8)(ids), lambda: VocabHead(8, 10).loss(x, ids)):
        with pytest.raises(SpionError, match="CUDA"):
            call()


def test_modules_refuse_what_they_do_not_serve():
    from spion_b200.tokens import ScaledEmbedding
    from spion_b200.vocab import VocabHead
    for kw in (dict(max_norm=1.0), dict(scale_grad_by_freq=True), dict(sparse=True)):
        with pytest.raises(ValueError, match="not served"):
            ScaledEmbedding(10, 8, **kw)
    assert ScaledEmbedding(10, 8, max_norm=None, sparse=False).scale == 1.0
    made = ScaledEmbedding.from_pretrained(torch.ones(4, 8), padding_idx=1)
    assert type(made) is ScaledEmbedding and not made.weight.requires_grad and made.padding_idx == 1
    table = ScaledEmbedding(10, 8)
    assert VocabHead(8, 10, tied=table).weight is table.weight
    with pytest.raises(ValueError, match="tied"):
        VocabHead(8, 11, tied=table)


def test_token_rows_arguments_at_the_c_boundary():
    L, d = _lib.lib, ctypes.c_void_p(4096)
    F32, BF16, E4M3 = _lib.F32, _lib.BF16, _lib.E4M3

    def forward(ids=d, w=d, ldw=8, wt=F32, y=d, yt=F32, T=4, V=10, N=8):
        return L.spion_token_rows_forward(ids, w, ldw, wt, y, yt, 1.0, T, V, N, None)

    assert forward(T=0) == 0
    assert forward(T=-1) == -1 and forward(V=-1) == -1 and forward(N=0) == -1 and forward(ldw=7) == -1
    assert forward(ids=None) == -1 and forward(w=None) == -1 and forward(y=None) == -1 and forward(wt=E4M3) == -1 and forward(yt=E4M3) == -1
    assert forward(T=2 ** 31) == -2 and forward(V=2 ** 31) == -2 and forward(N=2 ** 30, ldw=2 ** 30) == -2

    def backward(ids=d, g=d, ldg=8, gt=F32, dw=d, dt=F32, pad=-1, T=4, V=10, N=8, ws=d):
        return L.spion_token_rows_backward(ids, g, ldg, gt, dw, dt, 1.0, pad, T, V, N, ws, None)

    assert backward(V=0) == 0
    assert backward(T=-1) == -1 and backward(V=-1) == -1 and backward(N=0) == -1 and backward(ldg=-1) == -1
    assert backward(ids=None) == -1 and backward(g=None) == -1 and backward(dw=None) == -1 and backward(ws=None) == -1
    assert backward(ws=ctypes.c_void_p(4100)) == -1 and backward(gt=E4M3) == -1 and backward(dt=E4M3) == -1 and backward(T=2 ** 31) == -2
    assert L.spion_token_rows_workspace_bytes(0, 10, 8) == 0 and L.spion_token_rows_workspace_bytes(4, 10, 8) >= 64
    # orders, counts and sums of whole pieces: small beside the gradient
    assert L.spion_token_rows_workspace_bytes(1 << 17, 32000, 1024) < (1 << 17) * 1024 * 4 / 8


def test_vocabulary_loss_arguments_at_the_c_boundary():
    L, d = _lib.lib, ctypes.c_void_p(4096)

    def problem(**kw):
        p = dict(x=d, w=d, bias=None, teacher=None, labels=d, ldx=8, ldw=8, T=4, K=8, V=10, k=1, ignore_index=-100, type=_lib.BF16, bias_type=_lib.F32, teacher_type=_lib.F32,
                 reduction=1, temperature=1.0)
        return _lib.VocabProblem(**{**p, **kw})

    def sizes(**kw):
        return L.spion_vocab_sizes(problem(**kw), None, None, None)

    assert L.spion_vocab_sizes(None, None, None, None) == -1
    for bad in (dict(T=-1), dict(K=0), dict(V=0), dict(k=0), dict(type=_lib.E4M3), dict(temperature=0.0), dict(temperature=float("inf")), dict(temperature=float("nan")),
                dict(ldx=-1), dict(ldw=7), dict(reduction=3), dict(reduction=-1)):
        assert sizes(**bad) == -1, bad
    assert sizes(k=129) == -5
    assert sizes(T=2 ** 30) == -2 and sizes(V=2 ** 30) == -2 and sizes(K=2 ** 30, ldw=2 ** 30) == -2
    assert L.spion_vocab_loss_forward(problem(K=0), d, d, d, None) == -1
    assert L.spion_vocab_loss_backward(problem(V=-3), d, d, d, d, d, _lib.F32, d, None) == -1
