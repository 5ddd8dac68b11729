"""Losses over a vocabulary whose saved tensors come back as other tensors (offloading, hooks, recomputed segments): the same bits, wherever and in rows of whatever strides the values lie.

What the forward leaves for the backward follows from how it could read x and w; the backward's own operands may be readable otherwise."""
import ctypes

import pytest
import torch

from spion_b200 import _lib

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def laid_out(t, pad, offset):
    """The same values, rows `pad` elements further apart, beginning `offset` elements behind a boundary of 512 bytes."""
    if t.dim() == 0:
        return t.clone()
    n = t.shape[-1]
    rows = t.numel() // max(n, 1)
    out = torch.empty(rows * (n + pad) + offset, dtype=t.dtype, device=t.device)[offset:].view(*t.shape[:-1], n + pad)[..., :n]
    return out.copy_(t)


def close_up(t):
    return laid_out(t, 0, 0)


def odd(t):
    return laid_out(t, 3, 1)


def wide(t):
    return laid_out(t, 64 + -t.shape[-1] % 64 if t.dim() else 0, 0)


LAYOUTS = {"close": close_up, "odd": odd, "wide": wide}


def operands(T, K, V, dtype, kept, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + T + K + V)
    x, w = torch.randn(T, K, generator=g, device="cuda").to(dtype), (torch.randn(V, K, generator=g, device="cuda") / K ** 0.5).to(dtype)
    b, labels = torch.randn(V, generator=g, device="cuda"), torch.randint(0, V, (T,), generator=g, device="cuda")
    if kept < 1:
        labels[torch.rand(T, generator=g, device="cuda") >= kept] = -100
        labels[0] = V - 1
    return x, w, b, labels


def gradients(x, w, b, labels, back=None, reduction="mean"):
    from spion_b200.vocab import linear_cross_entropy
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    if back is None:
        loss = linear_cross_entropy(*leaves[:2], labels, leaves[2], reduction=reduction)
    elif back == "cpu":
        with torch.autograd.graph.save_on_cpu():
            loss = linear_cross_entropy(*leaves[:2], labels, leaves[2], reduction=reduction)
    else:
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), back):
            loss = linear_cross_entropy(*leaves[:2], labels, leaves[2], reduction=reduction)
    return [loss.detach(), *torch.autograd.grad(loss, leaves, torch.ones_like(loss))]


def same(got, want):
    return all(torch.equal(p, q) for p, q in zip(got, want)) and all(bool(q.isfinite().all()) for q in want)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,K,V", [(200, 700, 300), (70, 13, 257), (130, 72, 1000)])
@pytest.mark.parametrize("kept", [1.0, 0.6])
def test_operands_that_come_back_laid_out_otherwise(T, K, V, dtype, kept):
    x, w, b, labels = operands(T, K, V, dtype, kept)
    want = gradients(x, w, b, labels)
    for as_x in LAYOUTS.values():
        for as_w in LAYOUTS.values():
            given = as_x(x), as_w(w)
            assert same(gradients(*given, b, labels), want)
            for back in ("cpu", close_up, odd, wide):
                assert same(gradients(*given, b, labels, back), want)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("only", ["x", "w"])
def test_one_operand_alone_comes_back_laid_out_otherwise(dtype, only):
    """... and the other one as it was."""
    x, w, b, labels = operands(150, 72, 333, dtype, 1.0)
    want = gradients(x, w, b, labels)
    shape = tuple(x.shape if only == "x" else w.shape)
    for as_ in LAYOUTS.values():
        for back in LAYOUTS.values():
            given = (as_(x), w) if only == "x" else (x, as_(w))
            assert same(gradients(*given, b, labels, lambda t: back(t) if tuple(t.shape) == shape else t), want)


# copies of w, and of x, too large to stay from the forward
@gpu
@pytest.mark.parametrize("T,K,V", [(40, 1024, 33000), (36000, 1000, 40)])
@pytest.mark.parametrize("kept", [1.0, 0.6])
def test_operands_too_large_to_be_kept(T, K, V, kept):
    x, w, b, labels = operands(T, K, V, torch.bfloat16, kept)
    want = gradients(x, w, b, labels)
    for as_ in LAYOUTS.values():
        for back in ("cpu", close_up, odd, wide):
            assert same(gradients(as_(x), as_(w), b, labels, back), want)


@gpu
@pytest.mark.parametrize("back", ["close", "odd", "wide"])
def test_few_rows_of_fp32(back):
    """These are read as they lie, in other pieces where they lie otherwise: the order of the sums differs, not what is added.  A logit's 300 products, of magnitudes 11 in all, go through
    10 additions of a lane and 5 over lanes: 15 x 2^-24 x 11 = 1e-5; in two orders, in z and in the log of the sum, 4e-5 of a probability.  The sums of dx and dW round by 50 x 2^-24 more of
    magnitudes that are a few times the result: 1e-5."""
    x, w, b, labels = operands(6, 300, 5000, torch.float32, 1.0)
    want = gradients(x, w, b, labels)
    for as_ in LAYOUTS.values():
        for p, q in zip(gradients(as_(x), as_(w), b, labels, LAYOUTS[back]), want):
            assert float((p - q).norm()) <= 5e-5 * float(q.norm())


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_a_teacher_and_a_gradient_per_row(dtype):
    from spion_b200.vocab import distill_top_logits
    x, w, b, labels = operands(90, 72, 400, dtype, 1.0)
    idx = torch.stack([labels, (labels + 7) % 400, torch.full_like(labels, -1)], 1)
    teacher = torch.randn(90, 3, device="cuda")
    given = torch.randn(90, device="cuda")

    def run(x, w, back=None):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), back or (lambda t: t)):
            loss = distill_top_logits(*leaves[:2], idx, teacher, leaves[2], 1.5, "none")
        return [loss.detach(), *torch.autograd.grad(loss, leaves, given)]

    want = run(x, w)
    for as_ in LAYOUTS.values():
        for back in LAYOUTS.values():
            assert same(run(as_(x), as_(w), back), want)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kept", [1.0, 0.6])
def test_recomputed_segments(dtype, kept):
    from torch.utils.checkpoint import checkpoint

    from spion_b200.vocab import linear_cross_entropy
    x, w, b, labels = operands(150, 700, 300, dtype, kept)
    h, table = wide(x).detach(), odd(w).detach()
    results = []
    for recompute in (False, True):
        leaves = [h.detach().requires_grad_(), table.detach().requires_grad_(), b.detach().requires_grad_()]

        def f(h, table, b):
            return linear_cross_entropy(torch.tanh(h)[:, :699], table[:, :699], labels, b)

        loss = checkpoint(f, *leaves, use_reentrant=False) if recompute else f(*leaves)
        results.append([loss.detach(), *torch.autograd.grad(loss, leaves)])
    assert same(*results)


@gpu
def test_a_recorded_backward_of_what_came_back():
    x, w, b, labels = operands(30, 24, 50, torch.float32, 0.8)
    from spion_b200.vocab import linear_cross_entropy
    leaves = [t.requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(linear_cross_entropy(x, w, labels, b), leaves, create_graph=True)
    second = torch.autograd.grad(sum((t ** 2).sum() for t in want), leaves)
    with torch.autograd.graph.save_on_cpu():
        loss = linear_cross_entropy(x, w, labels, b)
    got = torch.autograd.grad(loss, leaves, create_graph=True)
    for p, q in zip(got, want):
        assert torch.equal(p, q)
    assert all(bool(t.isfinite().all()) for t in second)


@gpu
@pytest.mark.parametrize("change", [lambda t: t[:-1] if t.dim() else t, lambda t: t.double() if t.is_floating_point() else t, lambda t: t.cpu()])
def test_what_a_hook_must_not_change(change):
    x, w, b, labels = operands(60, 24, 50, torch.float32, 1.0)
    with pytest.raises(_lib.SpionError, match="hook"):
        gradients(x, w, b, labels, change)
    assert all(bool(t.isfinite().all()) for t in gradients(x, w, b, labels))


def test_layouts_at_the_c_boundary():
    d = ctypes.c_void_p(4096)

    def sizes(**kw):
        p = dict(x=d, w=d, labels=d, ldx=8, ldw=8, T=40, K=8, V=10, k=1, ignore_index=-100, type=_lib.BF16, bias_type=_lib.F32, teacher_type=_lib.F32, reduction=1, temperature=1.0)
        return _lib.lib.spion_vocab_sizes(_lib.VocabProblem(**{**p, **kw}), None, None, None)

    for layout in (-1, 2, 4, 6, 8, 9):
        assert sizes(layout=layout) == -1, layout
    for layout in (1, 5, 7):                               # fp32 is copied, w and x
        assert sizes(type=_lib.F32, layout=layout) == -1, layout
    assert sizes(type=_lib.F32, layout=3, T=4, K=1000, V=1000, ldx=1000, ldw=1000) == -1      # but for few rows and many weights
    assert _lib.lib.spion_vocab_layout(None) == -1 and _lib.lib.spion_vocab_layout(_lib.VocabProblem(T=-1)) == -1
