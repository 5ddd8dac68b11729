"""Losses over a vocabulary (csrc/vocab_loss.cu) against fp64: sizes, types, masks, reductions, targets, strides, values that are not finite, captured calls.

Bounds, u = 2^-24 and S = sum |x w| + |b| of a logit.  Products of two 16-bit numbers are exact in fp32; an fp32 operand in three bf16 parts is exact, and what six of nine
products leave out is below 3 u of a product.  A sum in the tensor cores is truncated, 2 u of the partial sum a step, no more than 64 steps an accumulator (256 where a result has
16 bits), and the accumulators are added in fp32: (128 + accumulators + 24) u S of a logit.  The log of the sum: exponentials to 4 u, sums of up to 128 numbers a thread, then of
V / 64 partial sums by 32 lanes: (192 + V / 2048) u, and 8 u of the numbers themselves in units of log2.  G = r (p - q) carries p's error, and one rounding to 16 bits where
the operands have 16 bits (h = eps / 2; fp16 holds 2^13 G over a power of two near the largest g, whose smallest step is 2^-24).  dx and dW: that error times the other operand's
magnitudes, the sums' (512 + accumulators + 24) u, one rounding.  db is summed before G is rounded."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def inputs(T, K, V, dtype, seed=0, bias=True, size=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + T * 7 + K * 3 + V)
    x = torch.randn(T, K, generator=g, device="cuda").to(dtype)
    w = (torch.randn(V, K, generator=g, device="cuda") * size / math.sqrt(K)).to(dtype)
    b = torch.randn(V, generator=g, device="cuda") if bias else None
    labels = torch.randint(0, V, (T,), generator=g, device="cuda")
    return x, w, b, labels, g


def oracle(x, w, b, rows, idx, q, given, tau):
    """For the rows that count, in fp64: their losses, gradients and bounds of all.  idx, q [rows, k]; given [rows]: what arrives at each row's loss."""
    X, W = x.double()[rows], w.double()
    K, V, n = x.shape[1], w.shape[0], len(rows)
    wide = x.dtype == torch.float32
    bias = torch.zeros(V, dtype=torch.float64, device="cuda") if b is None else b.double()
    z, S = X @ W.t() + bias, X.abs() @ W.abs().t() + bias.abs()
    steps = (6 if wide else 1) * (-(-K // 64)) * 4
    dz = S * U * (2 * min(steps, 64) + steps / 64 + 24) / tau
    z, delta = z / tau, dz.amax(1, keepdim=True)
    lse = torch.logsumexp(z, 1, keepdim=True)
    delta = delta + (192 + V / 2048) * U + 8 * U * torch.maximum(z.abs().amax(1, keepdim=True), lse.abs())
    log_q = torch.where(q > 0, torch.log(q), 0.0)
    each = (q * (log_q - torch.gather(z, 1, idx) + lse)).sum(1)
    each_bound = (2 * delta.squeeze(1)) * q.sum(1) + (q * (log_q.abs() * 8 + 16) * U).sum(1) + 16 * U * each.abs()
    p = torch.exp(z - lse)
    G = p.clone().scatter_add_(1, idx, -q) * given[:, None] / tau
    size = given.abs()[:, None] / tau
    h = 0.0 if wide else torch.finfo(x.dtype).eps / 2
    fine = (p * (2 * delta + 16 * U) + torch.zeros_like(p).scatter_add_(1, idx, q) * 64 * U) * size
    floor = 2.0 ** -25 / 8192 * 2 * given.abs().max() / tau if x.dtype == torch.float16 and n else 0.0
    E = fine + G.abs() * h + floor
    least = 2.0 ** -25 if x.dtype == torch.float16 else 1e-37

    def product(A, dA, B, length):
        steps = (6 if wide else 1) * (-(-length // 64)) * 4
        most = 64 if wide else 256
        want = A @ B
        bound = dA @ B.abs() + (A.abs() @ B.abs()) * U * (2 * min(steps, most) + steps / most + 40)
        return want, bound + want.abs() * (torch.finfo(x.dtype).eps / 2 + 8 * U) + least

    dx, dx_bound = product(G, E, W, V)
    dw, dw_bound = product(G.t(), E.t(), X, n)
    db, db_bound = G.sum(0), fine.sum(0) + G.abs().sum(0) * U * (40 + n / 256) + 1e-37
    return dict(each=(each, each_bound), dx=(dx, dx_bound), dw=(dw, dw_bound), db=(db, db_bound))


def close(got, want, bound, what):
    off = (got.double() - want).abs()
    assert got.shape == want.shape and bool((off <= bound).all()), (what, float((off / bound).nan_to_num(nan=float("inf")).max()))


def check(call, x, w, b, rows, idx, q, tau, reduction, g):
    """call(x, w, b) -> loss.  Losses, gradients, and nothing where a row does not count."""
    T, n = x.shape[0], len(rows)
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    b = None if b is None else b.detach().requires_grad_()
    loss = call(x, w, b)
    assert loss.dtype == torch.float32 and loss.shape == ((T,) if reduction == "none" else ())
    given = torch.randn(loss.shape, generator=g, device="cuda") if reduction == "none" else torch.tensor(1.7, device="cuda")
    grads = torch.autograd.grad(loss, [t for t in (x, w, b) if t is not None], given)
    each_given = given.double()[rows] if reduction == "none" else (given.double() / (n if reduction == "mean" else 1)).expand(n)
    o = oracle(x.detach(), w.detach(), None if b is None else b.detach(), rows, idx, q, each_given, tau)
    each, bound = o["each"]
    if reduction == "none":
        close(loss.detach()[rows], each, bound, "loss")
        out = torch.ones(T, dtype=torch.bool, device="cuda")
        out[rows] = False
        assert bool((loss.detach()[out] == 0).all())
    else:
        scale = n if reduction == "mean" else 1
        close(loss.detach(), each.sum() / scale, bound.sum() / scale + U * each.abs().sum() / scale * 4, "loss")
    dx = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    dx_bound = torch.zeros_like(dx)
    dx[rows], dx_bound[rows] = o["dx"]
    close(grads[0], dx, dx_bound, "dx")
    close(grads[1], *o["dw"], "dw")
    assert grads[0].dtype == x.dtype and grads[1].dtype == w.dtype
    if b is not None:
        want, bound = o["db"]
        rounding = 0.0 if b.dtype == torch.float32 else want.abs() * torch.finfo(b.dtype).eps / 2 + (2.0 ** -25 if b.dtype == torch.float16 else 0.0)
        close(grads[2], want, bound + rounding, "db")
        assert grads[2].dtype == b.dtype
    return loss, grads


def labelled(x, w, b, labels, g, reduction="mean", ignore=-100):
    from spion_b200.vocab import linear_cross_entropy
    rows = (labels != ignore).nonzero().squeeze(1)
    idx = labels[rows].long()[:, None]
    return check(lambda x, w, b: linear_cross_entropy(x, w, labels, b, ignore, reduction), x, w, b, rows, idx, torch.ones(idx.shape, dtype=torch.float64, device="cuda"), 1.0,
                 reduction, g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,K,V", [(1, 1, 1), (1, 64, 2), (2, 16, 10), (31, 64, 128), (64, 77, 129), (65, 100, 257), (129, 256, 1000), (300, 1000, 1003), (5, 2064, 5003),
                                   (1000, 8, 300), (256, 128, 256)])
def test_sizes(T, K, V, dtype):
    x, w, b, labels, g = inputs(T, K, V, dtype)
    labelled(x, w, b, labels, g)
    labelled(x, w, None, labels, g, "none")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,K,V", [(70, 5000, 300), (3, 8, 300000), (70000, 1, 2), (4097, 20, 130), (16385, 8, 40)])
def test_long_in_one_direction(T, K, V, dtype):
    x, w, b, labels, g = inputs(T, K, V, dtype)
    labels[torch.rand(T, generator=g, device="cuda") < 0.1] = -100
    labels[0] = 0
    labelled(x, w, b, labels, g, "mean")


@pytest.mark.parametrize("dtype", TYPES)
def test_large_logits_an_ignored_id_of_the_vocabulary_and_one_tensor_as_both_operands(dtype):
    from spion_b200.vocab import linear_cross_entropy
    x, w, b, labels, g = inputs(200, 64, 300, dtype, size=30.0)
    labelled(x, w, b, labels, g, "none")
    labels[::2] = 3
    labelled(x, w, b, labels, g, "mean", ignore=3)
    table = w.detach()[:90].clone().requires_grad_()
    own = torch.arange(90, device="cuda").flip(0)
    both, = torch.autograd.grad(linear_cross_entropy(table, table, own, reduction="sum"), table)
    rows, cols = table.detach().clone().requires_grad_(), table.detach().clone().requires_grad_()
    dx, dw = torch.autograd.grad(linear_cross_entropy(rows, cols, own, reduction="sum"), (rows, cols))
    torch.testing.assert_close(both, dx + dw)


# (2600, 2064, 5000): pairs of CTAs in all products; (17000, 64, 9000): pieces of the vocabulary; (3000, 64, 256): the contraction of dW shared out; (40, 200, 33000): that of dx
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,K,V", [(2600, 2064, 5000), (17000, 64, 9000), (3000, 64, 256), (40, 200, 33000), (7000, 300, 1100)])
def test_every_kind_of_tile(T, K, V, dtype):
    x, w, b, labels, g = inputs(T, K, V, dtype)
    labelled(x, w, b, labels, g, "sum")
    labels[torch.rand(T, generator=g, device="cuda") < 0.85] = -100
    labelled(x, w, b, labels, g, "mean")


@pytest.mark.parametrize("seed", range(36))
def test_drawn_calls(seed):
    """Sizes, types, masks, targets, strides and reductions at random."""
    import random

    from spion_b200.vocab import distill_top_logits
    rng = random.Random(seed)
    dtype = rng.choice(TYPES)
    T, K, V = (int(2 ** rng.uniform(0, m)) for m in (10.5, 10.5, 12.5))
    if rng.random() < 0.25:
        T, K, V = T * 4, min(K * 3, 3000), V * 2           # on both sides of the tiles of pairs
    x, w, b, labels, g = inputs(T, K, V, dtype, seed=seed, bias=rng.random() < 0.6)
    if rng.random() < 0.3:
        pad = rng.choice([1, 3, 8])
        x = torch.nn.functional.pad(x, (pad, pad))[:, pad:pad + K]
        w = torch.nn.functional.pad(w, (0, pad))[:, :K]
    if b is not None and rng.random() < 0.4:
        b = b.to(rng.choice([torch.bfloat16, torch.float16]))
    reduction, kept = rng.choice(["mean", "sum", "none"]), rng.choice([1.0, 1.0, 0.7, 0.1])
    labels[torch.rand(T, generator=g, device="cuda") >= kept] = -100
    labels[rng.randrange(T)] = rng.randrange(V)
    if rng.random() < 0.5:
        labelled(x, w, b, labels, g, reduction)
        return
    k, tau = int(2 ** rng.uniform(0, 7)), rng.choice([1.0, 2.0, 0.8])
    idx = torch.randint(-1, V, (T, k), generator=g, device="cuda")
    idx[labels < 0] = -1
    idx[(idx >= 0).any(1).logical_not() & (labels >= 0), 0] = 0
    teacher = (2 * torch.randn(T, k, generator=g, device="cuda")).to(rng.choice(TYPES))
    there = idx >= 0
    rows = there.any(1).nonzero().squeeze(1)
    q = torch.softmax(torch.where(there, teacher.double(), -float("inf"))[rows] / tau, 1)
    check(lambda x, w, b: distill_top_logits(x, w, idx, teacher, b, tau, reduction), x, w, b, rows, idx[rows].clamp_min(0), q, tau, reduction, g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kept", [0.0, 0.01, 0.5, 0.99])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_rows_that_do_not_count(dtype, kept, reduction):
    """Whatever they hold, and whatever arrives at their losses."""
    from spion_b200.vocab import linear_cross_entropy
    x, w, b, labels, g = inputs(517, 72, 300, dtype, seed=1)
    out = torch.rand(517, generator=g, device="cuda") >= kept
    labels[out] = -7
    x[out] = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min], device="cuda").to(dtype).repeat(18)
    if not bool((~out).any()):
        x, w, b = x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
        loss = linear_cross_entropy(x, w, labels, b, -7, reduction)
        if reduction == "mean":
            assert bool(loss.isnan())
        else:
            assert bool((loss == 0).all())
        for t in torch.autograd.grad(loss, (x, w, b), torch.ones_like(loss)):
            assert bool((t == 0).all())
        return
    labelled(x, w, b, labels, g, reduction, ignore=-7)
    if reduction == "none":
        x, w = x.requires_grad_(), w.requires_grad_()
        loss = linear_cross_entropy(x, w, labels, b, -7, "none")
        given = torch.where(out, float("nan"), 1.0)
        for t in torch.autograd.grad(loss, (x, w), given):
            assert bool(t.isfinite().all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k,tau", [(1, 1.0), (3, 2.0), (32, 0.7), (33, 1.0), (128, 3.0)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_distillation(dtype, k, tau, reduction):
    from spion_b200.vocab import distill_top_logits
    T, V = 200, 700
    x, w, b, _, g = inputs(T, 80, V, dtype, seed=k)
    idx = torch.rand(T, V, generator=g, device="cuda").argsort(1)[:, :k].contiguous()
    if k > 2:
        idx[:20, 1] = idx[:20, 0]                          # twice: counts twice
    teacher = (3 * torch.randn(T, k, generator=g, device="cuda")).to(dtype)
    idx[(torch.rand(T, k, generator=g, device="cuda") < 0.2)] = -1
    idx[5] = -1
    teacher[7, 0] = -float("inf")
    teacher[9] = -float("inf")
    teacher[11] = torch.finfo(dtype).min                   # equal, however low
    idx[11] = torch.arange(k, device="cuda")
    there = (idx >= 0) & (teacher != -float("inf"))
    rows = there.any(1).nonzero().squeeze(1)
    q = torch.softmax(torch.where(there, teacher.double() / tau, -float("inf"))[rows], 1)
    q = torch.where(there[rows], q, 0.0)
    assert 5 not in rows and 9 not in rows and 11 in rows
    check(lambda x, w, b: distill_top_logits(x, w, idx, teacher, b, tau, reduction), x, w, b, rows, idx[rows].clamp_min(0), q, tau, reduction, g)


@pytest.mark.parametrize("dtype", TYPES)
def test_targets_side_by_side_and_many_times_the_same(dtype):
    """More targets among a thread's 64 columns than it remembers."""
    from spion_b200.vocab import distill_top_logits
    T, V, k = 140, 500, 40
    x, w, b, _, g = inputs(T, 64, V, dtype, seed=9)
    idx = torch.randint(0, V - k, (T, 1), generator=g, device="cuda") + torch.arange(k, device="cuda")
    idx[:40] = idx[:40, :1]                                # one id, forty times
    idx[40:60, ::3] = 77
    teacher = torch.randn(T, k, generator=g, device="cuda")
    q = torch.softmax(teacher.double(), 1)
    rows = torch.arange(T, device="cuda")
    check(lambda x, w, b: distill_top_logits(x, w, idx, teacher, b), x, w, b, rows, idx, q, 1.0, "mean", g)
    check(lambda x, w, b: distill_top_logits(x, w, idx, teacher, b, reduction="none"), x, w, None, rows, idx, q, 1.0, "none", g)


def test_more_rows_than_one_pass_takes():
    """Partial sums are kept for a part of the rows at a time; a row's are its own."""
    from spion_b200.vocab import linear_cross_entropy
    x, w, b, labels, g = inputs(40000, 16, 64000, torch.bfloat16)
    for kept in (1.0, 0.9):
        labels[torch.rand(40000, generator=g, device="cuda") >= kept] = -100
        each = linear_cross_entropy(x, w, labels, b, reduction="none")
        parts = torch.cat([linear_cross_entropy(x[i:i + 20000], w, labels[i:i + 20000], b, reduction="none") for i in (0, 20000)])
        assert torch.equal(each, parts)
        mean, n = each.double().sum() / (labels >= 0).sum(), int((labels >= 0).sum())
        assert abs(float(linear_cross_entropy(x, w, labels, b)) - float(mean)) <= 2.0 ** -23 * float(mean)
        assert abs(float(linear_cross_entropy(x, w, labels, b, reduction="sum")) - float(mean) * n) <= 2.0 ** -23 * float(mean) * n


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,K,V", [(1, 64, 20000), (16, 200, 32000), (64, 72, 37888), (64, 64, 37700), (33, 8, 37889), (5, 1100, 32001), (2, 24, 128000)])
def test_few_rows_and_a_large_vocabulary(T, K, V, dtype):
    """Tiles as wide as the vocabulary asks for, targets on both sides of their ends."""
    from spion_b200.vocab import distill_top_logits
    x, w, b, labels, g = inputs(T, K, V, dtype)
    labels[-1] = V - 1
    labelled(x, w, b, labels, g, "none")
    idx = (torch.randint(0, V // 32, (T, 30), generator=g, device="cuda") * 32 + torch.arange(-15, 15, device="cuda") % 4).clamp(0, V - 1)
    idx[:, 5:] = (idx[:, :1] + torch.arange(25, device="cuda")).clamp(0, V - 1)
    teacher = torch.randn(T, 30, generator=g, device="cuda")
    rows = torch.arange(T, device="cuda")
    check(lambda x, w, b: distill_top_logits(x, w, idx, teacher, b, 1.3), x, w, None, rows, idx, torch.softmax(teacher.double() / 1.3, 1), 1.3, "mean", g)


def test_one_entry_of_weight_one_is_the_cross_entropy():
    from spion_b200.vocab import distill_top_logits, linear_cross_entropy
    x, w, b, labels, g = inputs(100, 64, 500, torch.bfloat16)
    assert torch.equal(linear_cross_entropy(x, w, labels, b, reduction="none"),
                       distill_top_logits(x, w, labels[:, None], torch.zeros(100, 1, device="cuda"), b, reduction="none"))


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_offsets_shapes_and_label_types(dtype):
    from spion_b200.vocab import linear_cross_entropy
    x, w, b, labels, g = inputs(6 * 50, 72, 333, dtype)
    want = linear_cross_entropy(x, w, labels, b, reduction="none")

    def grads(x, w, b, labels):
        x, w, b = x.detach().requires_grad_(), w.detach().requires_grad_(), b.detach().requires_grad_()
        loss = linear_cross_entropy(x, w, labels, b)
        return [loss, *torch.autograd.grad(loss, (x, w, b))]

    plain = grads(x, w, b, labels)
    off = torch.empty(300 * 75 + 1, device="cuda", dtype=dtype)[1:].view(300, 75)[:, :72]
    off.copy_(x)
    woff = torch.empty(333 * 73 + 3, device="cuda", dtype=dtype)[3:].view(333, 73)[:, 1:]
    woff.copy_(w)
    boff = torch.empty(333, 2, device="cuda")[:, 1]
    boff.copy_(b)
    for a in ((off, w, b, labels), (x, woff, b, labels), (x.t().contiguous().t(), w.t().contiguous().t(), boff, labels.int())):
        for p, q in zip(plain, grads(*a)):
            assert torch.equal(p, q)
    assert torch.equal(linear_cross_entropy(x.view(6, 50, 72), w, labels.view(6, 50), b, reduction="none"), want.view(6, 50))
    assert torch.equal(linear_cross_entropy(x.view(6, 50, 72).transpose(0, 1), w, labels.view(6, 50).t(), b, reduction="none"), want.view(6, 50).t())
    assert torch.equal(linear_cross_entropy(x[0], w, labels[0], b, reduction="none"), want[0])
    one = linear_cross_entropy(x[:1].expand(300, 72), w, labels, b, reduction="none")
    assert torch.equal(one, linear_cross_entropy(x[:1].repeat(300, 1), w, labels, b, reduction="none"))
    same = w[:1].expand(333, 72)
    close(linear_cross_entropy(x, same, labels, None), torch.tensor(math.log(333), dtype=torch.float64, device="cuda"), torch.tensor(1e-4, device="cuda"), "equal logits")
    empty = torch.empty(0, 72, device="cuda", dtype=dtype, requires_grad=True)
    none = torch.empty(0, dtype=torch.long, device="cuda")
    assert linear_cross_entropy(empty, w, none, b, reduction="none").shape == (0,)
    assert bool(linear_cross_entropy(empty, w, none, b).isnan()) and bool(linear_cross_entropy(empty, w, none, b, reduction="sum") == 0)
    w2 = w.detach().requires_grad_()
    dw, dx = torch.autograd.grad(linear_cross_entropy(empty, w2, none, b, reduction="sum"), (w2, empty))
    assert bool((dw == 0).all()) and dx.shape == (0, 72)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_are_not_finite_and_labels_outside(dtype):
    from spion_b200.vocab import distill_top_logits, linear_cross_entropy
    x, w, b, labels, g = inputs(90, 64, 200, dtype)
    x[3, 5] = float("nan")
    x[4, 6] = float("inf")
    labels[7], labels[8], labels[9] = 200, -1, 2 ** 40
    bad = torch.tensor([3, 4, 7, 8, 9], device="cuda")
    good = torch.ones(90, dtype=torch.bool, device="cuda")
    good[bad] = False
    leaf = x.detach().requires_grad_()
    loss = linear_cross_entropy(leaf, w, labels, b, reduction="none")
    assert bool(loss.detach()[bad].isnan().all()) and bool(loss.detach()[good].isfinite().all())
    dx, = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
    assert bool(dx[bad].isnan().all()) and bool(dx[good].isfinite().all())
    idx = labels[:, None].repeat(1, 2)
    idx[:, 1] = 3
    loss = distill_top_logits(x, w, idx, torch.zeros(90, 2, device="cuda"), b, reduction="none")
    assert bool(loss[torch.tensor([3, 4, 7, 9], device="cuda")].isnan().all()) and bool(loss[8].isfinite())        # -1: left out
    # a column that no row can have
    b = b.clone()
    b[11] = -float("inf")
    x, w, _, labels, g = inputs(90, 64, 200, dtype, seed=2)
    labels[labels == 11] = 12
    leaf, table = x.requires_grad_(), w.requires_grad_()
    loss = linear_cross_entropy(leaf, table, labels, b)
    dx, dw = torch.autograd.grad(loss, (leaf, table))
    assert bool(loss.isfinite()) and bool(dx.isfinite().all()) and bool((dw[11] == 0).all())


def test_large_and_small_gradients_of_rows():
    """fp16 holds G over the largest of the rows' g."""
    from spion_b200.vocab import linear_cross_entropy
    for dtype in TYPES:
        x, w, b, labels, g = inputs(64, 64, 100, dtype)
        x, w = x.requires_grad_(), w.requires_grad_()
        loss = linear_cross_entropy(x, w, labels, b, reduction="none")
        unit = torch.autograd.grad(loss, (x, w), torch.full((64,), 2.0 ** -4, device="cuda"), retain_graph=True)
        for power in (-10, 3):
            scaled = torch.autograd.grad(loss, (x, w), torch.full((64,), 2.0 ** (power - 4), device="cuda"), retain_graph=True)
            for p, q in zip(unit, scaled):
                if dtype != torch.float16:
                    assert torch.equal(p * 2.0 ** power, q)
        given = torch.ones(64, device="cuda")
        given[5] = float("inf")
        dx, dw = torch.autograd.grad(loss, (x, w), given, retain_graph=True)
        assert not bool(dx[5].isfinite().any()) and bool(dx[:5].isfinite().all()) and bool(dx[6:].isfinite().all())
        zero = torch.autograd.grad(loss, (x, w), torch.zeros(64, device="cuda"))
        assert all(bool((t == 0).all()) for t in zero)


def test_differences():
    """The gradient along a direction against differences of the loss in fp32."""
    from spion_b200.vocab import distill_top_logits, linear_cross_entropy
    x, w, b, labels, g = inputs(50, 40, 90, torch.float32)
    idx, teacher = torch.randint(0, 90, (50, 4), generator=g, device="cuda"), torch.randn(50, 4, generator=g, device="cuda")
    for f in (lambda x, w, b: linear_cross_entropy(x, w, labels, b, reduction="sum"), lambda x, w, b: distill_top_logits(x, w, idx, teacher, b, 1.5, "sum")):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        loss = f(*leaves)
        grads = torch.autograd.grad(loss, leaves)
        for i in range(3):
            d = torch.randn(leaves[i].shape, generator=g, device="cuda")
            d /= d.norm()
            e = 2.0 ** -4
            args = [[t.detach() + (s * e * d if j == i else 0) for j, t in enumerate(leaves)] for s in (1, -1, 0.5, -0.5)]
            a, c = ((f(*args[0]) - f(*args[1])) / (2 * e)).double(), ((f(*args[2]) - f(*args[3])) / e).double()
            want = (4 * c - a) / 3                         # error e^4; the losses (about 300) are known to 1e-6 of them, here over 2^-4
            assert abs(float(want - (grads[i] * d).sum())) < 300 * 1e-6 * 2 / e + 1e-3 * abs(float(want))


def test_only_some_gradients_and_twice():
    from spion_b200.vocab import linear_cross_entropy
    x, w, b, labels, g = inputs(100, 64, 300, torch.bfloat16)
    all_ = [t.detach().requires_grad_() for t in (x, w, b)]
    loss = linear_cross_entropy(*all_[:2], labels, all_[2])
    want = torch.autograd.grad(loss, all_, retain_graph=True)
    again = torch.autograd.grad(loss, all_)
    for i in range(3):
        assert torch.equal(want[i], again[i])
        some = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        only, = torch.autograd.grad(linear_cross_entropy(*some[:2], labels, some[2]), some[i])
        assert torch.equal(only, want[i])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, all_)
    with torch.no_grad():
        assert not linear_cross_entropy(*all_[:2], labels, all_[2]).requires_grad
    loss = linear_cross_entropy(*all_[:2], labels, all_[2])
    with torch.no_grad():
        all_[1].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


def test_a_recorded_backward():
    from spion_b200.vocab import distill_top_logits
    x, w, b, _, g = inputs(30, 24, 50, torch.float32)
    idx, teacher = torch.randint(-1, 50, (30, 3), generator=g, device="cuda"), torch.randn(30, 3, generator=g, device="cuda")
    leaves = [t.requires_grad_() for t in (x, w, b)]
    for reduction in ("mean", "none"):
        loss = distill_top_logits(*leaves[:2], idx, teacher, leaves[2], 1.5, reduction)
        given = torch.rand(loss.shape, generator=g, device="cuda")
        plain = torch.autograd.grad(loss, leaves, given, retain_graph=True)
        graph = torch.autograd.grad(loss, leaves, given, create_graph=True)
        for p, q in zip(plain, graph):
            torch.testing.assert_close(p, q, rtol=2e-5, atol=2e-6)
        assert all(torch.isfinite(t).all() for t in torch.autograd.grad(sum((t ** 2).sum() for t in graph), leaves))


def test_captured_replayed_and_on_two_streams():
    from spion_b200.vocab import linear_cross_entropy
    x, w, b, labels, g = inputs(300, 64, 700, torch.bfloat16)
    x2, w2, b2, labels2, _ = inputs(300, 64, 700, torch.bfloat16, seed=5)
    labels2[::3] = -100                                    # another number of rows that count

    def step(x, w, b, labels):
        loss = linear_cross_entropy(x, w, labels, b)
        return [loss.detach(), *torch.autograd.grad(loss, (x, w, b))]

    first, second = [[t.requires_grad_() for t in s] for s in ((x, w, b), (x2, w2, b2))]
    want, want2 = step(*first, labels), step(*second, labels2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    hold = [t.detach().clone().requires_grad_() for t in first]
    lab = labels.clone()
    with torch.cuda.stream(side):
        step(*hold, lab)
        graphs = []
        for _ in range(2):                                 # two graphs of the same call
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = step(*hold, lab)
            graphs.append((graph, out))
    torch.cuda.synchronize()
    for data, labels_, expect in ((second, labels2, want2), (first, labels, want)):
        with torch.no_grad():
            for h, t in zip(hold, data):
                h.copy_(t)
            lab.copy_(labels_)
        for graph, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, expect))
    other = torch.cuda.Stream()
    for _ in range(5):
        other.wait_stream(torch.cuda.current_stream())
        a = step(*first, labels)
        with torch.cuda.stream(other):
            c = step(*second, labels2)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(a, want)) and all(torch.equal(p, q) for p, q in zip(c, want2))


def test_a_first_backward_of_a_process():
    """On the autograd engine's thread, which has not used the device yet."""
    import os
    import subprocess
    import sys
    code = ("import torch\nfrom spion_b200.vocab import linear_cross_entropy\n"
            "x = torch.randn(200, 64, device='cuda', requires_grad=True)\nw = torch.randn(300, 64, device='cuda', requires_grad=True)\n"
            "l = torch.zeros(200, dtype=torch.long, device='cuda')\n"
            "g = torch.autograd.grad(linear_cross_entropy(x, w, l), (x, w), torch.tensor(1.0, device='cuda'))\n"
            "torch.cuda.synchronize()\nassert all(bool(t.isfinite().all()) for t in g)\nprint('done')\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, r.stderr[-2000:]


def test_a_first_call_under_a_capture():
    """The first use of the operators in a process, kernels not loaded yet."""
    import os
    import subprocess
    import sys
    code = ("import torch\nfrom spion_b200.vocab import linear_cross_entropy\nfrom spion_b200.tokens import embed_tokens\n"
            "ids = torch.arange(200, device='cuda') % 50\ntable = torch.randn(50, 64, device='cuda', requires_grad=True)\n"
            "w = torch.randn(300, 64, device='cuda', requires_grad=True)\none = torch.ones((), device='cuda')\n"
            "s = torch.cuda.Stream()\ns.wait_stream(torch.cuda.current_stream())\ng = torch.cuda.CUDAGraph()\n"
            "with torch.cuda.stream(s):\n  with torch.cuda.graph(g, stream=s):\n"
            "    loss = linear_cross_entropy(embed_tokens(ids, table), w, ids)\n    grads = torch.autograd.grad(loss, (table, w), one)\n"
            "torch.cuda.synchronize()\ng.replay()\ntorch.cuda.synchronize()\n"
            "want = torch.autograd.grad(linear_cross_entropy(embed_tokens(ids, table), w, ids), (table, w))\n"
            "assert all(torch.equal(a, b) for a, b in zip(grads, want))\nprint('done')\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, r.stderr[-2000:]


def test_autocast_and_the_module():
    from spion_b200.tokens import ScaledEmbedding
    from spion_b200.vocab import VocabHead, linear_cross_entropy
    table = ScaledEmbedding(300, 64).cuda()
    head = VocabHead(64, 300, tied=table).cuda()
    assert head.weight is table.weight
    x = torch.randn(50, 64, device="cuda")
    labels = torch.randint(0, 300, (50,), device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = head.loss(x, labels)
    want = linear_cross_entropy(x.bfloat16(), head.weight.bfloat16(), labels, head.bias)
    assert torch.equal(loss, want)
    loss.backward()
    assert table.weight.grad.dtype == torch.float32
    assert torch.equal(head.distill(x, labels[:, None], torch.zeros(50, 1, device="cuda")), head.loss(x, labels))


def test_refusals():
    from spion_b200._lib import SpionError
    from spion_b200.vocab import distill_top_logits, linear_cross_entropy
    x, w, b, labels, g = inputs(10, 16, 20, torch.float32)
    idx, t = labels[:, None].repeat(1, 2), torch.zeros(10, 2, device="cuda")
    for call in (lambda: linear_cross_entropy(x, w.bfloat16(), labels), lambda: linear_cross_entropy(x, w[:, :8], labels), lambda: linear_cross_entropy(x, w, labels[:9]),
                 lambda: linear_cross_entropy(x, w, labels.float()), lambda: linear_cross_entropy(x, w, labels.cpu()), lambda: linear_cross_entropy(x, w, labels, b[:3]),
                 lambda: linear_cross_entropy(x, w, labels, reduction="average"), lambda: linear_cross_entropy(x.double(), w.double(), labels),
                 lambda: linear_cross_entropy(x, w, labels, b.double()), lambda: distill_top_logits(x, w, idx, t[:, :1]), lambda: distill_top_logits(x, w, idx, t.double()),
                 lambda: distill_top_logits(x, w, idx, t, temperature=0.0), lambda: distill_top_logits(x, w, idx, t, temperature=float("inf")),
                 lambda: distill_top_logits(x, w, idx, t.requires_grad_()),
                 lambda: distill_top_logits(x, w, labels[:, None].repeat(1, 129), torch.zeros(10, 129, device="cuda"))):
        with pytest.raises(SpionError):
            call()


@pytest.mark.parametrize("T", [1, 2, 3, 8, 9, 15, 16, 17])
@pytest.mark.parametrize("K,V", [(1, 1048581), (7, 150001), (64, 20000), (130, 9001), (1276, 900), (1284, 1000), (2656, 427), (1030, 4099), (4100, 300), (40000, 31), (16, 70001), (17, 5003), (3, 40001)])
def test_few_rows_of_fp32_and_many_weights(T, K, V):
    """A sum over the contraction or the vocabulary takes K / 32 or V / 148 numbers one after another at most, each rounded to half a step: below the bounds of the accumulators."""
    x, w, b, labels, g = inputs(T, K, V, torch.float32, seed=5, bias=V != 900)
    labels[T // 2] = labels[0]
    labelled(x, w, b, labels, g, "none")


@pytest.mark.parametrize("T", [4, 16])
@pytest.mark.parametrize("k", [1, 5, 128])
def test_few_rows_of_fp32_and_a_teacher(T, k):
    from spion_b200.vocab import distill_top_logits
    V = 4099
    x, w, b, _, g = inputs(T, 300, V, torch.float32, seed=k)
    idx = torch.rand(T, V, generator=g, device="cuda").argsort(1)[:, :k].contiguous()
    teacher = 2 * torch.randn(T, k, generator=g, device="cuda")
    idx[1] = -1
    if k > 1:
        idx[0, 1] = idx[0, 0]
        idx[2, k // 2:] = -1
    rows = (idx >= 0).any(1).nonzero().squeeze(1)
    q = torch.softmax(torch.where(idx >= 0, teacher.double() / 2, -float("inf"))[rows], 1)
    check(lambda x, w, b: distill_top_logits(x, w, idx, teacher, b, 2.0, "sum"), x, w, b, rows, idx[rows].clamp_min(0), q, 2.0, "sum", g)


@pytest.mark.parametrize("T", [5, 12])
def test_few_rows_of_fp32_strides_masks_and_what_is_not_finite(T):
    from spion_b200.vocab import linear_cross_entropy
    x, w, b, labels, g = inputs(T, 204, 11000, torch.float32, seed=9)
    labels[1::3] = -100
    labels[2] = -100

    def grads(x, w, b, labels, reduction="mean"):
        x, w, b = (t.detach().requires_grad_() for t in (x, w, b))
        loss = linear_cross_entropy(x, w, labels, b, reduction=reduction)
        return [loss.detach(), *torch.autograd.grad(loss, (x, w, b))]

    for a in ((x[:, 1:201], w[:, 1:201]), (x[:, :200], w[:, 4:204]), (x[:1, :200].expand(T, 200), w[::2, :200])):
        labelled(*a, b[:a[1].shape[0]], torch.where(labels < 0, labels, labels % a[1].shape[0]), g)
    want = grads(x, w, b, labels)
    bad = x.clone()
    bad[1] = float("nan")                                  # a row that does not count
    for a, e in zip(grads(bad, w, b, labels), want):
        assert torch.equal(a, e)
    assert bool((want[1][1] == 0).all())
    bad[0, 3] = float("inf")                               # one that does
    got = grads(bad, w, b, labels)
    assert bool(got[0].isnan()) and bool(got[1][0].isnan().all()) and bool(got[1][3].isfinite().all()) and bool((got[1][1] == 0).all())
    masked = b.clone()
    masked[10000:] = -float("inf")                         # entries that no row can have: as if they were not there (their exponentials are zeros)
    inside = torch.where(labels < 0, labels, labels % 10000)
    loss, dx, dw, db = grads(x, w, masked, inside)
    assert bool((dw[10000:] == 0).all()) and bool((db[10000:] == 0).all()) and bool(dx.isfinite().all())
    labelled(x, w[:10000], b[:10000], inside, g)
    close(loss, *(t.double() for t in (grads(x, w[:10000], b[:10000], inside)[0], torch.tensor(2.0 ** -18))), "masked entries")
    outside = labels.clone()
    outside[0] = 11000
    assert bool(grads(x, w, b, outside)[0].isnan())
    outside[:] = -100                                      # no row counts
    loss, dx, dw, db = grads(x, w, b, outside, "sum")
    assert bool(loss == 0) and not any(bool(t.any()) for t in (dx, dw, db))
    assert bool(grads(x, w, b, outside)[0].isnan())


def test_few_rows_of_fp32_some_gradients_and_a_captured_call():
    from spion_b200.vocab import linear_cross_entropy
    x, w, b, labels, g = inputs(6, 256, 5000, torch.float32, seed=4)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(linear_cross_entropy(leaves[0], leaves[1], labels, leaves[2]), leaves)
    for i, t in enumerate((x, w, b)):
        one = [x, w, b]
        one[i] = t.detach().requires_grad_()
        got, = torch.autograd.grad(linear_cross_entropy(one[0], one[1], labels, one[2]), one[i])
        assert torch.equal(got, want[i])
    del leaves, one
    stream = torch.cuda.Stream()
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    with torch.cuda.stream(stream):
        for _ in range(2):
            torch.autograd.grad(linear_cross_entropy(leaves[0], leaves[1], labels, leaves[2]), leaves)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = torch.autograd.grad(linear_cross_entropy(leaves[0], leaves[1], labels, leaves[2]), leaves)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for a, e in zip(got, want):
        assert torch.equal(a, e)
    with torch.no_grad():
        x2 = torch.randn_like(x)
        leaves[0].copy_(x2)
    graph.replay()
    torch.cuda.synchronize()
    fresh = [t.detach().requires_grad_() for t in (x2, w, b)]
    for a, e in zip(got, torch.autograd.grad(linear_cross_entropy(fresh[0], fresh[1], labels, fresh[2]), fresh)):
        assert torch.equal(a, e)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,K,V", [(1, 64, 200), (5, 64, 200), (150, 64, 200), (3, 400, 200), (1, 64, 20000)])
def test_rows_that_are_sure_of_their_target(T, K, V, dtype):
    """Large logits, and losses far below 1: 1 - p and -ln p keep the accuracy of what is left.  Of a row's sum, 1 and little more, each of fewer than 40 additions and the logarithm
    round by U at most (16 of a thread's numbers, 3 of its four sums, 16 of the parts, 5 over lanes): 48 U; the others' exponentials bring twice a logit's error."""
    from spion_b200.vocab import distill_top_logits, linear_cross_entropy
    x, w, _, _, g = inputs(T, K, V, dtype, seed=11, size=0.2)
    b = torch.full((V,), 300.0, device="cuda")
    b[3] = 300 + 7 + math.log(V)
    labels = torch.full((T,), 3, device="cuda")
    leaf = b.detach().requires_grad_()
    loss = linear_cross_entropy(x, w, labels, leaf, reduction="none")
    db, = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
    z = x.double() @ w.double().t() + b.double()
    S = x.double().abs() @ w.double().abs().t() + b.double()
    steps = (6 if dtype == torch.float32 else 1) * (-(-K // 64)) * 4
    delta = (S * U * (2 * min(steps, 64) + steps / 64 + 24)).amax(1)
    others = torch.logsumexp(z[:, torch.arange(V, device="cuda") != 3], 1)
    want = torch.log1p(torch.exp(others - z[:, 3]))
    bound = 2 * delta * want + 48 * U
    assert float(want.max()) < 2e-3
    close(loss.detach(), want, bound, "loss")
    close(db[3], torch.expm1(-want).sum(), bound.sum() + 2 * T * U * float(want.max()), "db")
    two = torch.tensor([[3, -1]], device="cuda").expand(T, 2).contiguous()
    close(distill_top_logits(x, w, two, torch.zeros(T, 2, device="cuda"), b, reduction="none"), want, bound, "one entry of two")
