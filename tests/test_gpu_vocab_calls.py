"""Calls of the operators at a model's two ends that other tests do not make: traced, mapped and with tangents (refused), recorded backward passes of the cross entropy, gradients of rows
that are far apart, captured training steps."""
import pytest
import torch

from spion_b200._lib import SpionError
from test_gpu_harness_tokens import start, trainer
from test_gpu_vocab import close, inputs, oracle

pytestmark = pytest.mark.gpu


def operands():
    x, w, b, labels, g = inputs(12, 16, 30, torch.float32)
    return x, w, b, labels, labels[:, None].repeat(1, 2), torch.zeros(12, 2, device="cuda")


def calls():
    from spion_b200.tokens import embed_tokens
    from spion_b200.vocab import distill_top_logits, linear_cross_entropy
    x, w, b, labels, idx, t = operands()
    return {"embed": (lambda w: embed_tokens(labels, w), w), "loss_x": (lambda x: linear_cross_entropy(x, w, labels, b), x), "loss_w": (lambda w: linear_cross_entropy(x, w, labels, b), w),
            "loss_b": (lambda b: linear_cross_entropy(x, w, labels, b), b), "distill_x": (lambda x: distill_top_logits(x, w, idx, t, b), x),
            "distill_t": (lambda t: distill_top_logits(x, w, idx, t, b), t)}


@pytest.mark.parametrize("name", ["embed", "loss_x", "loss_w", "loss_b", "distill_x", "distill_t"])
@pytest.mark.filterwarnings("ignore")
def test_what_would_not_be_seen_is_refused(name):
    """Tracers, function transforms, tangents and modes without real tensors."""
    import torch.autograd.forward_ad as fwad
    from torch._subclasses.fake_tensor import FakeTensorMode
    call, arg = calls()[name]
    want = call(arg)
    with pytest.raises(SpionError):
        torch.jit.trace(call, (arg,))
    with pytest.raises(SpionError):
        torch.func.vmap(call)(torch.stack([arg, arg]))
    with pytest.raises(SpionError):
        torch.func.grad(lambda a: call(a).sum())(arg)
    with fwad.dual_level():
        with pytest.raises(SpionError):
            call(fwad.make_dual(arg, torch.ones_like(arg)))
    with FakeTensorMode(allow_non_fake_inputs=True):
        with pytest.raises(SpionError):
            call(arg)
    assert torch.equal(call(arg), want)


def test_ids_and_labels_of_a_map_are_refused():
    from spion_b200.tokens import embed_tokens
    from spion_b200.vocab import linear_cross_entropy
    x, w, b, labels, _, _ = operands()
    for call in (lambda i: embed_tokens(i, w), lambda i: linear_cross_entropy(x, w, i, b)):
        with pytest.raises(SpionError):
            torch.func.vmap(call)(torch.stack([labels, labels]))


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_a_recorded_backward_of_the_cross_entropy(reduction):
    """Its gradients and theirs against torch's in fp64: sums of 24 to 50 numbers, 1e-5 of the largest."""
    from spion_b200.vocab import linear_cross_entropy
    x, w, b, labels, g = inputs(30, 24, 50, torch.float32)
    labels[::4] = -100
    given = torch.rand((30,) if reduction == "none" else (), generator=g, device="cuda")
    got = []
    for own in (True, False):
        leaves = [(t if own else t.double()).detach().requires_grad_() for t in (x, w, b)]
        if own:
            loss = linear_cross_entropy(*leaves[:2], labels, leaves[2], reduction=reduction)
        else:
            loss = torch.nn.functional.cross_entropy(leaves[0] @ leaves[1].t() + leaves[2], labels, reduction=reduction)
        first = torch.autograd.grad(loss, leaves, given.to(loss.dtype), create_graph=True)
        second = torch.autograd.grad(sum((t ** 2).sum() for t in first), leaves)
        got.append([loss.detach(), *(t.detach() for t in first), *second])
    for p, q in zip(*got):
        assert float((p.double() - q).abs().max()) <= 1e-5 * float(q.abs().max())


@pytest.mark.parametrize("V", [100, 3000])
def test_gradients_of_rows_that_are_far_apart(V):
    """fp16 holds G in units of 2^-13 of the largest |g|, its smallest step 2^-24 of that: an entry p of a row whose g is a part r of the largest keeps all its bits while p r >= 2^-26.
    Here from 1 down to 2^-16; every row within its own bound, without what underflows where nothing does."""
    from spion_b200.vocab import linear_cross_entropy
    x, w, b, labels, g = inputs(64, 64, V, torch.float16, size=1.0)
    ratio = 2.0 ** -(torch.arange(64, device="cuda") / 4.0)
    given = ratio * 512 * torch.where(torch.rand(64, generator=g, device="cuda") < 0.5, -1, 1)
    given = given[torch.randperm(64, generator=g, device="cuda")]
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(linear_cross_entropy(*leaves[:2], labels, leaves[2], reduction="none"), leaves, given)
    rows = torch.arange(64, device="cuda")
    q = torch.ones(64, 1, dtype=torch.float64, device="cuda")
    o = oracle(x, w, b, rows, labels[:, None], q, given.double(), 1.0)
    for name, got in zip(("dx", "dw", "db"), grads):
        close(got, *o[name], name)
    # rows one by one: the bound that is not in proportion to the largest g
    p = torch.softmax(x.double() @ w.double().t() + b.double(), 1)
    whole = p.amin(1) * given.abs().double() / 512 >= 2.0 ** -26
    assert 20 < int(whole.sum()) < 64 or V == 100
    some = whole.nonzero().squeeze(1)
    for row in some.tolist():
        one = oracle(x, w, b, rows[row:row + 1], labels[row:row + 1, None], q[:1], given[row:row + 1].double(), 1.0)
        want, bound = one["dx"]
        floor = 2.0 ** -25 / 8192 * 2 * float(given[row].abs()) * w.double().abs().sum(0)
        close(grads[0][row], want[0], bound[0] - floor, "dx of one row")


def test_a_common_factor_of_the_gradients_in_fp16():
    """A power of two comes back as it is; where a result is below the normal numbers of fp16, to half a step of theirs on either side."""
    from spion_b200.vocab import linear_cross_entropy
    x, w, b, labels, g = inputs(64, 64, 100, torch.float16)
    x, w = x.requires_grad_(), w.requires_grad_()
    loss = linear_cross_entropy(x, w, labels, b, reduction="none")
    unit = torch.autograd.grad(loss, (x, w), torch.ones(64, device="cuda"), retain_graph=True)
    for power in (-10, -3, 4):
        scaled = torch.autograd.grad(loss, (x, w), torch.full((64,), 2.0 ** power, device="cuda"), retain_graph=True)
        for p, q in zip(unit, scaled):
            p, q = p.double() * 2.0 ** power, q.double()
            # (the least normal number itself can be a smaller one that was rounded up, in steps of 2^-24)
            normal = (p.abs() > 2.0 ** (power - 14)) & (q.abs() > 2.0 ** -14)
            assert torch.equal(p[normal], q[normal])
            assert bool(((p - q).abs() <= 2.0 ** -25 * (1 + 2.0 ** power)).all())


@pytest.mark.parametrize("dtype,optimizer", [("fp32", "torch"), ("bf16", "fused")])
@pytest.mark.parametrize("tied", [False, True])
def test_a_captured_step_leaves_the_eager_ones_gradients_and_parameters(dtype, optimizer, tied):
    """Bit for bit: every kernel of the step sums in a fixed order."""
    runs = []
    for captured in (False, True):
        tr, ids, labels, _ = trainer("text" if dtype == "bf16" else "image", dtype, optimizer=optimizer, tied_weights=tied)
        start(tr, ids, labels)
        if captured:
            tr.capture_sparse_step(ids, labels, warmup=2)
        losses = [(tr.step_graph(ids, labels) if captured else tr.step(ids, labels)[0]).clone() for _ in range(2 if captured else 4)][-2:]
        tr.check_device_status()
        runs.append((losses, tr.bucket.flat.clone(), {n: p.detach().clone() for n, p in tr.model.named_parameters()}))
    (la, ga, pa), (lb, gb, pb) = runs
    assert all(torch.equal(a, b) for a, b in zip(la, lb)) and torch.equal(ga, gb)
    assert bool(ga.isfinite().all()) and float(ga.abs().max()) > 0
    for n in pa:
        assert torch.equal(pa[n], pb[n]), n
