"""Tables, rows and gradients of more than 2^31 elements: the same as the small part of them that matters, wherever it lies."""
import pytest
import torch

pytestmark = pytest.mark.gpu

FAR, K = 530000, 4096                                      # 2.17e9 elements


def near(got, want, size=None):
    """Two roundings to bf16 of numbers that differ in the last bits of fp32: a step apart at most.  size, of gradients of a loss: the magnitudes that are added up.  Tiles of another kind add
    a logit up in another order; where that moves an entry of the logits' gradient across a tie it comes out a step, 2^-8 of it, apart: 2^-8 of size at most, if all of them do."""
    got, want = got.double(), want.double()
    return bool(((got - want).abs() <= want.abs() * 2.0 ** -7 + (1e-5 * float(want.abs().max()) if size is None else 2.0 ** -8 * size)).all())


def sizes(x, w, labels, given):
    """Sums of magnitudes of dx and dw; given: what arrives at each row."""
    x, w = x.detach().double(), w.detach().double()
    G = torch.softmax(x @ w.t(), 1)
    G[torch.arange(len(x), device="cuda"), labels] -= 1
    G = (G * given.double()[:, None]).abs()
    return G @ w.abs(), G.t() @ x.abs()


def only(grad, rows):
    """Nothing but zeros outside of `rows` (of the first dimension)."""
    return all(not bool(part.any()) for part in (grad[:rows.start], grad[rows.stop:]))


def test_a_table_of_rows():
    from spion_b200.tokens import embed_tokens
    w = torch.zeros(FAR, K, device="cuda", dtype=torch.bfloat16)
    last = slice(FAR - 50, FAR)
    w[last] = torch.randn(50, K, device="cuda").bfloat16()
    w.requires_grad_()
    ids = torch.randint(FAR - 50, FAR, (300,), device="cuda")
    y = embed_tokens(ids, w, 2.0)
    small = w.detach()[last].clone().requires_grad_()
    want = embed_tokens(ids - (FAR - 50), small, 2.0)
    dy = torch.randn(300, K, device="cuda").bfloat16()
    dw, = torch.autograd.grad(y, w, dy)
    assert torch.equal(y, want) and torch.equal(dw[last], torch.autograd.grad(want, small, dy)[0]) and only(dw, last)


def test_many_rows_looked_up():
    from spion_b200.tokens import embed_tokens
    w = torch.randn(100, K, device="cuda").bfloat16().requires_grad_()
    ids = torch.full((FAR,), -1, device="cuda")
    ids[-300:] = torch.randint(0, 100, (300,), device="cuda")
    y = embed_tokens(ids, w, 2.0)
    small = w.detach().clone().requires_grad_()
    want = embed_tokens(ids[-300:], small, 2.0)
    assert torch.equal(y.detach()[-300:], want.detach()) and bool(y.detach()[:-300:1000].isnan().all())
    dy = torch.randn_like(y)
    dw, = torch.autograd.grad(y, w, dy)
    assert near(dw, torch.autograd.grad(want, small, dy[-300:])[0])


@pytest.mark.parametrize("T", [40, 700])
def test_a_large_vocabulary(T):
    from spion_b200.vocab import linear_cross_entropy
    w, b = torch.zeros(FAR, K, device="cuda", dtype=torch.bfloat16), torch.full((FAR,), -float("inf"), device="cuda")
    last = slice(FAR - 500, FAR)
    w[last], b[last] = (torch.randn(500, K, device="cuda") / 64).bfloat16(), 0.0
    x, labels = torch.randn(T, K, device="cuda").bfloat16(), torch.randint(0, 500, (T,), device="cuda")
    leaves = [t.requires_grad_() for t in (x, w)]
    loss = linear_cross_entropy(*leaves, labels + (FAR - 500), b)
    dx, dw = torch.autograd.grad(loss, leaves)
    small = [x.detach().requires_grad_(), w.detach()[last].clone().requires_grad_()]
    want = linear_cross_entropy(*small, labels, torch.zeros(500, device="cuda"))
    assert abs(float(loss.detach() - want.detach())) <= 1e-5 * float(want.detach())
    for p, q, size in zip((dx, dw[last]), torch.autograd.grad(want, small), sizes(*small, labels, torch.full((T,), 1.0 / T, device="cuda"))):
        assert near(p, q, size)
    assert only(dw, last)


@pytest.mark.parametrize("counted", ["some", "all"])
def test_many_rows(counted):
    from spion_b200.vocab import linear_cross_entropy
    x, w = torch.randn(FAR, K, device="cuda", dtype=torch.bfloat16), (torch.randn(200, K, device="cuda") / 64).bfloat16()
    labels = torch.randint(0, 200, (FAR,), device="cuda")
    last = slice(FAR - 300, FAR)
    given = torch.zeros(FAR, device="cuda")
    given[last] = torch.randn(300, device="cuda")
    if counted == "some":
        labels[:FAR - 300] = -100
    leaves = [t.requires_grad_() for t in (x, w)]
    loss = linear_cross_entropy(*leaves, labels, reduction="none")
    dx, dw = torch.autograd.grad(loss, leaves, given)
    small = [x.detach()[last].clone().requires_grad_(), w.detach().requires_grad_()]
    want = linear_cross_entropy(*small, labels[last], reduction="none")
    assert bool(((loss.detach()[last] - want.detach()).abs() <= 1e-5 * want.detach().abs()).all())
    assert bool(loss.detach().isfinite().all()) and (counted == "all" or only(loss.detach(), last))
    for p, q, size in zip((dx[last], dw), torch.autograd.grad(want, small, given[last]), sizes(*small, labels[last], given[last])):
        assert near(p, q, size)
    assert only(dx, last)
