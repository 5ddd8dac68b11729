"""Rows of several targets a row of which one has all the weight: 1 - p keeps the accuracy of what the other entries leave, as where there is one target only.

Bounds as of single targets (u = 2^-24): z and the log of the sum are some thousand here and rounded to u of that, which a difference of p and 1 would carry.  From the loss, 48 u for the sum
and its logarithm, and twice a logit's error times what is left."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,K,V", [(1, 64, 200), (5, 64, 200), (3, 400, 200), (1, 64, 20000), (12, 64, 20000), (1, 16, 9)])
@pytest.mark.parametrize("targets,logits", [([3, -1], [0.0, 0.0]), ([5, 3], [-200.0, 0.0]), ([-1, 5, 3, 6], [3.0, -1e30, 1.0, -float("inf")])])
def test_one_target_that_has_all_the_weight(T, K, V, dtype, targets, logits):
    from spion_b200.vocab import distill_top_logits, linear_cross_entropy
    g = torch.Generator(device="cuda").manual_seed(T + K + V)
    x = torch.randn(T, K, generator=g, device="cuda").to(dtype)
    w = (torch.randn(V, K, generator=g, device="cuda") * (0.2 / math.sqrt(K))).to(dtype)
    b = torch.full((V,), 3000.0, device="cuda")
    b[3] = 3007 + math.log(V)
    z = x.double() @ w.double().t() + b.double()
    S = x.double().abs() @ w.double().abs().t() + b.double()
    steps = (6 if dtype == torch.float32 else 1) * (-(-K // 64)) * 4
    delta = (S * U * (2 * min(steps, 64) + steps / 64 + 24)).amax(1)
    left = torch.log1p(torch.exp(torch.logsumexp(z[:, torch.arange(V, device="cuda") != 3], 1) - z[:, 3]))
    assert float(left.max()) < 2e-3
    want, bound = torch.expm1(-left), 2 * delta * left + 48 * U + 2 * U * left
    idx = torch.tensor(targets, device="cuda").expand(T, -1).contiguous()
    teacher = torch.tensor(logits, device="cuda").expand(T, -1).contiguous()
    for row in range(T):
        one = torch.zeros(T, device="cuda")
        one[row] = 1.0
        got = []
        for call in (lambda leaf: distill_top_logits(x, w, idx, teacher, leaf, reduction="none"),
                     lambda leaf: linear_cross_entropy(x, w, torch.full((T,), 3, device="cuda"), leaf, reduction="none")):
            leaf = b.detach().requires_grad_()
            loss = call(leaf)
            db, = torch.autograd.grad(loss, leaf, one)
            assert bool(((loss.detach().double() - left).abs() <= bound).all())
            assert abs(float(db[3]) - float(want[row])) <= float(bound[row]), (row, float(db[3]), float(want[row]))
            got.append((loss.detach(), db))
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_weights_that_are_shared_out():
    """Two targets with half of it each, one id twice, and an id that has all of it and none."""
    from spion_b200.vocab import distill_top_logits
    g = torch.Generator(device="cuda").manual_seed(4)
    x, w = torch.randn(3, 16, generator=g, device="cuda"), torch.randn(50, 16, generator=g, device="cuda") / 4
    idx = torch.tensor([[7, 9], [7, 7], [7, 7]], device="cuda")
    teacher = torch.tensor([[1.0, 1.0], [1.0, 1.0], [1.0, -300.0]], device="cuda")
    leaf = torch.zeros(50, device="cuda", requires_grad=True)
    for row in range(3):
        one = torch.zeros(3, device="cuda")
        one[row] = 1.0
        db, = torch.autograd.grad(distill_top_logits(x, w, idx, teacher, leaf, reduction="none"), leaf, one)
        want = torch.softmax((x[row].double() @ w.double().t()), 0)
        want[7] -= 0.5 if row == 0 else 1.0
        want[9] -= 0.5 if row == 0 else 0.0
        assert bool(((db.double() - want).abs() <= 200 * U).all())      # p to 2 of a logit's 70 u, as in test_sizes
