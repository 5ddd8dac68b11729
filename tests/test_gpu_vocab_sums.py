"""How far the sums of the losses over a vocabulary are truncated in the tensor cores.

u = 2^-24.  A step there (16 products) loses 2 u of the sum at most, u in the mean of many, and always towards zero: over an accumulator of n steps 2 n u, n u in the mean.  16-bit operands: 16
steps an accumulator where tiles are small, 64 where pairs of CTAs share large ones.  fp32 operands are three parts and six products; the five small ones of an accumulator go first, 2^-7 of its sum
or less, so 8 of its 48 steps count, and the others no more than a ninth.  The accumulators are added in fp32, each addition rounded to u / 2 at most."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,K,V", [(3, 1024, 2), (40, 1000, 5), (200, 4096, 3), (200, 1024, 40000), (3, 1024, 50000), (300, 64, 700)])
def test_logits(T, K, V, dtype):
    """One entry has a logit of 30 to 40 (a sum of positive products), the others none: its distance to another entry, the label, is the loss."""
    from spion_b200.vocab import linear_cross_entropy
    g = torch.Generator(device="cuda").manual_seed(K + V)
    x = (torch.rand(T, K, generator=g, device="cuda") + 0.5).to(dtype)
    w = torch.zeros(V, K, device="cuda")
    w[0] = (torch.rand(K, generator=g, device="cuda") + 0.5) * (34.0 / K)
    w = w.to(dtype)
    z = (x.double() @ w[:1].double().t()).squeeze(1)
    want = torch.logaddexp(z, torch.log(torch.tensor(float(V - 1), dtype=torch.float64, device="cuda")))
    loss = linear_cross_entropy(x, w, torch.ones(T, dtype=torch.long, device="cuda"), reduction="none")
    wide = dtype == torch.float32
    few = wide and T <= 16 and V * K >= 65536               # ordinary units: rounded to nearest, K / 32 additions of a lane
    steps = 9 if wide else 64 if V == 40000 else 16
    accumulators = -(-K // 16) * (6 if wide else 1) / (48 if wide else steps)
    # ... and the logit in units of log2, its distances, their sum's logarithm and the loss: six roundings
    bound = (K / 32 + 8) * U if few else (2 * steps + accumulators / 2 + 6) * U
    off = ((loss.double() - want).abs() / want).max()
    assert float(off) <= bound, (float(off) / U, bound / U)


@pytest.mark.parametrize("T,K,V", [(529, 16, 4), (11175, 121, 21), (32489, 288, 10), (43963, 400, 64)])
def test_gradients_of_fp32(T, K, V):
    """Of the norm: 9 u for the truncations; the additions of N accumulators whose signs are at random, u / 2 of sums that grow as the root of their number, together at most the root of N / 2
    times u / 2; 4 u for G (an exponential to two steps of its last place, a difference, a product) and the result."""
    from spion_b200.vocab import linear_cross_entropy
    g = torch.Generator(device="cuda").manual_seed(T)
    w = torch.randn(V, K, generator=g, device="cuda") * (2.0 / K ** 0.5)
    labels = torch.randint(0, V, (T,), generator=g, device="cuda")
    x = torch.randn(T, K, generator=g, device="cuda") + torch.rand(T, 1, generator=g, device="cuda") * w[labels]
    got, want = [], []
    for out, dtype in ((got, torch.float32), (want, torch.float64)):
        leaves = [t.to(dtype).requires_grad_() for t in (x, w)]
        loss = linear_cross_entropy(*leaves, labels) if dtype == torch.float32 else torch.nn.functional.cross_entropy(leaves[0] @ leaves[1].t(), labels)
        out += torch.autograd.grad(loss, leaves)
    for p, q, length in zip(got, want, (V, T)):
        bound = (9 + (length / 128 / 2) ** 0.5 / 2 + 4) * U
        off = float((p.double() - q).norm() / q.norm())
        assert off <= bound, (off / U, bound / U)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,K,V", [(1, 64, 50), (1, 1304, 4), (2, 32, 9704), (6, 29, 2760), (11, 2, 63111), (40, 256, 30000), (64, 128, 20000), (300, 16, 5)])
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_gradients_of_few_rows_are_rounded_once(T, K, V, dtype, reduction):
    """A row's gradient hangs on its target's entry of G, whose rounding to 16 bits would be the whole row's: up to twice the result's own.  With twice the bits, 2^-16 or less of an entry, the
    result is as far off as its own rounding makes it; next to a tie that may be the other way, of no more than a part 2^-16 / (half a step) of the numbers: a tenth covers it."""
    from spion_b200.vocab import linear_cross_entropy
    for seed in range(8):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x = torch.randn(T, K, generator=g, device="cuda").to(dtype).requires_grad_()
        w = (torch.randn(V, K, generator=g, device="cuda") / K ** 0.5).to(dtype).requires_grad_()
        b = torch.zeros(V, device="cuda")
        b[0] = torch.log(torch.tensor(float(V))) + torch.randn((), generator=g, device="cuda")      # a likely entry, and the label: its probability is a half or so
        labels = torch.zeros(T, dtype=torch.long, device="cuda")
        given = torch.randn(T, generator=g, device="cuda") if reduction == "none" else torch.ones((), device="cuda")
        got = torch.autograd.grad(linear_cross_entropy(x, w, labels, b, reduction=reduction), (x, w), given)
        a, c = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
        want = torch.autograd.grad(torch.nn.functional.cross_entropy(a @ c.t() + b.double(), labels, reduction=reduction), (a, c), given.double())
        for p, q in zip(got, want):
            own = float((q.to(dtype).double() - q).norm())
            assert float((p.double() - q).norm()) <= 1.1 * own + 2.0 ** -15 * float(q.norm()), (seed, float((p.double() - q).norm()) / own)
