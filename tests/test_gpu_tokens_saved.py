"""Rows of a token table whose ids, saved for the gradient, come back as another tensor (offloading, hooks, recomputed segments)."""
import pytest
import torch

from spion_b200._lib import SpionError

pytestmark = pytest.mark.gpu


def gradient(ids, w, dy, back=None):
    from spion_b200.tokens import embed_tokens
    w = w.detach().requires_grad_()
    if back == "cpu":
        with torch.autograd.graph.save_on_cpu():
            y = embed_tokens(ids, w, 0.5, 3)
    else:
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), back or (lambda t: t)):
            y = embed_tokens(ids, w, 0.5, 3)
    return torch.autograd.grad(y, w, dy)[0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1,), (7, 33), (4, 5000)])
def test_ids_that_come_back_spread_out(dtype, shape):
    g = torch.Generator(device="cuda").manual_seed(1)
    ids, w = torch.randint(0, 500, shape, generator=g, device="cuda"), torch.randn(500, 40, generator=g, device="cuda").to(dtype)
    dy = torch.randn(*shape, 40, generator=g, device="cuda").to(dtype)
    want = gradient(ids, w, dy)

    def spread(t):
        out = torch.full((*t.shape, 2), 499, dtype=t.dtype, device=t.device)
        out[..., 1] = t
        return out[..., 1]

    def turned(t):
        return t.mT.contiguous().mT if t.dim() > 1 else t.clone()

    for back in ("cpu", spread, turned):
        assert torch.equal(gradient(ids, w, dy, back), want)


def test_recomputed_lookups():
    from torch.utils.checkpoint import checkpoint

    from spion_b200.tokens import embed_tokens
    ids, w = torch.randint(0, 90, (6, 50), device="cuda"), torch.randn(90, 24, device="cuda", requires_grad=True)

    def f(w):
        return embed_tokens(ids, w).tanh().sum(0)

    dy = torch.randn(50, 24, device="cuda")
    assert torch.equal(torch.autograd.grad(checkpoint(f, w, use_reentrant=False), w, dy)[0], torch.autograd.grad(f(w), w, dy)[0])


@pytest.mark.parametrize("change", [lambda t: t.int(), lambda t: t[:-1], lambda t: t.cpu()])
def test_what_a_hook_must_not_change(change):
    ids, w, dy = torch.randint(0, 90, (50,), device="cuda"), torch.randn(90, 24, device="cuda"), torch.randn(50, 24, device="cuda")
    with pytest.raises(SpionError, match="hook"):
        gradient(ids, w, dy, change)
