"""Hooks and wrappers of the last layer, whose losses call no forward of it."""
import pytest
import torch
from torch import nn

from spion_b200._lib import SpionError
from spion_b200.vocab import VocabHead


def both(head, x, labels):
    return (lambda: head.loss(x, labels), lambda: head.distill(x, labels[:, None], torch.zeros(len(labels), 1, device=x.device)))


def calls_on_cpu(head):
    return both(head, torch.randn(3, 8), torch.zeros(3, dtype=torch.long))


@pytest.mark.parametrize("hook", [lambda m: m.register_forward_pre_hook(lambda m, a: None), lambda m: m.register_forward_hook(lambda m, a, y: None),
                                  lambda m: m.register_full_backward_hook(lambda m, a, y: None), lambda m: m.register_full_backward_pre_hook(lambda m, y: None),
                                  lambda m: nn.utils.weight_norm(m), lambda m: nn.utils.spectral_norm(m),
                                  lambda m: nn.utils.prune.l1_unstructured(m, "weight", amount=0.5), lambda m: setattr(m, "forward", lambda x: x)])
@pytest.mark.filterwarnings("ignore")
def test_a_layer_with_hooks_has_no_loss(hook):
    import torch.nn.utils.prune  # noqa: F401
    head = VocabHead(8, 10)
    removable = hook(head)
    for call in calls_on_cpu(head):
        with pytest.raises(SpionError, match="forward"):
            call()
    if hasattr(removable, "remove"):
        removable.remove()
        for call in calls_on_cpu(head):
            with pytest.raises(SpionError, match="CUDA"):      # what a layer without hooks says here
                call()


def test_a_class_with_a_forward_of_its_own_has_no_loss():
    class Scaled(VocabHead):
        def forward(self, x):
            return 2 * super().forward(x)

    class Named(VocabHead):
        pass

    for call in calls_on_cpu(Scaled(8, 10)):
        with pytest.raises(SpionError, match="forward"):
            call()
    for head in (Named(8, 10), nn.utils.parametrizations.weight_norm(Named(8, 10))):
        for call in calls_on_cpu(head):
            with pytest.raises(SpionError, match="CUDA"):
                call()


@pytest.mark.gpu
def test_weights_that_are_formed_by_parametrisations_are_served():
    """These change the attribute, not the forward."""
    head = nn.utils.parametrizations.weight_norm(VocabHead(16, 50).cuda())
    x, labels = torch.randn(20, 16, device="cuda"), torch.randint(0, 50, (20,), device="cuda")
    with torch.no_grad():
        head.parametrizations.weight.original0.mul_(2)
    want = nn.functional.cross_entropy(head(x).double(), labels)
    loss = head.loss(x, labels)
    assert abs(float(loss.detach()) - float(want)) <= 1e-5 * float(want)
    loss.backward()
    assert all(bool(p.grad.isfinite().all()) for p in head.parameters())
