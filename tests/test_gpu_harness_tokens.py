"""The operators at a model's two ends together, as a training run uses them: table rows in, a loss over the vocabulary or against a teacher out, eager and captured."""
import numpy as np
import pytest
import torch

from spion_b200 import synthetic

pytestmark = pytest.mark.gpu


def trainer(task="image", dtype="fp32", L=256, batch=4, vocab=700, **overrides):
    from spion_b200 import harness
    cfg = harness.task_config(task, batch, native=True, dtype=dtype)
    cfg.update(max_seq_len=L, dropout_prob=0.0, attention_dropout=0.0, threshold=0.85, vocab_size=vocab, objective="tokens", embedding="table", embedding_scale=8.0)
    cfg.update(overrides)
    tr = harness.Trainer(cfg, lr=1e-3, seed=3)
    g = torch.Generator(device="cuda").manual_seed(7)
    ids = torch.randint(1, vocab, (batch, L), generator=g, device="cuda")
    ids[0, L // 2:] = 0
    labels = torch.where(torch.rand(batch, L, generator=g, device="cuda") < 0.15, ids, -100)
    labels[ids == 0] = -100
    return tr, ids, labels, g


def start(tr, ids, lab):
    _, maps = tr.step(ids, lab, is_attn=True)
    tr.discover(maps)


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_the_losss_gradients_are_torchs(tied, dtype):
    """On the encoder's own output: 1e-5 of the norm in fp32 (sums of a few hundred numbers to 2^-24 each, a probability's exponential to 2^-20), 2^-6 in bf16 (operands, G and
    results rounded to 2^-8 each)."""
    tr, ids, labels, _ = trainer("text" if dtype == "bf16" else "image", dtype, tied_weights=tied)
    start(tr, ids, labels)
    model = tr.model
    assert (model.head.weight is model.model.embeddings.tok.weight) == tied
    with torch.no_grad():
        t = model.scores(ids, tr.mat_lst).float()
    got, want = [], []
    for out, own in ((got, True), (want, False)):
        leaves = [t.clone().requires_grad_(), model.head.weight.detach().clone().requires_grad_(), model.head.bias.detach().clone().requires_grad_()]
        if own:
            from spion_b200.vocab import linear_cross_entropy
            with torch.autocast("cuda", dtype=torch.bfloat16, enabled=dtype == "bf16"):
                loss = linear_cross_entropy(leaves[0], leaves[1], labels, leaves[2])
        else:
            z = leaves[0].double() @ leaves[1].double().t() + leaves[2].double()
            loss = torch.nn.functional.cross_entropy(z.flatten(0, 1), labels.flatten())
        out += [loss.detach().double()] + [g.double() for g in torch.autograd.grad(loss, leaves)]
    for p, q in zip(got, want):
        assert float((p - q).norm()) <= (1e-5 if dtype == "fp32" else 2.0 ** -6) * float(q.norm())
    loss, _ = model(ids, labels, tr.mat_lst)
    assert abs(float(loss.detach()) - float(want[0])) <= (1e-5 if dtype == "fp32" else 2.0 ** -6) * float(want[0])


@pytest.mark.parametrize("dtype,optimizer", [("fp32", "torch"), ("bf16", "fused")])
def test_captured_steps_are_the_eager_ones(dtype, optimizer):
    """Every sum of the loss and of the table has a fixed order: the same steps, the same parameters."""
    runs = []
    for captured in (False, True):
        tr, ids, labels, _ = trainer("text" if dtype == "bf16" else "image", dtype, optimizer=optimizer, tied_weights=True)
        start(tr, ids, labels)
        losses = []
        if captured:
            tr.capture_sparse_step(ids, labels, warmup=2)
            losses = [float(tr.step_graph(ids, labels)) for _ in range(2)]
        else:
            for i in range(4):
                loss = float(tr.step(ids, labels)[0])
                losses += [loss] if i >= 2 else []
        tr.check_device_status()
        runs.append((losses, [p.detach().clone() for p in tr.model.parameters()]))
    assert np.isfinite(runs[0][0]).all()
    for a, b in zip(*[r[0] for r in runs]):
        assert abs(a - b) <= 1e-4 * abs(a)
    assert all(bool(torch.isfinite(p).all()) for p in runs[1][1])


def test_a_teachers_logits_and_evaluation():
    tr, ids, labels, g = trainer("text", "bf16", temperature=2.0)
    start(tr, ids, labels)
    idx = torch.randint(0, 700, (*ids.shape, 8), generator=g, device="cuda")
    idx[labels < 0] = -1
    logits = torch.randn(idx.shape, generator=g, device="cuda")
    losses = [float(tr.step(ids, (idx, logits))[0]) for _ in range(3)]
    assert np.isfinite(losses).all()
    tr.capture_sparse_step(ids, (idx, logits), warmup=2)
    assert np.isfinite(float(tr.step_graph(ids, (idx, logits * 0.5))))
    assert torch.equal(tr._g_lab[1], logits * 0.5)
    loss, right = tr.evaluate(ids, labels)
    assert right is None and bool(torch.isfinite(loss))
    loss8 = trainer("text", "bf16", eval_linear_bits=8)
    start(*loss8[:3])
    assert bool(torch.isfinite(loss8[0].evaluate(*loss8[1:3])[0]))


def test_a_wait_that_gave_up_is_reported_and_no_step_is_taken():
    from spion_b200 import _lib
    tr, ids, labels, _ = trainer("text", "bf16", optimizer="fused")
    start(tr, ids, labels)
    before = [p.detach().clone() for p in tr.model.parameters()]
    _lib.check(_lib.lib.spion_linear_selftest_bounded_wait(1000, _lib.current_stream_ptr()))
    torch.cuda.synchronize()
    from spion_b200.vocab import linear_cross_entropy
    x, w = torch.randn(40, 64, device="cuda", requires_grad=True), torch.randn(300, 64, device="cuda", requires_grad=True)
    lab = torch.randint(0, 300, (40,), device="cuda")
    loss = linear_cross_entropy(x, w, lab)
    grads = torch.autograd.grad(loss, (x, w))
    assert bool(loss.isnan()) and all(bool(t.isnan().all()) for t in grads)
    tr.step(ids, labels)
    assert all(torch.equal(a, b) for a, b in zip(before, tr.model.parameters()))
    with pytest.raises(_lib.SpionError):
        tr.check_device_status()
    assert bool(torch.isfinite(linear_cross_entropy(x, w, lab)))
    tr.step(ids, labels)
    assert not all(torch.equal(a, b) for a, b in zip(before, tr.model.parameters()))


def test_configurations_that_are_refused():
    from spion_b200 import harness
    base = harness.task_config("image", 2, native=True)
    for bad in (dict(objective="words"), dict(embedding="big"), dict(embedding_scale=2.0), dict(objective="tokens", dual=True)):
        with pytest.raises(ValueError):
            harness.Trainer({**base, **bad})
