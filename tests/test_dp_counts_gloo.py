"""Two ranks whose losses are means over different numbers of labels (gloo, no GPU): the gradients are those of the mean over all labels."""
import os
import sys
from types import SimpleNamespace

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INF = float("inf")


def model_and_data(counts):
    torch.manual_seed(0)
    model = torch.nn.Linear(8, 5)
    g = torch.Generator().manual_seed(1)
    x, labels = torch.randn(2, 9, 8, generator=g), torch.randint(0, 5, (2, 9), generator=g)
    for rank, n in enumerate(counts):
        labels[rank, n:] = -100
    return model, x, labels


def loss_of(model, x, labels):
    """The mean over what has a label; gradients of 0 where nothing has, as the losses over a vocabulary."""
    rows = labels != -100
    if not bool(rows.any()):
        return (model(x) * 0).sum()
    return torch.nn.functional.cross_entropy(model(x[rows]), labels[rows])


def as_teacher(labels):
    """The same positions as entries of a teacher: one that is left out by its index, one by its logit."""
    idx = torch.stack([labels, torch.full_like(labels, -1), labels], -1)
    idx = torch.where(idx == -100, -1, idx)
    logits = torch.zeros(idx.shape)
    idx[..., 2], logits[..., 2] = 1, -INF
    return idx, logits


def _worker(rank, port, counts, teacher, out):
    sys.path.insert(0, ROOT)
    os.environ.update(RANK=str(rank), WORLD_SIZE="2", MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    from spion_b200 import dp, harness
    dp.init_from_env("gloo", timeout_s=60)
    model, x, labels = model_and_data(counts)
    trainer = harness.Trainer.__new__(harness.Trainer)
    trainer.model, trainer.bucket = SimpleNamespace(counted=harness.TokenModel.counted), dp.FlatGradBucket(model.parameters())
    trainer.bucket.backward(loss_of(model, x[rank], labels[rank]))
    trainer._average(as_teacher(labels[rank]) if teacher else labels[rank])
    torch.save(trainer.bucket.flat.clone(), f"{out}.{rank}")
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize("counts,teacher", [((9, 2), False), ((5, 0), False), ((0, 0), False), ((3, 7), True)])
def test_the_mean_is_that_of_all_labels(tmp_path, counts, teacher):
    out = str(tmp_path / "flat")
    mp.spawn(_worker, args=(31000 + (os.getpid() * 8 + sum(counts)) % 2000, counts, teacher, out), nprocs=2, join=True)
    got = [torch.load(f"{out}.{rank}") for rank in (0, 1)]
    model, x, labels = model_and_data(counts)
    loss_of(model, x.flatten(0, 1), labels.flatten()).backward()
    want = torch.cat([p.grad.reshape(-1) for p in model.parameters()])
    assert torch.equal(*got)
    torch.testing.assert_close(got[0], want, rtol=1e-5, atol=1e-6)


def test_counts():
    from spion_b200.harness import Classifier, TokenModel
    labels = torch.tensor([[3, -100, -100], [0, 1, -100]])
    assert int(TokenModel.counted(labels)) == 3 and int(TokenModel.counted(as_teacher(labels))) == 3
    assert Classifier.counted(labels) is None
