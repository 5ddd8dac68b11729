"""Operators at the two ends of a model with a vocabulary, as cases to time and compare: rows of a token table with a scale and their gradient, the cross
entropy over the vocabulary from the rows before the last layer, and the same loss against a teacher's largest logits.

``run`` computes each in its plain form (elementary torch operations in fp32); with ``own`` set it calls this framework's operators.
``exact`` is the definition in fp64.  Sizes are the encoder's own (width 64, vocabulary 256, sequences of 4096) and generic ones.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
IGNORE = -100


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one id on its way into a decoder of width 4096: latency
        {"name": "embed_token", "op": "embed", "ids": 1, "vocab": 32000, "width": 4096, "type": "bf16", "scale": 1.0, "padding": 0.0, "train": False},
        # a training step's batch of 32 sequences of 4096, ids as unequally frequent as words are
        {"name": "embed_step", "op": "embed", "ids": 131072, "vocab": 32000, "width": 1024, "type": "bf16", "scale": 32.0, "padding": 0.0, "train": True},
        # the encoder's width, a table beyond shared memory, sequences half of which are padding
        {"name": "embed_padded", "op": "embed", "ids": 131072, "vocab": 8192, "width": 64, "type": "fp32", "scale": 1.0, "padding": 0.5, "train": True},
        # odd sizes
        {"name": "embed_odd", "op": "embed", "ids": 4099, "vocab": 10007, "width": 769, "type": "fp16", "scale": 27.7, "padding": 0.1, "train": True},
        # a few tokens scored, one loss each: the weights are what has to be read
        {"name": "loss_score_few", "op": "loss", "rows": 16, "width": 2048, "vocab": 32000, "type": "fp16", "bias": False, "counted": 1.0, "reduction": "none",
         "train": False},
        # masked-token training of the encoder: 32 sequences of 4096, one position in seven asked for, its vocabulary of bytes
        {"name": "loss_encoder_masked", "op": "loss", "rows": 131072, "width": 64, "vocab": 256, "type": "bf16", "bias": True, "counted": 0.15, "reduction": "mean",
         "train": True},
        # a training step of a wide model: 8192 positions, a large vocabulary
        {"name": "loss_step", "op": "loss", "rows": 8192, "width": 4096, "vocab": 128000, "type": "bf16", "bias": False, "counted": 1.0, "reduction": "mean",
         "train": True},
        # masked-token training, a vocabulary that is no multiple of anything, bias
        {"name": "loss_masked_odd", "op": "loss", "rows": 16384, "width": 1024, "vocab": 50021, "type": "bf16", "bias": True, "counted": 0.15, "reduction": "mean",
         "train": True},
        # everything in fp32, a gradient for each row's loss
        {"name": "loss_fp32_odd", "op": "loss", "rows": 777, "width": 300, "vocab": 5003, "type": "fp32", "bias": True, "counted": 0.9, "reduction": "none",
         "train": True},
        # distillation of a small model on the encoder's vocabulary: latency
        {"name": "distill_small", "op": "distill", "rows": 64, "width": 64, "vocab": 256, "type": "fp32", "bias": True, "counted": 1.0, "top": 8, "temperature": 1.0,
         "reduction": "mean", "train": True},
        # a training step against 32 logits a position
        {"name": "distill_step", "op": "distill", "rows": 8192, "width": 2048, "vocab": 32000, "type": "bf16", "bias": False, "counted": 1.0, "top": 32,
         "temperature": 2.0, "reduction": "mean", "train": True},
        # odd sizes, rows of fewer logits and rows of none
        {"name": "distill_odd", "op": "distill", "rows": 1001, "width": 770, "vocab": 10007, "type": "fp16", "bias": True, "counted": 0.8, "top": 11,
         "temperature": 1.5, "reduction": "none", "train": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embed", "embed", "loss", "loss", "distill"])
    kind = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if op == "embed":
        width = _log(rng, 1, 4096)
        if rng.random() < 0.6:
            width = -(-width // 8) * 8
        return {"op": op, "ids": _log(rng, 1, min(262144, (1 << 27) // width)), "vocab": _log(rng, 1, min(200000, (1 << 28) // width)), "width": width, "type": kind,
                "scale": rng.choice([1.0, 0.3, math.sqrt(width)]), "padding": rng.choice([0.0, 0.0, 0.1, 0.6]), "train": rng.random() < 0.8}
    width = _log(rng, 1, 4096)
    if rng.random() < 0.6:
        width = -(-width // 16) * 16
    vocab = _log(rng, 2, 100000)
    rows = _log(rng, 1, max(1, min(65536, (1 << 38) // (width * vocab), (1 << 32) // vocab)))
    case = {"op": op, "rows": rows, "width": width, "vocab": vocab, "type": kind, "bias": rng.random() < 0.5, "counted": rng.choice([1.0, 1.0, 0.8, 0.15]),
            "reduction": rng.choice(["mean", "mean", "sum", "none"]), "train": rng.random() < 0.8}
    if op == "distill":
        case.update(top=min(vocab, _log(rng, 1, 64)), temperature=rng.choice([1.0, 1.0, 2.0, 0.7]))
    return case


def _counted(c):
    return max(1, round(c["rows"] * c["counted"]))


def work(c):
    e = 4 if c["type"] == "fp32" else 2
    if c["op"] == "embed":
        t, n, v = c["ids"], c["width"], c["vocab"]
        read = min(t, v)                                               # rows of the table, each once
        forward = 8 * t + (t + read) * n * e
        return {"bytes": forward + ((t + v) * n * e if c["train"] else 0), "flops": (2 if c["train"] else 1) * t * n}
    t, k, v, n = c["rows"], c["width"], c["vocab"], _counted(c)
    target = 12 * n * c["top"] if c["op"] == "distill" else 8 * t
    read = n * k * e + v * k * e + target + (4 * v if c["bias"] else 0)
    written = (t if c["reduction"] == "none" else 1) * 4
    if c["train"]:
        written += t * k * e + v * k * e + (4 * v if c["bias"] else 0)
    return {"bytes": read + written, "flops": (6 if c["train"] else 2) * n * k * v}


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _word_ids(count, vocab, g):
    """Ids as unequally frequent as words: the r-th has a share of about 1 / r, in an order of their own."""
    r = torch.exp(torch.rand(count, generator=g, device="cuda", dtype=torch.float64) * math.log(vocab + 1.0)).long() - 1
    return torch.randperm(vocab, generator=g, device="cuda")[r.clamp(0, vocab - 1)]


def prepare(c, seed):
    g = _generator(seed)
    dt = DTYPES[c["type"]]
    s = {"case": c}
    if c["op"] == "embed":
        ids = _word_ids(c["ids"], c["vocab"], g)
        s["padding_idx"] = None
        if c["padding"] > 0:
            s["padding_idx"] = 0                                       # a tail of the sequence, which has no gradient
            ids[c["ids"] - int(c["ids"] * c["padding"]):] = 0
        s["ids"] = ids
        s["w"] = (0.02 * torch.randn(c["vocab"], c["width"], generator=g, device="cuda")).to(dt).requires_grad_(c["train"])
        if c["train"]:
            s["dy"] = (1e-2 * torch.randn(c["ids"], c["width"], generator=g, device="cuda")).to(dt)
        return s
    t, k, v, n = c["rows"], c["width"], c["vocab"], _counted(c)
    size = 2.0                                                         # standard deviation of the logits
    w = torch.randn(v, k, generator=g, device="cuda") * (size / math.sqrt(k))
    x = torch.randn(t, k, generator=g, device="cuda")
    likely = _word_ids(t, v, g)
    x += torch.rand(t, 1, generator=g, device="cuda") * (2.0 / size) * w[likely]      # what is asked for is likely, more or less
    counted = torch.zeros(t, dtype=torch.bool, device="cuda")
    counted[torch.randperm(t, generator=g, device="cuda")[:n]] = True
    s["x"], s["w"] = x.to(dt).requires_grad_(c["train"]), w.to(dt).requires_grad_(c["train"])
    s["b"] = (0.3 * torch.randn(v, generator=g, device="cuda")).requires_grad_(c["train"]) if c["bias"] else None
    if c["train"] and c["reduction"] == "none":
        s["g"] = torch.randn(t, generator=g, device="cuda") / t
    if c["op"] == "loss":
        s["labels"] = torch.where(counted, likely, IGNORE)
        return s
    top = c["top"]
    gaps = 1 + (torch.rand(t, top, generator=g, device="cuda") * (v // top)).long().clamp(max=max(0, v // top - 1))
    idx = (likely[:, None] + torch.cumsum(gaps, 1) - gaps[:, :1]) % v  # different ones, from the likely one on
    logits = 8.0 - torch.cumsum(torch.rand(t, top, generator=g, device="cuda"), 1)
    if c["counted"] < 1.0:                                             # some teachers gave fewer, and nothing where nothing is asked for
        left = torch.randint(1, top + 1, (t, 1), generator=g, device="cuda")
        idx = torch.where((torch.arange(top, device="cuda") < left) & counted[:, None], idx, -1)
    s["idx"], s["teacher"] = idx, logits.to(dt)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    op = s["case"]["op"]
    if op == "embed":
        return _embed_own(s) if own else _embed_plain(s)
    return _loss_own(s) if own else _loss_plain(s)


def _embed_own(s):
    from spion_b200.tokens import embed_tokens
    y = embed_tokens(s["ids"], s["w"], scale=s["case"]["scale"], padding_idx=s["padding_idx"])
    if not s["case"]["train"]:
        return {"y": y}
    return {"y": y, "dw": torch.autograd.grad(y, s["w"], s["dy"])[0]}


def _loss_own(s):
    c = s["case"]
    if c["op"] == "loss":
        from spion_b200.vocab import linear_cross_entropy
        loss = linear_cross_entropy(s["x"], s["w"], s["labels"], s["b"], ignore_index=IGNORE, reduction=c["reduction"])
    else:
        from spion_b200.vocab import distill_top_logits
        loss = distill_top_logits(s["x"], s["w"], s["idx"], s["teacher"], s["b"], temperature=c["temperature"], reduction=c["reduction"])
    if not c["train"]:
        return {"loss": loss}
    leaves = [s["x"], s["w"]] + ([s["b"]] if c["bias"] else [])
    return dict(zip(("dx", "dw", "db"), torch.autograd.grad(loss, leaves, s.get("g")))) | {"loss": loss}


# ------------------------------------------------------------------------------------------------ plain forms
def _embed_plain(s):
    c, w, ids = s["case"], s["w"].detach(), s["ids"]
    y = (w[ids].float() * c["scale"]).to(w.dtype)
    if not c["train"]:
        return {"y": y}
    dw = torch.zeros(w.shape, device="cuda")
    dw.index_add_(0, ids, s["dy"].float())
    if s["padding_idx"] is not None:
        dw[s["padding_idx"]] = 0
    return {"y": y, "dw": (dw * c["scale"]).to(w.dtype)}


def _loss_plain(s):
    c, x, w = s["case"], s["x"].detach(), s["w"].detach()
    tau = c.get("temperature", 1.0)
    if c["op"] == "loss":
        rows = (s["labels"] != IGNORE).nonzero().squeeze(1)
        idx = s["labels"][rows][:, None]
        q = torch.ones(idx.shape, device="cuda")
        entropy = 0.0
    else:
        rows = (s["idx"] >= 0).any(1).nonzero().squeeze(1)
        idx = s["idx"][rows]
        there = idx >= 0
        t = torch.where(there, s["teacher"][rows].float() / tau, -torch.inf)
        e = torch.exp(t - t.amax(1, keepdim=True))
        q = e / e.sum(1, keepdim=True)
        entropy = torch.where(q > 0, q * torch.log(q), 0.0).sum(1)
        idx = idx.clamp_min(0)
    xr, wf = x[rows].float(), w.float()
    z = xr @ wf.t()
    if s["b"] is not None:
        z += s["b"].detach()
    z /= tau
    top = z.amax(1, keepdim=True)
    asked = (z.gather(1, idx) * q).sum(1)
    z = torch.exp(z - top)
    total = z.sum(1, keepdim=True)
    each = entropy - asked + (torch.log(total) + top).squeeze(1)
    n = len(rows)
    if c["reduction"] == "none":
        loss = torch.zeros(c["rows"], device="cuda")
        loss[rows] = each
    else:
        loss = each.sum() / (n if c["reduction"] == "mean" else 1)
    if not c["train"]:
        return {"loss": loss}
    z /= total
    z.scatter_add_(1, idx, -q)
    if c["reduction"] == "none":
        z *= s["g"][rows][:, None] / tau
    else:
        z /= tau * (n if c["reduction"] == "mean" else 1)
    dx = torch.zeros(x.shape, dtype=x.dtype, device="cuda")
    dx[rows] = (z @ wf).to(x.dtype)
    out = {"dx": dx, "dw": (z.t() @ xr).to(w.dtype), "loss": loss}
    if s["b"] is not None:
        out["db"] = z.sum(0)
    return out


# ------------------------------------------------------------------------------------------------ the definitions in fp64
def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "embed":
        w = s["w"].detach().double()
        y = (w * c["scale"]).index_select(0, s["ids"])
        if not c["train"]:
            return {"y": y}
        given = s["dy"].double()
        if s["padding_idx"] is not None:
            given = given * (s["ids"] != s["padding_idx"])[:, None]
        order = torch.argsort(s["ids"], stable=True)
        ends = torch.cumsum(torch.bincount(s["ids"], minlength=c["vocab"]), 0)
        dw = torch.zeros(c["vocab"], c["width"], dtype=torch.float64, device="cuda")
        for column in range(0, c["width"], 256):                       # differences of running sums, a few columns at a time
            sums = torch.nn.functional.pad(torch.cumsum(given[order, column:column + 256], 0), (0, 0, 1, 0))[ends]
            dw[:, column:column + 256] = torch.diff(sums, dim=0, prepend=torch.zeros_like(sums[:1])) * c["scale"]
        return {"y": y, "dw": dw}
    tau = c.get("temperature", 1.0)
    leaves = [t.detach().double().requires_grad_(c["train"]) for t in (s["x"], s["w"], s["b"]) if t is not None]
    if c["op"] == "loss":
        keep = s["labels"] != IGNORE
        target = s["labels"].clamp_min(0)[:, None]
        log_q = torch.zeros_like(target, dtype=torch.float64)
    else:
        keep = s["idx"].amax(1) >= 0
        target = s["idx"].clamp_min(0)
        log_q = torch.log_softmax(torch.where(s["idx"] < 0, -torch.inf, s["teacher"].double() / tau), 1)
        log_q = torch.where(s["idx"] < 0, -torch.inf, log_q)
    target, log_q = target[keep], log_q[keep]
    z = torch.nn.functional.linear(leaves[0][keep], leaves[1], leaves[2] if c["bias"] else None) / tau
    log_p = torch.take_along_dim(z, target, 1) - torch.logsumexp(z, 1, keepdim=True)
    q = torch.exp(log_q)
    each = torch.where(q > 0, q * (torch.where(q > 0, log_q, 0.0) - log_p), 0.0).sum(1)
    if c["reduction"] == "none":
        loss = torch.zeros(c["rows"], dtype=torch.float64, device="cuda").masked_scatter(keep, each)
    else:
        loss = each.mean() if c["reduction"] == "mean" else each.sum()
    if not c["train"]:
        return {"loss": loss}
    del log_p
    grads = torch.autograd.grad(loss, leaves, s["g"].double() if c["reduction"] == "none" else None)
    return dict(zip(("dx", "dw", "db"), grads)) | {"loss": loss.detach()}
