"""The encoder's operators together, as a training run uses them: root-mean-square norms, the fused AdamW step with moments in 32 and 8 bits, captured steps,
and evaluation with the linear layers on 8-bit operands."""
import numpy as np
import pytest
import torch

from spion_b200 import synthetic

pytestmark = pytest.mark.gpu


def trainer(task="image", dtype="fp32", L=256, batch=4, **overrides):
    from spion_b200 import harness
    cfg = harness.task_config(task, batch, native=True, dtype=dtype)
    cfg.update(max_seq_len=L, dropout_prob=0.0, attention_dropout=0.0, threshold=0.85, norm="rms", optimizer="fused")
    cfg.update(overrides)
    tr = harness.Trainer(cfg, lr=1e-3, seed=3)
    ids = synthetic.token_ids(5, batch, L).cuda()
    ids = (ids, synthetic.token_ids(6, batch, L).cuda()) if cfg["dual"] else ids
    return tr, ids, synthetic.labels(5, batch, cfg["num_classes"]).cuda()


def start(tr, ids, lab):
    _, maps = tr.step(ids, lab, is_attn=True)
    tr.discover(maps)


def test_first_step_is_the_frameworks():
    """The same gradients through both optimizers: a first step moves every parameter by at most lr, the quotient is some tens of units in its last place off
    (test_gpu_optim.py: 16 u), and the parameter itself 3 u."""
    a, ids, lab = trainer()
    b, _, _ = trainer(optimizer="torch")
    assert all(torch.equal(x, y) for x, y in zip(a.model.parameters(), b.model.parameters()))
    start(a, ids, lab), start(b, ids, lab)
    assert torch.equal(a.bucket.flat.clamp(-1, 1), b.bucket.flat)         # the fused step clips as it reads
    for x, y in zip(a.model.parameters(), b.model.parameters()):
        assert bool(((x - y).abs() <= 1e-3 * 32 * 2.0 ** -24 + 4 * 2.0 ** -24 * x.abs()).all())


@pytest.mark.parametrize("task,dtype,L,bits", [("image", "fp32", 256, 32), ("image", "fp32", 256, 8), ("text", "bf16", 512, 8), ("retrieval", "bf16", 512, 32)])
def test_training_then_evaluation(task, dtype, L, bits):
    tr, ids, lab = trainer(task, dtype, L, batch=2, optimizer_state_bits=bits, eval_linear_bits=8)
    start(tr, ids, lab)
    losses = [float(tr.step(ids, lab)[0]) for _ in range(3)]
    assert np.isfinite(losses).all()
    if tr._shadow is not None:                                             # written by the optimizer's own pass
        for p, c in zip(*tr._shadow):
            assert torch.equal(c, p.detach().to(c.dtype))
    before = [p.detach().clone() for p in tr.model.parameters()]
    loss8, right8 = tr.evaluate(ids, lab)
    tr.config["eval_linear_bits"] = 16
    loss, right = tr.evaluate(ids, lab)
    assert tr.model.training and all(torch.equal(a, b) for a, b in zip(before, tr.model.parameters()))
    # Operands within 2^-4 each, errors of independent signs: a sum over 64 features or more is off by less than 2^-4 of its size, and six of them lead
    # to scores of order one here
    assert bool(torch.isfinite(loss8)) and abs(float(loss8 - loss)) < 0.25
    assert 0 <= float(right8) <= 1 and 0 <= float(right) <= 1
    again, _ = tr.evaluate(ids, lab)
    assert float(again) == float(loss)
    assert np.isfinite(float(tr.step(ids, lab)[0]))


def test_evaluation_in_8_bits_with_layer_norm_and_without_a_pattern():
    tr, ids, lab = trainer(norm="layer", optimizer="torch", eval_linear_bits=8)
    with pytest.raises(RuntimeError, match="discover"):
        tr.evaluate(ids, lab)
    start(tr, ids, lab)
    loss8, _ = tr.evaluate(ids, lab)
    assert bool(torch.isfinite(loss8))
    # quantised layers are for calls without gradients: a training step passes them by
    tr.model.quantize()
    loss, _ = tr.step(ids, lab)
    tr.model.quantize(False)
    assert np.isfinite(float(loss))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps(bits):
    """Three steps and a captured one replayed three times are the same six steps: the same losses up to the order of sums that atomics may change, which
    Adam's sign-like first steps can turn into lr per parameter and step."""
    a, ids, lab = trainer(optimizer_state_bits=bits)
    b, _, _ = trainer(optimizer_state_bits=bits)
    start(a, ids, lab), start(b, ids, lab)
    b.capture_sparse_step(ids, lab, warmup=3)
    for _ in range(3):
        a.step(ids, lab)
    for _ in range(3):
        want, _ = a.step(ids, lab)
        got = b.step_graph(ids, lab)
        assert abs(float(got) - float(want)) <= 1e-3 * max(1.0, abs(float(want)))
    steps = [float(s["step"]) for s in b.opt.state.values()]
    assert set(steps) == {7.0}


def test_unknown_norm_is_refused():
    with pytest.raises(ValueError, match="norm"):
        trainer(norm="batch")


def test_evaluation_leaves_what_was_quantised_as_it_was():
    """quantize() keeps its weights until quantize(False), whatever is evaluated between; evaluate() is on what the configuration says and on the weights of
    the moment."""
    tr, ids, lab = trainer()
    start(tr, ids, lab)
    plain, _ = tr.evaluate(ids, lab)
    tr.config["eval_linear_bits"] = 8
    eight, _ = tr.evaluate(ids, lab)
    assert float(eight) != float(plain)
    layers = tr.model.model.layers
    assert not tr.model.model.quantized and all(m.mha.linear8 is None and m.mlp8 is None for m in layers)
    tr.model.quantize()
    kept = [(m.mha.linear8, m.mlp8) for m in layers]
    codes = [m.values.clone() for a, b in kept for m in (*a, *b)]
    with torch.no_grad():
        for p in tr.model.model.layers.parameters():
            p.mul_(1.25)
    with torch.no_grad():
        tr.model.eval()
        scores = tr.model.scores(ids, tr.mat_lst)
        tr.model.train()
    moved, _ = tr.evaluate(ids, lab)                                       # of the new weights
    tr.config["eval_linear_bits"] = None
    other, _ = tr.evaluate(ids, lab)                                       # not in 8 bits
    tr.model.quantize(False)
    assert float(tr.evaluate(ids, lab)[0]) == float(other)
    tr.config["eval_linear_bits"] = 8
    assert float(tr.evaluate(ids, lab)[0]) == float(moved) and float(moved) != float(eight)
    tr.model.quantize()
    for m, k in zip(layers, kept):
        m.mha.linear8, m.mlp8 = k
    tr.evaluate(ids, lab)
    assert tr.model.model.quantized and all(m.mha.linear8 is a and m.mlp8 is b for m, (a, b) in zip(layers, kept))
    assert all(torch.equal(m.values.view(torch.uint8), c.view(torch.uint8)) for m, c in zip([m for a, b in kept for m in (*a, *b)], codes))
    with torch.no_grad():
        tr.model.eval()
        assert torch.equal(tr.model.scores(ids, tr.mat_lst), scores)


@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_replaced_and_hooked_modules_of_an_8_bit_evaluation(norm):
    """A norm that is hooked is called as a module; of linear layers, of the attention and of what lies between them an 8-bit evaluation calls no forward of their
    own, so a hook or another module there is refused."""
    from spion_b200._lib import SpionError
    tr, ids, lab = trainer(norm=norm, eval_linear_bits=8)
    start(tr, ids, lab)
    want, _ = tr.evaluate(ids, lab)
    layer, seen = tr.model.model.layers[1], []
    hook = layer.norm2.register_forward_hook(lambda m, x, y: seen.append(y.shape))
    got, _ = tr.evaluate(ids, lab)
    hook.remove()
    assert seen == [(4, 256, 64)] and abs(float(got) - float(want)) < 1e-2     # the same codes but for ties
    hook = layer.norm1.register_forward_hook(lambda m, x, y: y * 2)            # a power of two: the same codes, other scales
    doubled, _ = tr.evaluate(ids, lab)
    hook.remove()
    assert float(doubled) != float(want)

    def refused():
        with pytest.raises(SpionError, match="hook"):
            tr.evaluate(ids, lab)
        assert not tr.model.model.quantized and layer.mha.linear8 is None and layer.mlp8 is None and tr.model.training

    for m in (layer.mha.W_q, layer.mha.W_k, layer.mha.W_v, layer.mha.ff, layer.mha, layer.mlpblock, layer.mlpblock[0], layer.mlpblock[3], layer.mlpblock[4], layer.dropout1):
        hook = m.register_forward_hook(lambda m, x, y: None)
        refused()
        hook.remove()
        hook = m.register_forward_pre_hook(lambda m, x: None)
        refused()
        hook.remove()
    for owner, name in ((layer.mha, "W_k"), (layer.mha, "ff"), (layer.mlpblock, "0"), (layer.mlpblock, "2"), (layer, "dropout1")):
        was = owner._modules[name]
        owner._modules[name] = torch.nn.Identity()
        refused()
        owner._modules[name] = was
    hook = torch.nn.modules.module.register_module_forward_hook(lambda m, x, y: None)
    refused()
    hook.remove()
    tr.model.quantize()
    hook = layer.mha.W_v.register_forward_hook(lambda m, x, y: None)           # hooked after it was quantised
    with torch.no_grad(), pytest.raises(SpionError, match="hook"):
        tr.model.eval()
        tr.model.scores(ids, tr.mat_lst)
    hook.remove()
    tr.model.train()
    tr.model.quantize(False)
    assert float(tr.evaluate(ids, lab)[0]) == float(want)


def test_8_bit_layers_go_where_their_model_goes():
    tr, ids, lab = trainer()
    start(tr, ids, lab)
    keys = list(tr.model.state_dict())
    tr.model.quantize()
    assert list(tr.model.state_dict()) == keys
    tr.model.to("cpu")
    layers = [m for x in tr.model.model.layers for m in (*x.mha.linear8, *x.mlp8)]
    assert all(t.device.type == "cpu" for m in layers for t in (m.values, m.scales, m.bias))
    tr.model.to("cuda")
    assert all(t.is_cuda for m in layers for t in (m.values, m.scales, m.bias))


def test_unknown_optimizers_and_widths_are_refused():
    for bad, match in ((dict(optimizer="adam8"), "optimizer"), (dict(optimizer="Fused"), "optimizer"), (dict(eval_linear_bits=4), "eval_linear_bits"),
                       (dict(optimizer="torch", optimizer_state_bits=8), "optimizer_state_bits"), (dict(optimizer_state_bits=16), "state_bits")):
        with pytest.raises(ValueError, match=match):
            trainer(**bad)
    tr, ids, lab = trainer(optimizer="torch")
    start(tr, ids, lab)
    tr.config["eval_linear_bits"] = 6
    with pytest.raises(ValueError, match="eval_linear_bits"):
        tr.evaluate(ids, lab)


def test_every_stage_of_an_8_bit_evaluation(monkeypatch):
    """The encoder's pass on 8-bit operands, stage by stage: every value that a stage hands on is the next one's operand, in the place where it belongs, and each
    stage is its formula on the operands that it got, in fp64.

    Bounds, u = 2^-24: a linear layer as in test_gpu_linear_e4m3.py (U * (K / 8 + 16) of the sum of sizes, then a rounding to its type).  Rows in 8 bits: 2^-4 of
    the value, half of the smallest step 2^-9 of the row's scale, and for the norm (K(N) / 2 + 8) u as in test_gpu_rmsnorm.py, 2^-7 more where the layer norm's
    output was bf16 before."""
    from spion_b200 import harness, quant
    u = 2.0 ** -24
    for norm, task, dtype, L in (("rms", "text", "fp32", 512), ("layer", "text", "bf16", 512), ("rms", "image", "bf16", 256), ("layer", "image", "fp32", 256)):
        tr, ids, lab = trainer(task, dtype, L, batch=2, norm=norm)
        ids = ids.clone()
        ids[0, L - 100:], ids[1, 7:] = 0, 0                                # padding
        start(tr, ids, lab)
        encoder, linears, norms, attended = tr.model.model, [], [], []

        def linear(x, w, bias=None, out_dtype=None, plain=quant.linear_e4m3):
            y = plain(x, w, bias, out_dtype)
            linears.append((x, w, bias, y))
            return y

        def rows8(m, x, res=None, plain=harness.norm_rows8):
            y = plain(m, x, res)
            norms.append((m, x, res, y))
            return y

        monkeypatch.setattr(quant, "linear_e4m3", linear)
        monkeypatch.setattr(harness, "norm_rows8", rows8)
        hooks = [x.mha.block_attn.register_forward_hook(lambda m, args, y: attended.append((m, args, y[0]))) for x in encoder.layers]
        tr.model.eval()
        mask = (ids != 0).float()
        amp = lambda: torch.autocast("cuda", dtype=torch.bfloat16, enabled=tr.model.amp)      # noqa: E731
        with torch.no_grad(), amp():
            unquantised, _ = encoder(ids, mask, tr.mat_lst)
            attended.clear()
            tr.model.quantize()
            out, _ = encoder(ids, mask, tr.mat_lst)
            tr.model.quantize(False)
            X = encoder.embeddings(ids)
            again = [(m, args, m(*args)[0]) for m, args, _ in list(attended)]
        [h.remove() for h in hooks]
        monkeypatch.undo()
        attended = attended[:len(encoder.layers)]
        assert len(linears) == 6 * len(encoder.layers) and len(norms) == 2 * len(encoder.layers) and len(attended) == len(encoder.layers)

        def check_linear(call, x, layer):
            got, w, bias, y = call
            assert got is x if isinstance(x, quant.Rows8) else torch.equal(got, x)
            codes = quant.quantize_rows(layer.weight.detach())
            assert torch.equal(w.values.view(torch.uint8), codes.values.view(torch.uint8)) and torch.equal(w.scales, codes.scales)
            assert torch.equal(bias, layer.bias)
            q = x if isinstance(x, quant.Rows8) else quant.quantize_rows(x)
            A, B = q.values.double() * q.scales.double()[..., None], w.values.double() * w.scales.double()[:, None]
            want, size = A @ B.t() + bias.double(), A.abs() @ B.abs().t() + bias.double().abs()
            bound = size * u * (A.shape[-1] / 8 + 16) + want.abs() * torch.finfo(y.dtype).eps / 2 + 1e-38
            assert bool(((y.double() - want).abs() <= bound).all())
            return y

        def check_rows(call, layer, x, res):
            m, got, r, y = call
            assert m is layer and (got is x or torch.equal(got, x)) and (r is res if res is None else torch.equal(r, res))
            s, q = (x, y) if res is None else y
            if res is not None:
                want = x.double() + res.double()
                assert bool(((s.double() - want).abs() <= want.abs() * 3 * u).all())
            S = s.double()
            if norm == "layer":
                S = S - S.mean(-1, keepdim=True)
            n = S / torch.sqrt((S * S).mean(-1, keepdim=True) + m.eps) * m.weight.double() + (m.bias.double() if norm == "layer" else 0)
            rel = (64 / 2 + 64) * u + (2.0 ** -7 if norm == "layer" and dtype == "bf16" else 0)
            size = n.abs() + (S.abs().amax(-1, keepdim=True) * 64 * u if norm == "layer" else 0)      # (differences of the mean: absolute errors)
            off = (q.values.double() * q.scales.double()[..., None] - n).abs()
            assert bool((off <= size * (2.0 ** -4 + 2 * rel) + q.scales.double()[..., None] * 2.0 ** -10 * 1.01 + 1e-6).all())
            return s, q

        branch = None
        for i, layer in enumerate(encoder.layers):
            lin, mha = linears[6 * i:6 * i + 6], layer.mha
            X, n1 = check_rows(norms[2 * i], layer.norm1, X, branch)
            heads = [mha.split_heads(check_linear(lin[k], n1, w)) for k, w in enumerate((mha.W_q, mha.W_k, mha.W_v))]
            m, args, o = attended[i]
            assert m is mha.block_attn and all(torch.equal(a, b) for a, b in zip(args, (*heads, mask, tr.mat_lst[0][i])))
            assert torch.equal(again[i][2], o)
            out1 = check_linear(lin[3], mha.combine_heads(o), mha.ff)
            X, n2 = check_rows(norms[2 * i + 1], layer.norm2, X, out1)
            hidden = check_linear(lin[4], n2, layer.mlpblock[0])
            branch = check_linear(lin[5], torch.nn.functional.gelu(hidden), layer.mlpblock[3])
        with torch.no_grad(), amp():
            want = encoder.norm(X + branch) * mask[..., None]
        assert torch.equal(out, want.to(out.dtype)) and not bool(out[mask == 0].any())
        assert not torch.equal(out, unquantised)


@pytest.mark.parametrize("optimizer", ["fused", "torch"])
def test_a_wait_that_gave_up_ends_a_run(optimizer):
    """Training whose kernels have left asks for the status by itself, and evaluation and the optimizer's state do: each raises once, then goes on."""
    from spion_b200 import _lib
    tr, ids, lab = trainer(optimizer=optimizer)
    start(tr, ids, lab)
    tr.step(ids, lab)
    tr.check_device_status()

    def lost():
        _lib.check(_lib.lib.spion_linear_selftest_bounded_wait(1000, torch.cuda.current_stream().cuda_stream))

    def raises(call):
        lost()
        with pytest.raises(_lib.SpionError, match="timed out"):
            call()
        tr.check_device_status()

    raises(tr.check_device_status)
    raises(lambda: tr.evaluate(ids, lab))
    assert tr.model.training
    if optimizer == "fused":
        raises(tr.opt.state_dict)
    assert np.isfinite(float(tr.evaluate(ids, lab)[0]))
    tr.status_every = 3

    def steps(call):
        tr.steps = 0
        call(), call()
        with pytest.raises(_lib.SpionError, match="timed out"):
            call()
        tr.check_device_status()

    lost()
    steps(lambda: tr.step(ids, lab))
    start_again, ids, lab = trainer(optimizer=optimizer)
    start(start_again, ids, lab)
    tr = start_again
    tr.status_every = 3
    tr.capture_sparse_step(ids, lab)
    lost()
    steps(lambda: tr.step_graph(ids, lab))
    assert set(tr.opt.state_dict()["state"][0]) >= {"step", "exp_avg"}


def test_an_evaluation_and_a_state_under_a_capture():
    tr, ids, lab = trainer()
    start(tr, ids, lab)
    want, _ = tr.evaluate(ids, lab)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, _ = tr.evaluate(ids, lab)
        state = tr.opt.state_dict()
    graph.replay()
    assert float(loss) == float(want) and len(state["state"]) == len(tr.bucket.params)
