"""The AdamW step (csrc/adamw.cu) against its formula in fp64: moments in 32 and in 8 bits, types, sizes around blocks and chunks, views off their
boundaries, tensors without a gradient, values that are not finite, captured steps, state dicts.

Bounds, with u = 2^-24: the fp32 constants b1, 1 - b1, ... carry u each, a product u, a sum u.  m: 3 u of its two terms; v: 4 u; the update's quotient
adds both moments' errors, the factors' and its own roundings: 16 u of lr |m| / root with the terms of m in place of m; p: 3 u, and half a step of its type.
8-bit moments: a code is the floor of x / quantum + noise, so it differs from the fp64 one where that sum is within 16 times 8 u of a whole number: in less
than one of 2^15 values, by one quantum."""
import copy

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def half(t):
    return torch.finfo(t).eps / 2


def mix(x):
    x = x.astype(np.uint32)
    with np.errstate(over="ignore"):
        x ^= x >> np.uint32(16)
        x *= np.uint32(0x7FEB352D)
        x ^= x >> np.uint32(15)
        x *= np.uint32(0x846CA68B)
        return x ^ (x >> np.uint32(16))


def noise_of(n, seed, step, index):
    one = lambda v: np.array([v & 0xFFFFFFFF], dtype=np.uint64).astype(np.uint32)      # noqa: E731
    key = mix(one(seed + int(mix(one(step * 0x9E3779B1 + index))[0])))
    return mix(np.arange(n, dtype=np.uint32) ^ mix(key))


def blocks(x):
    out = np.zeros(-(-x.size // 256) * 256)
    out[:x.size] = x
    return out.reshape(-1, 256)


def reference(p, g, m, v, step, index, *, lr, betas, eps, weight_decay, clip_value, seed=0, bits=32):
    """One tensor in fp64: new p, m, v, the scales and the codes' values in units of their scale."""
    b1, b2 = betas
    t = step + 1
    if clip_value is not None:
        g = np.clip(g, -clip_value, clip_value)
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    root = np.sqrt(v1) / np.sqrt(1 - b2 ** t) + eps
    p1 = p * (1 - lr * weight_decay) - lr / (1 - b1 ** t) * m1 / root
    err_m = 3 * U * (np.abs(b1 * m) + np.abs((1 - b1) * g))
    err_p = 3 * U * np.abs(p) + lr / (1 - b1 ** t) / root * (16 * U * (np.abs(b1 * m) + np.abs((1 - b1) * g)) + err_m)
    out = {"p": p1, "m": m1, "v": v1, "err_m": err_m, "err_v": 4 * U * v1, "err_p": err_p}
    if bits == 8:
        r = noise_of(p.size, seed, int(t), index)
        for name, x, low, digits, above, u in (("m", m1, -6, 3, 7, r & np.uint32(0xFFFF)), ("v", v1, -14, 2, 14, r >> np.uint32(16))):
            # (a second moment that is infinite stays so and decides no scale: the largest that an e5m2 holds in the inputs below is 57344 units)
            top = np.maximum(np.where(np.isfinite(blocks(x)), np.abs(blocks(x)), 0).max(1), 2.0 ** -100).astype(np.float32)
            scale = np.ldexp(1.0, np.frexp(top)[1] - 1 - above)
            y = x / np.repeat(scale, 256)[:x.size]
            q = np.ldexp(1.0, np.maximum(np.frexp(y)[1] - 1, low) - digits)
            with np.errstate(invalid="ignore"):
                code = np.where(np.isfinite(y), np.floor(np.abs(y) / q + u / 65536.0) * q * np.sign(y), y)
            if name == "v":
                code = np.where(y > 0, np.maximum(code, 2.0 ** (low - digits)), code)
            out[name + "_scale"], out[name + "_code"], out[name + "_q"] = scale, code, q
    return out


HYPER = dict(lr=2e-3, betas=(0.9, 0.98), eps=1e-8, weight_decay=0.1)


def make(sizes, dtype, bits, seed, offset=0):
    """Parameters and gradients that are views `offset` elements off a boundary, and moments as some steps leave them."""
    from spion_b200.optim import BLOCK, places
    rng = np.random.default_rng(seed)

    def tensor(x):
        buf = torch.zeros(x.size + offset + 8, dtype=dtype, device="cuda")
        buf[offset:offset + x.size] = torch.from_numpy(x).to(dtype=dtype, device="cuda")
        return buf[offset:offset + x.size]

    ps = [tensor(rng.normal(size=n)) for n in sizes]
    gs = [tensor(rng.normal(size=n) * 10.0 ** rng.integers(-3, 1)) for n in sizes]
    at, total = places(ps)
    m, v = np.zeros(total), np.zeros(total)
    for a, n in zip(at, sizes):
        m[a:a + n] = rng.normal(size=n) * 0.1
        v[a:a + n] = np.exp(rng.normal(size=n)) * 0.01
    m, v = torch.from_numpy(m).float().cuda(), torch.from_numpy(v).float().cuda()
    scales = None
    if bits == 8:
        scales = (torch.full((total // BLOCK,), 2.0 ** -9, device="cuda"), torch.full((total // BLOCK,), 2.0 ** -17, device="cuda"))
        m, v = (m * 2.0 ** 9).to(torch.float8_e4m3fn), (v * 2.0 ** 17).to(torch.float8_e5m2)
    return ps, gs, m, v, scales, at


def values(x, scales, block=256):
    x = x.double().cpu().numpy()
    return x if scales is None else (x.reshape(-1, block) * scales.double().cpu().numpy()[:, None]).reshape(-1)


def check_step(sizes, dtype, bits, clip=None, offset=0, none=(), steps_before=3.0, seed=5):
    from spion_b200.optim import adamw_step
    ps, gs, m, v, scales, at = make(sizes, dtype, bits, seed, offset)
    gs = [None if i in none else g for i, g in enumerate(gs)]
    steps = torch.full((len(sizes),), steps_before, device="cuda")
    before = [p.double().cpu().numpy() for p in ps], values(m, scales and scales[0]), values(v, scales and scales[1])
    state_before = m.clone(), v.clone()
    adamw_step(ps, gs, m, v, steps, scales=scales, clip_value=clip, seed=11, **HYPER)
    after_m, after_v = values(m, scales and scales[0]), values(v, scales and scales[1])
    wrong = total = 0
    for i, (n, a) in enumerate(zip(sizes, at)):
        here = slice(a, a + n)
        got = ps[i].double().cpu().numpy()
        if gs[i] is None:
            assert np.array_equal(got, before[0][i]) and float(steps[i]) == steps_before
            assert torch.equal(m[here].float(), state_before[0][here].float()) and torch.equal(v[here].float(), state_before[1][here].float())
            continue
        want = reference(before[0][i], gs[i].double().cpu().numpy(), before[1][here], before[2][here], steps_before, i, clip_value=clip, seed=11, bits=bits, **HYPER)
        assert float(steps[i]) == steps_before + 1
        assert (np.abs(got - want["p"]) <= want["err_p"] + np.abs(want["p"]) * half(dtype) * 1.01 + (2.0 ** -25 if dtype == torch.float16 else 1e-30)).all()
        pad = slice(a + n, a + -(-n // 256) * 256)
        assert not after_m[pad].any() and not after_v[pad].any()
        if bits == 32:
            assert (np.abs(after_m[here] - want["m"]) <= want["err_m"] + 1e-38).all() and (np.abs(after_v[here] - want["v"]) <= want["err_v"] + 1e-38).all()
            continue
        for name, after, sc in (("m", after_m, scales[0]), ("v", after_v, scales[1])):
            b = slice(a // 256, a // 256 + want[name + "_scale"].size)
            # the exponent of a block's largest value: where that is within its error (3 u or 4 u) of a power of two, either side may be taken
            other = sc[b].double().cpu().numpy() != want[name + "_scale"]
            top = np.where(np.isfinite(blocks(want[name])), np.abs(blocks(want[name])), 0).max(1)[other]
            near = 2.0 ** np.round(np.log2(top))
            assert (np.abs(top / near - 1) <= 8 * U).all()
            np.seterr(invalid="ignore")                                   # (infinite beside infinite)
            got = after[here] / np.repeat(want[name + "_scale"], 256)[:n]
            there = np.repeat(other, 256)[:n]
            assert (np.abs(got - want[name][:n] / np.repeat(want[name + "_scale"], 256)[:n])[there] <= 2 * want[name + "_q"][there] * 1.0001).all()
            got[there] = want[name + "_code"][there]
            off = np.abs(np.where(got == want[name + "_code"], 0, got) - np.where(got == want[name + "_code"], 0, want[name + "_code"]))
            assert (off <= want[name + "_q"] * 1.0001).all()
            wrong, total = wrong + int((off > 0).sum()), total + n
    assert wrong <= 4 + total / 2 ** 15


SIZES = [[1], [255, 256, 257], [2048, 2047, 2049, 1], [5, 0, 100003, 64, 7], [300000]]


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_one_step(sizes, bits, dtype):
    check_step(sizes, dtype, bits)


@pytest.mark.parametrize("bits", [32, 8])
def test_clipping_views_tensors_without_a_gradient_and_first_steps(bits):
    check_step([300, 4096, 77], torch.float32, bits, clip=0.05)
    check_step([300, 4096, 77], torch.bfloat16, bits, clip=0.05, offset=1)
    check_step([3000, 40], torch.float32, bits, offset=4)
    check_step([256, 300, 10, 5000], torch.float32, bits, none=(1, 3))
    check_step([300], torch.float32, bits, steps_before=0.0)
    check_step([300], torch.float32, bits, steps_before=100000.0)


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_a_launch_takes(bits):
    rng = np.random.default_rng(3)
    check_step([int(n) for n in rng.integers(0, 700, size=65)], torch.float32, bits)
    check_step([int(n) for n in rng.integers(1, 300, size=1100)], torch.float32, bits, none=tuple(range(3, 1100, 7)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_values(dtype):
    """Enough of them for the kernel that copies ahead: tensors that end inside a chunk, small ones, one without a gradient; and tensors off their boundaries."""
    check_step([6_000_001, 77, 2048, 9_200_000, 0, 5, 70_000], dtype, 8, clip=0.5, none=(6,))
    check_step([14_800_003, 300], dtype, 8, offset=1)


def test_values_that_are_not_finite_stay_where_they_are():
    from spion_b200.optim import adamw_step
    for bits, n in ((32, 1000), (8, 1000), (8, 15_000_000)):
        ps, gs, m, v, scales, _ = make([n], torch.float32, bits, 1)
        v.copy_(torch.where(torch.isfinite(v.float()), v.float(), 1.0).to(v.dtype))
        gs[0][10], gs[0][700] = float("nan"), float("inf")
        for _ in range(2):
            adamw_step(ps, gs, m, v, torch.ones(1, device="cuda"), scales=scales, **HYPER)
        bad = ~torch.isfinite(ps[0])
        assert bad.nonzero().flatten().tolist() == [10, 700]
        got = values(m, scales and scales[0])[:n], values(v, scales and scales[1])[:n]
        for x in got:
            assert np.flatnonzero(~np.isfinite(x)).tolist() == [10, 700]
        # clipped, an infinity is the limit; a NaN stays one
        ps, gs, m, v, scales, _ = make([n], torch.float32, bits, 1)
        v.copy_(torch.where(torch.isfinite(v.float()), v.float(), 1.0).to(v.dtype))
        gs[0][10], gs[0][700] = float("nan"), float("inf")
        adamw_step(ps, gs, m, v, torch.ones(1, device="cuda"), scales=scales, clip_value=1.0, **HYPER)
        assert (~torch.isfinite(ps[0])).nonzero().flatten().tolist() == [10]


def test_eight_bit_moments_follow_on_average():
    """Rounded to nearest, a second moment whose codes are 12 to 25 % apart would never move by 0.1 %.  Rounded at random each step is exact on average: of 65536
    values the mean is off by the deviation of one (at most 12 % after any number of steps, the random walk being pulled back by b2) over 256, four times that is 0.2 %."""
    from spion_b200.optim import adamw_step
    n = 65536
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 0.1, device="cuda")
    m, v = torch.zeros(n, device="cuda").to(torch.float8_e4m3fn), torch.full((n,), 16384.0, device="cuda").to(torch.float8_e5m2)
    scales = torch.ones(n // 256, device="cuda"), torch.full((n // 256,), 2.0 ** -14, device="cuda")
    steps = torch.zeros(1, device="cuda")
    want = 1.0
    for _ in range(300):
        adamw_step([p], [g], m, v, steps, scales=scales, betas=(0.9, 0.999))
        want = 0.999 * want + 0.001 * 0.01
    got = values(v, scales[1])
    assert abs(got.mean() / want - 1) < 0.01 and abs(values(m, scales[0]).mean() / 0.1 - 1) < 0.01
    assert float(steps[0]) == 300


def small_model(dtype=torch.float32):
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(48, 33), torch.nn.ReLU(), torch.nn.Linear(33, 5)).cuda().to(dtype)


def gradients(model, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    for p in model.parameters():
        p.grad = torch.randn(p.shape, generator=g, device="cuda").to(p.dtype)


def test_optimizer_beside_the_frameworks_and_state_dicts():
    from spion_b200.optim import AdamW
    a, b = small_model(), small_model()
    groups = lambda m: [{"params": [m[0].weight, m[2].weight], "weight_decay": 0.1}, {"params": [m[0].bias, m[2].bias], "lr": 1e-2}]      # noqa: E731
    mine, theirs = AdamW(groups(a), lr=1e-3, weight_decay=0.0), torch.optim.AdamW(groups(b), lr=1e-3, weight_decay=0.0)

    def both(first, n):
        for k in range(first, first + n):
            gradients(a, k), gradients(b, k)
            mine.step(), theirs.step()

    def close():
        # ten steps of at most 1e-2 each, every one a few u off its own size
        for x, y in zip(a.parameters(), b.parameters()):
            assert float((x - y).detach().abs().max()) <= 20 * (32 * U * 1e-2 + 4 * U)
    both(0, 5)
    close()
    # each goes on from the other's state
    sa, sb = copy.deepcopy(mine.state_dict()), copy.deepcopy(theirs.state_dict())
    assert set(sa["state"][0]) == set(sb["state"][0]) == {"step", "exp_avg", "exp_avg_sq"}
    mine.load_state_dict(sb)
    theirs.load_state_dict(sa)
    both(5, 5)
    close()
    # a fresh optimizer goes on with the same bits
    fresh = AdamW(groups(c := copy.deepcopy(a)), lr=5.0)
    fresh.load_state_dict(mine.state_dict())
    gradients(a, 99), gradients(c, 99)
    mine.step(), fresh.step()
    assert all(torch.equal(x, y) for x, y in zip(a.parameters(), c.parameters()))


@pytest.mark.parametrize("bits", [32, 8])
def test_state_of_this_optimizer_and_what_it_refuses(bits, tmp_path):
    from spion_b200._lib import SpionError
    from spion_b200.optim import AdamW
    a = small_model()
    opt = AdamW(a.parameters(), state_bits=bits, seed=4)
    for k in range(3):
        gradients(a, k)
        opt.step()
    torch.save(opt.state_dict(), tmp_path / "opt.pt")
    b = copy.deepcopy(a)
    other = AdamW(b.parameters(), state_bits=bits, seed=4)
    other.load_state_dict(torch.load(tmp_path / "opt.pt"))
    both = copy.deepcopy((a, opt))
    for model, o in ((a, opt), (b, other), both):
        gradients(model, 7)
        o.step()
    for x, y, z in zip(a.parameters(), b.parameters(), both[0].parameters()):
        assert torch.equal(x, y) and torch.equal(x, z)
    with pytest.raises(ValueError):
        AdamW(b.parameters(), state_bits=40 - bits).load_state_dict(opt.state_dict())
    with pytest.raises(ValueError):
        AdamW(list(b.parameters())[:2], state_bits=bits).load_state_dict(opt.state_dict())
    opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(3))]})
    with pytest.raises(SpionError, match="GPU"):
        opt.step()
    fresh = AdamW(b.parameters(), state_bits=bits)
    gradients(b, 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x = torch.zeros(4, device="cuda") + 1
        with pytest.raises(SpionError, match="captured"):
            fresh.step()


def test_mixed_types_and_skipped_parameters():
    from spion_b200.optim import AdamW
    ps = [torch.nn.Parameter(torch.randn(100, device="cuda").to(t)) for t in (torch.float32, torch.bfloat16, torch.float32, torch.float16)]
    opt = AdamW(ps, lr=0.1)
    before = [p.detach().clone() for p in ps]
    for p in ps[:2] + ps[3:]:
        p.grad = torch.ones_like(p)
    opt.step()
    assert torch.equal(ps[2], before[2]) and all(not torch.equal(ps[i], before[i]) for i in (0, 1, 3))
    assert float(opt.state[ps[2]]["step"]) == 0 and float(opt.state[ps[3]]["step"]) == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_with_a_rate_on_the_device(bits):
    from spion_b200.optim import AdamW
    a, b = small_model(), small_model()
    lr = torch.tensor(1e-2, device="cuda")
    copies = [torch.empty_like(p, dtype=torch.bfloat16) for p in a.parameters()]
    one, two = AdamW(a.parameters(), lr=lr, state_bits=bits, clip_value=0.5), AdamW(b.parameters(), lr=1e-2, state_bits=bits, clip_value=0.5)
    one.write_copies(a.parameters(), copies)
    gradients(a, 0), gradients(b, 0)
    one.step(), two.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one.step()
    for k, rate in ((1, 1e-2), (2, 3e-2)):
        lr.fill_(rate)
        two.param_groups[0]["lr"] = float(np.float32(rate))
        graph.replay()
        two.step()
    for x, y, c in zip(a.parameters(), b.parameters(), copies):
        assert float((x - y).detach().abs().max()) <= 3 * (U * 1e-1 + 4 * U) and torch.equal(c, x.detach().bfloat16())
    assert float(one.state[next(a.parameters())]["step"]) == 3


def test_what_a_step_refuses():
    from spion_b200._lib import SpionError
    from spion_b200.optim import adamw_step
    ps, gs, m, v, scales, _ = make([300, 40], torch.float32, 32, 0)
    steps = torch.zeros(2, device="cuda")
    state = [t.clone() for t in (*ps, m, v)]

    def refused(match, *args, **kw):
        with pytest.raises(SpionError, match=match):
            adamw_step(*args, **kw)

    refused("gradients", ps, gs[:1], m, v, steps)
    refused("type", ps, [gs[0].half(), gs[1]], m, v, steps)
    refused("shape", ps, [gs[0][:299], gs[1]], m, v, steps)
    refused("contiguous", [ps[0].view(20, 15).t(), ps[1]], [gs[0].view(15, 20), gs[1]], m, v, steps)
    refused("exp_avg", ps, gs, m[:256], v, steps)
    refused("exp_avg_sq", ps, gs, m, v.half(), steps)
    refused("steps", ps, gs, m, v, steps[:1])
    refused("share memory", [ps[0], ps[0][:40]], gs, m, v, steps)
    refused("share memory", ps, gs, m, m, steps)
    refused("exp_avg", ps, gs, m, v, steps, scales=(steps, steps))
    refused("lr", ps, gs, m, v, steps, lr=-1.0)
    refused("betas", ps, gs, m, v, steps, betas=(1.0, 0.9))
    refused("copy", ps, gs, m, v, steps, copies=[None, ps[1].double()])
    refused("two types", ps, gs, m, v, steps, copies=[ps[0].half(), ps[1].bfloat16()])
    refused("CUDA", [p.cpu() for p in ps], gs, m, v, steps)
    refused("not a tensor", [1, 2], gs, m, v, steps)
    refused("clip_value", ps, gs, m, v, steps, clip_value=-1.0)
    assert all(torch.equal(a, b) for a, b in zip(state, (*ps, m, v))) and not steps.any()
    adamw_step([], [], m, v, steps)
    adamw_step(ps, [None, None], m, v, steps)
    assert not steps.any()


def test_gradients_with_other_strides_and_another_stream():
    from spion_b200.optim import adamw_step
    p, g = torch.randn(30, 20, device="cuda"), torch.randn(20, 30, device="cuda").t()
    m, v = torch.zeros(768, device="cuda"), torch.zeros(768, device="cuda")
    q, m2, v2, steps = p.clone(), m.clone(), v.clone(), torch.zeros(2, device="cuda")
    adamw_step([p], [g], m, v, steps[:1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        adamw_step([q], [g.contiguous()], m2, v2, steps[1:])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(p, q) and torch.equal(m, m2) and torch.equal(v, v2)
    # a tensor that a backward has saved is known to have changed
    w = torch.randn(8, device="cuda", requires_grad=True)
    y = (w * w).sum()
    adamw_step([w], [torch.ones(8, device="cuda")], m, v, steps[:1])
    with pytest.raises(RuntimeError, match="modified"):
        y.backward()


def test_steps_follow_the_parameter_groups():
    """A group that leaves or moves takes its moments along; a parameter put in another's place starts anew, as torch's; groups mixed anew are refused."""
    from spion_b200._lib import SpionError
    from spion_b200.optim import AdamW
    tensors = lambda: [torch.nn.Parameter(torch.full((300,), 1.0 + k, device="cuda")) for k in range(3)]      # noqa: E731

    def both(call):
        out = []
        for make in (lambda ps: AdamW([{"params": [p]} for p in ps], lr=1e-2), lambda ps: torch.optim.AdamW([{"params": [p]} for p in ps], lr=1e-2)):
            ps = tensors()
            opt = make(ps)
            for k in range(2):
                for p in ps:
                    p.grad = torch.full_like(p, 0.1 * (k + 1))
                opt.step()
            ps = call(opt, ps)
            for p in ps:
                p.grad = torch.full_like(p, -0.2)
            opt.step()
            out.append([p.detach().clone() for p in ps])
        for a, b in zip(*out):
            assert float((a - b).abs().max()) <= 3 * (32 * U * 1e-2 + 4 * U)

    def removed(opt, ps):
        del opt.param_groups[0]
        return ps

    def reordered(opt, ps):
        opt.param_groups.reverse()
        return ps

    def replaced(opt, ps):
        new = torch.nn.Parameter(torch.full((300,), 7.0, device="cuda"))
        opt.param_groups[1]["params"] = [new]
        return [*ps, new]

    for change in (removed, reordered, replaced):
        both(change)
    ps = tensors()
    opt = AdamW(ps)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    before = [p.detach().clone() for p in ps]
    opt.param_groups[0]["params"] = [ps[0], torch.nn.Parameter(torch.zeros(300, device="cuda")), ps[2]]
    with pytest.raises(SpionError, match="changed"):
        opt.step()
    assert all(torch.equal(p, b) for p, b in zip(ps, before))


@pytest.mark.parametrize("bits", [32, 8])
def test_copies_of_an_optimizer_that_has_a_scheduler(bits):
    """A scheduler puts a step of its own into the optimizer's attributes: a copy has the class's, and steps its own parameters."""
    import pickle

    from spion_b200.optim import AdamW
    a = small_model()
    opt = AdamW(a.parameters(), lr=1e-2, state_bits=bits, seed=2)
    scheduler = torch.optim.lr_scheduler.LambdaLR(opt, lambda k: 1.0)
    gradients(a, 0)
    opt.step()
    scheduler.step()
    copies = [copy.deepcopy((a, opt)), pickle.loads(pickle.dumps((a, opt)))]
    before = [p.detach().clone() for p in a.parameters()]
    for model, o in copies:
        gradients(model, 1)
        o.step()
        assert all(torch.equal(p, b) for p, b in zip(a.parameters(), before))
    gradients(a, 1)
    opt.step()
    want = opt.state_dict()["state"]
    for model, o in copies:
        assert all(torch.equal(p, q) for p, q in zip(a.parameters(), model.parameters()))
        for i, s in o.state_dict()["state"].items():                      # what it keeps is what it steps on
            assert all(torch.equal(s[k].float(), want[i][k].float()) for k in want[i])


def test_hooks_of_loading_a_state():
    from spion_b200.optim import AdamW
    a = small_model()
    opt = AdamW(a.parameters())
    gradients(a, 0)
    opt.step()
    saved, calls = copy.deepcopy(opt.state_dict()), []
    saved["state"][0]["step"] = torch.tensor(5.0)

    def before(o, state):
        calls.append(("before", o is opt))
        return {**state, "state": {**state["state"], 1: {**state["state"][1], "step": torch.tensor(9.0)}}}

    opt.register_load_state_dict_pre_hook(before)
    opt.register_load_state_dict_post_hook(lambda o: calls.append(("after", float(o.state[a[0].weight]["step"]))))
    opt.load_state_dict(saved)
    assert calls == [("before", True), ("after", 5.0)]
    assert float(opt.state[a[0].bias]["step"]) == 9 and float(saved["state"][1]["step"]) == 1


def test_loaded_groups():
    """Whatever a group carries is loaded with it (a scheduler's first rate), in tensors of this optimizer's own."""
    from spion_b200.optim import AdamW
    a, b = small_model(), small_model()
    theirs = torch.optim.AdamW(a.parameters(), lr=torch.tensor(1e-2, device="cuda"), capturable=True)
    torch.optim.lr_scheduler.LambdaLR(theirs, lambda k: 0.5)
    gradients(a, 0)
    theirs.step()
    theirs.param_groups[0]["name"] = "all of them"
    saved = theirs.state_dict()
    mine = AdamW(b.parameters(), clip_value=3.0)
    mine.load_state_dict(saved)
    group = mine.param_groups[0]
    assert group["name"] == "all of them" and float(group["initial_lr"]) == float(saved["param_groups"][0]["initial_lr"]) and group["clip_value"] == 3.0
    assert float(group["lr"]) == float(theirs.param_groups[0]["lr"]) and group["lr"] is not theirs.param_groups[0]["lr"]
    group["lr"].fill_(1.0)
    assert float(theirs.param_groups[0]["lr"]) != 1.0
    assert group["params"] == list(b.parameters())
    torch.optim.lr_scheduler.LambdaLR(mine, lambda k: 0.5, last_epoch=3)   # asks for the first rate


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_states_of_16_bit_parameters(dtype):
    """torch keeps their moments in the parameter's type, this optimizer in fp32: each takes the other's, rounded where it is narrower."""
    from spion_b200.optim import AdamW
    a, b = small_model(dtype), small_model(dtype)
    theirs, mine = torch.optim.AdamW(a.parameters()), AdamW(b.parameters())
    gradients(a, 0)
    theirs.step()
    mine.load_state_dict(copy.deepcopy(theirs.state_dict()))
    for p, q in zip(a.parameters(), b.parameters()):
        for k in ("step", "exp_avg", "exp_avg_sq"):
            x, y = mine.state[q][k], theirs.state[p][k]
            assert x.dtype == torch.float32 and torch.equal(x, y.float().to(x.device))
    gradients(b, 1)
    mine.step()
    theirs.load_state_dict(copy.deepcopy(mine.state_dict()))
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(theirs.state[p]["exp_avg"], mine.state[q]["exp_avg"].to(dtype))
    bad = copy.deepcopy(theirs.state_dict())
    bad["state"][0]["exp_avg"] = bad["state"][0]["exp_avg"].int()
    with pytest.raises(ValueError, match="exp_avg"):
        mine.load_state_dict(bad)


@pytest.mark.parametrize("eps", [0.0, 1e-13, 2.0 ** -40, 1e-12, 2.0 ** -35, 1e-10, 1e-9])
def test_small_eps_beside_small_second_moments(eps):
    """Second moments on both sides of fp32's smallest normal number 2^-126, with the largest correction that b2 = 0.9999 has (100 at the first step): their roots
    are what the update is divided by.  The bound is that of every other step; the numbers below 2^-126 are off by at most 2^-150, a root of 2^-126 and more
    by 2^-25 of itself then, those of 2^-130 by 2^-21."""
    from spion_b200.optim import adamw_step
    n = 4096
    g = np.exp(np.linspace(np.log(3e-18), np.log(1e-15), n))              # v from 2^-130 to 2^-113
    for bits in (32, 8):
        p, d = torch.zeros(n, device="cuda"), torch.from_numpy(g).float().cuda()
        m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
        scales = None
        if bits == 8:
            m, v, scales = m.to(torch.float8_e4m3fn), v.to(torch.float8_e5m2), (torch.ones(n // 256, device="cuda"), torch.ones(n // 256, device="cuda"))
        hyper = dict(lr=1.0, betas=(0.9, 0.9999), eps=eps, weight_decay=0.0, clip_value=None)
        adamw_step([p], [d], m, v, torch.zeros(1, device="cuda"), scales=scales, **hyper)
        want = reference(np.zeros(n), d.double().cpu().numpy(), np.zeros(n), np.zeros(n), 0, 0, **hyper)
        off = np.abs(p.double().cpu().numpy() - want["p"])
        bound = want["err_p"] + np.abs(want["p"]) * np.minimum(2.0 ** -151 / want["v"], 1)
        assert (off <= bound).all(), (off / bound).max()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_nothing_is_written_beside_the_tensors(dtype, bits):
    """Parameters, copies and moments in the middle of other memory, on and off the boundaries of the wide accesses; sizes around blocks and chunks; a tensor without a
    gradient between others: what lies around them, and the places that fill the last block of each, stay."""
    from spion_b200.optim import adamw_step, places
    g = torch.Generator(device="cuda").manual_seed(8)
    for off in (0, 1, 8, 3):
        sizes = [1, 255, 256, 257, 2047, 2048, 2049, 5000, 70001, 3]
        spans, at = [], 64 + off
        for n in sizes:
            spans.append(slice(at, at + n))
            at += n + 16 + (off and 1)
        buf, copy_buf = torch.randn(at + 64, generator=g, device="cuda").to(dtype), torch.randn(at + 64, generator=g, device="cuda").bfloat16()
        was, copy_was = buf.clone(), copy_buf.clone()
        ps, cs = [buf[s] for s in spans], [copy_buf[s] for s in spans]
        gs = [None if i == 5 else torch.randn(n, generator=g, device="cuda").to(dtype) for i, n in enumerate(sizes)]
        cs[2] = None
        begins, total = places(ps)
        m, v = torch.full((total + 512,), 0.5, device="cuda"), torch.full((total + 512,), 0.5, device="cuda")
        scales = None
        if bits == 8:
            m, v = m.to(torch.float8_e4m3fn), v.to(torch.float8_e5m2)
            scales = torch.full((total // 256 + 2,), 0.25, device="cuda"), torch.full((total // 256 + 2,), 0.25, device="cuda")
        kept = [t.clone() for t in (m, v, *(scales or ()))]
        steps = torch.full((len(sizes) + 3,), 4.0, device="cuda")
        adamw_step(ps, gs, m, v, steps, scales=scales, copies=cs, seed=3, **HYPER)
        for i, (s, n, b) in enumerate(zip(spans, sizes, begins)):
            # (a step of lr = 2e-3 is up to half of a bf16's distance from the next one: a few values may all stay)
            assert (n < 4 or torch.equal(buf[s], was[s]) == (i == 5)) and float(steps[i]) == 4 + (i != 5)
            assert torch.equal(copy_buf[s], copy_was[s] if i in (2, 5) else buf[s].bfloat16()) or (dtype == torch.float16 and i not in (2, 5))
            was[s], copy_was[s] = buf[s], copy_buf[s]
            for t, k in zip((m, v), kept):
                k.view(torch.uint8 if bits == 8 else torch.float32)[b:b + n] = t.view(torch.uint8 if bits == 8 else torch.float32)[b:b + n]
            for t, k in zip(scales or (), kept[2:]):
                k[b // 256:(b + n + 255) // 256] = t[b // 256:(b + n + 255) // 256]
        raw = lambda t: t.view(torch.uint8)      # noqa: E731
        assert torch.equal(raw(buf), raw(was)) and torch.equal(raw(copy_buf), raw(copy_was)) and bool((steps[len(sizes):] == 4).all())
        assert all(torch.equal(raw(t), raw(k)) for t, k in zip((m, v, *(scales or ())), kept))
