"""Operators of the encoder around its attention call, as cases to time and compare: the root-mean-square norm with the residual's addition
(forward, backward, output in 8 bits), the linear layer on 8-bit operands, and the AdamW step over many tensors.

``run`` computes each in its plain form (elementary torch operations in fp32); with ``own`` set it calls this framework's operators.
``exact`` is the definition in fp64.  Sizes are the encoder's own (width 64, hidden width 128, sequences of 4096) and generic ones.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
SMALL = 2.0 ** -100                # smallest largest-value that a row's or a block's scale follows
BLOCK = 256                        # values of a tensor that share one scale in 8-bit optimizer states


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token of a decoder of width 4096, on its way into an 8-bit projection: latency
        {"name": "norm8_token", "op": "norm8", "rows": 1, "width": 4096, "stream": "bf16", "branch": "bf16"},
        # a batch of prompts before the 8-bit projections
        {"name": "norm8_prompts", "op": "norm8", "rows": 32768, "width": 2048, "stream": "bf16", "branch": "bf16"},
        # both directions of a norm of the encoder's training step: 16 pairs of sequences of 4096, fp32 stream, bf16 branches
        {"name": "norm_encoder_step", "op": "norm", "rows": 131072, "width": 64, "stream": "fp32", "branch": "bf16", "out": "bf16"},
        # the same in a wide model that keeps everything in bf16
        {"name": "norm_wide_step", "op": "norm", "rows": 8192, "width": 4096, "stream": "bf16", "branch": "bf16", "out": "bf16"},
        # a width that is no multiple of anything, without a residual
        {"name": "norm_odd_step", "op": "norm", "rows": 4099, "width": 769, "stream": "fp32", "branch": "none", "out": "fp16"},
        # one token through a projection: the weights are what has to be read
        {"name": "linear_token", "op": "linear", "rows": 1, "inner": 4096, "outer": 4096, "input": "rows8", "bias": True, "out": "bf16"},
        # the first layer of the encoder's feed-forward block on bf16 activations, which the call quantises
        {"name": "linear_encoder", "op": "linear", "rows": 131072, "inner": 64, "outer": 128, "input": "bf16", "bias": True, "out": "bf16"},
        # prompts through a wide projection: a large product
        {"name": "linear_prompts", "op": "linear", "rows": 8192, "inner": 4096, "outer": 4096, "input": "rows8", "bias": False, "out": "bf16"},
        # odd sizes, result in fp32 (a head)
        {"name": "linear_odd", "op": "linear", "rows": 777, "inner": 1000, "outer": 333, "input": "fp32", "bias": True, "out": "fp32"},
        # the optimizer of the two-layer encoder at 4096 positions, 32-bit states: many small tensors
        {"name": "adamw_encoder", "op": "adamw", "width": 64, "hidden": 128, "layers": 2, "vocab": 256, "positions": 4096, "extra": 0, "bits": 32,
         "param": "fp32", "clip": True, "weight_decay": 0.0},
        # a larger model of two wide layers with its embedding, 8-bit states
        {"name": "adamw_wide_8bit", "op": "adamw", "width": 1024, "hidden": 4096, "layers": 3, "vocab": 32000, "positions": 4096, "extra": 0, "bits": 8,
         "param": "fp32", "clip": False, "weight_decay": 0.01},
        # odd widths: tensors that end inside a block of states
        {"name": "adamw_odd_8bit", "op": "adamw", "width": 77, "hidden": 301, "layers": 2, "vocab": 1009, "positions": 0, "extra": 1000003, "bits": 8,
         "param": "fp32", "clip": True, "weight_decay": 0.1},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm8", "norm", "norm", "linear", "linear", "adamw", "adamw"])
    if op in ("norm8", "norm"):
        width = _log(rng, 16, 16384)
        if rng.random() < 0.6:
            width = -(-width // 16) * 16
        rows = _log(rng, 1, max(1, min(131072, (1 << 25) // width)))
        stream = rng.choice(["fp32", "bf16", "fp16"])
        branch = rng.choice(["none", stream, "bf16" if stream == "fp32" else stream])
        case = {"op": op, "rows": rows, "width": width, "stream": stream, "branch": branch}
        if op == "norm":
            case["out"] = rng.choice(["fp32", "bf16", "fp16"]) if stream == "fp32" else stream
        return case
    if op == "linear":
        inner, outer = _log(rng, 16, 4096), _log(rng, 8, 4096)
        if rng.random() < 0.6:
            inner, outer = -(-inner // 16) * 16, -(-outer // 8) * 8
        return {"op": op, "rows": _log(rng, 1, 8192), "inner": inner, "outer": outer, "input": rng.choice(["rows8", "bf16", "fp16", "fp32"]),
                "bias": rng.random() < 0.5, "out": rng.choice(["bf16", "fp16", "fp32"])}
    return {"op": op, "width": _log(rng, 16, 768), "hidden": _log(rng, 32, 2000), "layers": rng.randint(1, 3), "vocab": _log(rng, 64, 16000),
            "positions": rng.choice([0, 512, 1024, 4096]), "extra": _log(rng, 1, 4000000), "bits": rng.choice([8, 32]),
            "param": rng.choice(["fp32", "fp32", "bf16", "fp16"]), "clip": rng.random() < 0.5, "weight_decay": rng.choice([0.0, 0.01, 0.1])}


def _tensor_shapes(c):
    """The parameters of an encoder: embeddings, then norms, attention and feed-forward block of each layer, then one more tensor."""
    w, h = c["width"], c["hidden"]
    layer = [(w,), (w, w), (w,), (w, w), (w,), (w, w), (w,), (w, w), (w,), (w,), (h, w), (h,), (w, h), (w,)]
    shapes = [(c["vocab"], w)] + ([(c["positions"], w)] if c["positions"] else []) + layer * c["layers"] + [(w,)]
    return shapes + ([(c["extra"],)] if c["extra"] else [])


def _padded(n):
    return -(-n // BLOCK) * BLOCK


def work(c):
    if c["op"] in ("norm8", "norm"):
        n, size = c["rows"] * c["width"], {"fp32": 4, "bf16": 2, "fp16": 2, "none": 0}
        x, r = size[c["stream"]], size[c["branch"]]
        s = x if r else 0                                              # the sum is an output where there is a residual
        if c["op"] == "norm8":
            return {"bytes": n * (x + r + s + 1) + 4 * c["rows"] + 4 * c["width"], "flops": 6 * n}
        y = size[c["out"]]
        own_branch_gradient = r if r != x else 0
        forward = x + r + s + y
        backward = x + y + (x if r else 0) + x + own_branch_gradient   # the sum, both gradients that arrive, those that leave
        return {"bytes": n * (forward + backward) + 8 * c["rows"] + 12 * c["width"], "flops": 16 * n}
    if c["op"] == "linear":
        t, k, n = c["rows"], c["inner"], c["outer"]
        a = {"rows8": 1, "bf16": 2, "fp16": 2, "fp32": 4}[c["input"]]
        scales = 4 * t if c["input"] == "rows8" else 0
        return {"bytes": t * k * a + scales + n * k + 4 * n * (2 if c["bias"] else 1) + t * n * (4 if c["out"] == "fp32" else 2), "flops": 2 * t * n * k}
    n = sum(math.prod(s) for s in _tensor_shapes(c))
    e = 4 if c["param"] == "fp32" else 2
    state = 16 if c["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": int(n * (3 * e + state)), "flops": 15 * n}


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _activations(rows, width, g):
    """Rows of a residual stream: of unequal size, a few features much larger than the others."""
    x = torch.randn(rows, width, generator=g, device="cuda")
    x *= torch.exp(0.7 * torch.randn(rows, 1, generator=g, device="cuda"))
    x *= torch.exp(0.5 * torch.randn(1, width, generator=g, device="cuda"))
    return x + 0.1


def _rows8(x):
    """Rows in e4m3 with a scale each, in a buffer whose rows start on 16 bytes (what both sides are given: a layer's weights, a norm's output)."""
    a = x.abs().amax(1, keepdim=True).clamp_min(SMALL)
    buf = torch.zeros(x.shape[0], -(-x.shape[1] // 16) * 16, dtype=torch.float8_e4m3fn, device="cuda")
    buf[:, :x.shape[1]] = (x * (448.0 / a)).to(torch.float8_e4m3fn)
    return buf[:, :x.shape[1]], (a / 448.0).squeeze(1)


def prepare(c, seed):
    g = _generator(seed)
    s = {"case": c}
    if c["op"] in ("norm8", "norm"):
        rows, width, dt = c["rows"], c["width"], DTYPES[c["stream"]]
        train = c["op"] == "norm"
        s["x"] = _activations(rows, width, g).to(dt).requires_grad_(train)
        s["w"] = (1 + 0.2 * torch.randn(width, generator=g, device="cuda")).requires_grad_(train)
        s["r"] = None
        if c["branch"] != "none":
            s["r"] = torch.randn(rows, width, generator=g, device="cuda").to(DTYPES[c["branch"]]).requires_grad_(train)
        if train:
            s["dy"] = (torch.randn(rows, width, generator=g, device="cuda") * 1e-2).to(DTYPES[c["out"]])
            s["ds"] = (torch.randn(rows, width, generator=g, device="cuda") * 1e-2).to(dt) if s["r"] is not None else None
        return s
    if c["op"] == "linear":
        x = _activations(c["rows"], c["inner"], g)
        s["x"] = _rows8(x) if c["input"] == "rows8" else x.to(DTYPES[c["input"]])
        s["w"] = _rows8(torch.randn(c["outer"], c["inner"], generator=g, device="cuda") / math.sqrt(c["inner"]))
        s["b"] = torch.randn(c["outer"], generator=g, device="cuda") * 0.1 if c["bias"] else None
        return s
    shapes, dt = _tensor_shapes(c), DTYPES[c["param"]]
    s["p"], s["g"] = [], []
    for i, shape in enumerate(shapes):
        s["p"].append((0.05 * torch.randn(shape, generator=g, device="cuda")).to(dt))
        size = 10.0 ** (-2 - i % 3)                                    # gradients of unequal size, some entries far larger
        s["g"].append((size * torch.randn(shape, generator=g, device="cuda") * torch.exp(torch.randn(shape, generator=g, device="cuda"))).to(dt))
    total = sum(_padded(p.numel()) for p in s["p"])
    m, r = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
    at = 0
    for i, p in enumerate(s["p"]):
        n, size = p.numel(), 10.0 ** (-2 - i % 3)
        m[at:at + n] = 0.3 * size * torch.randn(n, generator=g, device="cuda")
        r[at:at + n] = size * torch.exp(0.5 * torch.randn(n, generator=g, device="cuda"))
        at += _padded(n)
    v = r * r
    s["scales"] = None
    if c["bits"] == 8:
        sm = torch.exp2(torch.floor(torch.log2(m.view(-1, BLOCK).abs().amax(1).clamp_min(SMALL))) - 7)
        sv = torch.exp2(torch.floor(torch.log2(v.view(-1, BLOCK).amax(1).clamp_min(SMALL))) - 14)
        m = (m.view(-1, BLOCK) / sm[:, None]).to(torch.float8_e4m3fn).view(-1)
        v = (v.view(-1, BLOCK) / sv[:, None]).to(torch.float8_e5m2).view(-1)
        s["scales"] = (sm, sv)
    s["m"], s["v"] = m, v
    s["steps"] = torch.full((len(shapes),), 100.0, device="cuda")
    s["hyper"] = {"lr": 1e-3, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": c["weight_decay"], "clip_value": 0.05 if c["clip"] else None,
                  "seed": seed & 0x7FFFFFFF}
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    op = s["case"]["op"]
    if op == "norm8":
        return _norm8_own(s) if own else _norm8_plain(s)
    if op == "norm":
        return _norm_own(s) if own else _norm_plain(s)
    if op == "linear":
        return _linear_own(s) if own else _linear_plain(s)
    return _adamw_own(s) if own else _adamw_plain(s)


def _norm8_own(s):
    from spion_b200.rmsnorm import rms_norm_e4m3
    out = rms_norm_e4m3(s["x"], s["w"], EPS, res=s["r"])
    rows = out if s["r"] is None else out[1]
    return {"values": rows.values, "scales": rows.scales, "sum": None if s["r"] is None else out[0]}


def _norm_own(s):
    from spion_b200.rmsnorm import rms_norm
    dt = DTYPES[s["case"]["out"]]
    if s["r"] is None:
        y = rms_norm(s["x"], s["w"], EPS, out_dtype=dt)
        dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
        return {"y": y, "dx": dx, "dw": dw}
    t, y = rms_norm(s["x"], s["w"], EPS, res=s["r"], out_dtype=dt)
    dx, dw, dr = torch.autograd.grad((t, y), (s["x"], s["w"], s["r"]), (s["ds"], s["dy"]))
    return {"y": y, "sum": t, "dx": dx, "dw": dw, "dr": dr}


def _linear_own(s):
    from spion_b200.quant import Rows8, linear_e4m3
    x = Rows8(*s["x"]) if s["case"]["input"] == "rows8" else s["x"]
    return linear_e4m3(x, Rows8(*s["w"]), s["b"], out_dtype=DTYPES[s["case"]["out"]])


def _adamw_own(s):
    from spion_b200.optim import adamw_step
    adamw_step(s["p"], s["g"], s["m"], s["v"], s["steps"], scales=s["scales"], **s["hyper"])
    return _adamw_outputs(s)


def _adamw_outputs(s):
    out = {"p": s["p"], "m": s["m"], "v": s["v"], "steps": s["steps"]}
    if s["scales"] is not None:
        out["m_scales"], out["v_scales"] = s["scales"]
    return out


# ------------------------------------------------------------------------------------------------ plain forms
def _sum_plain(s):
    x = s["x"].detach().float()
    return x if s["r"] is None else (x + s["r"].detach().float()).to(s["x"].dtype).float()


def _norm8_plain(s):
    t = _sum_plain(s)
    y = t / torch.sqrt((t * t).mean(1, keepdim=True) + EPS) * s["w"]
    a = y.abs().amax(1, keepdim=True).clamp_min(SMALL)
    return {"values": (y * (448.0 / a)).to(torch.float8_e4m3fn), "scales": (a / 448.0).squeeze(1),
            "sum": None if s["r"] is None else t.to(s["x"].dtype)}


def _norm_plain(s):
    t, w, dt = _sum_plain(s), s["w"].detach(), s["x"].dtype
    rho = 1 / torch.sqrt((t * t).mean(1, keepdim=True) + EPS)
    n, dy = t * rho, s["dy"].float()
    dn = dy * w
    dx = rho * (dn - n * (dn * n).mean(1, keepdim=True))
    out = {"y": (n * w).to(s["dy"].dtype), "dw": (dy * n).sum(0)}
    if s["r"] is None:
        return out | {"dx": dx.to(dt)}
    dx = dx + s["ds"].float()
    return out | {"sum": t.to(dt), "dx": dx.to(dt), "dr": dx.to(s["r"].dtype)}


def _linear_plain(s):
    x, dt = s["x"], DTYPES[s["case"]["out"]]
    if s["case"]["input"] != "rows8":
        a = x.float().abs().amax(1, keepdim=True).clamp_min(SMALL)
        x = ((x.float() * (448.0 / a)).to(torch.float8_e4m3fn), (a / 448.0).squeeze(1))
    y = (x[0].float() @ s["w"][0].float().t()) * x[1][:, None] * s["w"][1]
    return (y if s["b"] is None else y + s["b"]).to(dt)


def _mix(x):
    """A 32-bit integer hash (two rounds of xor-shift and multiply), on Python numbers or int64 tensors."""
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _key(seed, step, tensor):
    return _mix((seed + _mix((step * 0x9E3779B1 + tensor) & 0xFFFFFFFF)) & 0xFFFFFFFF)


def _to_codes(x, noise, top, bias, mantissa):
    """Values in units of their scale -> codes of an 8-bit float with this exponent bias and these mantissa bits, rounded up with the
    probability that the noise gives: below the last mantissa bit an fp32 number times 2^(bias - 127) has the code's own exponent."""
    drop = 23 - mantissa
    bits = (x.abs() * 2.0 ** (bias - 127)).view(torch.int32).to(torch.int64)
    code = (bits + (noise << (drop - 16))) >> drop
    code = torch.where(torch.isfinite(x), code, torch.where(torch.isnan(x), 0x7F, top))
    return code + torch.where(x < 0, 128, 0)


def _blocks(xs):
    """The tensors one after another, each padded to whole blocks: [blocks, 256]"""
    return torch.cat([torch.nn.functional.pad(x.reshape(-1), (0, _padded(x.numel()) - x.numel())) for x in xs]).view(-1, BLOCK).float()


def _exponent_scale(x, below):
    """2^(exponent of each block's largest finite value - below)"""
    a = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(1, keepdim=True).clamp_min(SMALL)
    return torch.exp2((a.view(torch.int32) >> 23).float() - 127 - below)


def _adamw_plain(s):
    h, (b1, b2) = s["hyper"], s["hyper"]["betas"]
    sizes = [p.numel() for p in s["p"]]
    counts = torch.tensor([_padded(n) // BLOCK for n in sizes])
    tensor = torch.repeat_interleave(torch.arange(len(sizes)), counts).pin_memory().to("cuda", non_blocking=True)       # of each block
    first = (torch.cumsum(counts, 0) - counts).pin_memory().to("cuda", non_blocking=True)[tensor]
    t = s["steps"][tensor].double()[:, None] + 1
    p, g = _blocks(s["p"]), _blocks(s["g"])
    if h["clip_value"] is not None:
        g = g.clamp(-h["clip_value"], h["clip_value"])
    m, v = s["m"].view(-1, BLOCK).float(), s["v"].view(-1, BLOCK).float()
    if s["scales"]:
        m, v = m * s["scales"][0][:, None], v * s["scales"][1][:, None]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    root = torch.sqrt(v) * (1 / torch.sqrt(1 - b2 ** t)).float() + h["eps"]
    p = p * (1 - h["lr"] * h["weight_decay"]) - (h["lr"] / (1 - b1 ** t)).float() * (m / root)
    [x.view(-1).copy_(y[:n]) for x, y, n in zip(s["p"], p.view(-1).split([_padded(n) for n in sizes]), sizes)]
    if s["scales"]:
        i = (torch.arange(len(tensor), device="cuda") - first)[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")       # in its tensor
        noise = _mix((i & 0xFFFFFFFF) ^ _mix(_key(h["seed"], t.long(), tensor[:, None]) + (i >> 32) & 0xFFFFFFFF))
        sm, sv = _exponent_scale(m, 7), _exponent_scale(v, 14)
        cm = _to_codes(m / sm, noise & 0xFFFF, 0x7F, 7, 3)
        cv = _to_codes(v / sv, noise >> 16, 0x7C, 15, 2)
        cv = torch.where(v > 0, cv.clamp_min(1), cv)                   # never zero beside a first moment that is not
        s["m"].view(torch.uint8).copy_(torch.where(m != 0, cm, 0).view(-1))       # (what pads a tensor's last block stays zero)
        s["v"].view(torch.uint8).copy_(torch.where(v != 0, cv, 0).view(-1))
        s["scales"][0].copy_(sm.view(-1))
        s["scales"][1].copy_(sv.view(-1))
    else:
        s["m"].copy_(m.view(-1))
        s["v"].copy_(v.view(-1))
    s["steps"] += 1
    return _adamw_outputs(s)


# ------------------------------------------------------------------------------------------------ the definitions in fp64
def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] in ("norm8", "norm"):
        return _norm_exact(s)
    if c["op"] == "linear":
        x = s["x"]
        if c["input"] != "rows8":
            top = torch.clamp(x.double().abs().max(1).values, min=SMALL).float()
            x = ((x.float() * (448.0 / top)[:, None]).to(torch.float8_e4m3fn), (top.double() / 448).float())   # the roundings that define the operands
        product = torch.einsum("tk,nk->tn", x[0].double() * x[1].double()[:, None], s["w"][0].double() * s["w"][1].double()[:, None])
        return product if s["b"] is None else product + s["b"].double()
    return _adamw_exact(s)


def _norm_exact(s):
    t = s["x"].detach().double()
    added = None
    if s["r"] is not None:
        added = t + s["r"].detach().double()
        t = added.to(s["x"].dtype).double()                            # the norm is that of the sum as it is kept
    width, w = t.shape[1], s["w"].detach().double()
    power = torch.einsum("tc,tc->t", t, t) / width + EPS
    y = t * w / power.sqrt()[:, None]
    if s["case"]["op"] == "norm8":
        top = torch.clamp(y.abs().max(1).values, min=SMALL)
        return {"values": y * (448 / top)[:, None], "scales": top / 448, "sum": added}
    dy = s["dy"].double()
    dw = torch.einsum("tc,tc,t->c", dy, t, power.rsqrt())
    # d/dt_j sum_c dy_c w_c t_c power^(-1/2)
    along = torch.einsum("tc,c,tc->t", dy, w, t)
    dx = dy * w / power.sqrt()[:, None] - t * (along / (width * power.pow(1.5)))[:, None]
    if s["r"] is None:
        return {"y": y, "dx": dx, "dw": dw}
    dx = dx + s["ds"].double()
    return {"y": y, "sum": added, "dx": dx, "dw": dw, "dr": dx}


def _adamw_exact(s):
    h, c = s["hyper"], s["case"]
    beta1, beta2 = h["betas"]
    out = {"p": [], "m": [], "v": [], "steps": s["steps"].double() + 1, "m_scales": [], "v_scales": []}
    begin = 0
    for i, p in enumerate(s["p"]):
        n, t = p.numel(), int(s["steps"][i]) + 1
        end = begin + -(-n // 256) * 256
        grad = s["g"][i].flatten().double()
        if h["clip_value"] is not None:
            grad = torch.minimum(torch.maximum(grad, torch.tensor(-h["clip_value"], device="cuda")), torch.tensor(h["clip_value"], device="cuda"))
        mean, square = s["m"][begin:end].double(), s["v"][begin:end].double()
        if c["bits"] == 8:
            mean = (mean.reshape(-1, 256).T * s["scales"][0][begin // 256:end // 256].double()).T.reshape(-1)
            square = (square.reshape(-1, 256).T * s["scales"][1][begin // 256:end // 256].double()).T.reshape(-1)
        mean[:n] += (1 - beta1) * (grad - mean[:n])
        square[:n] += (1 - beta2) * (grad ** 2 - square[:n])
        step = h["lr"] * (mean[:n] / (1 - beta1 ** t)) / ((square[:n] / (1 - beta2 ** t)).sqrt() + h["eps"])
        out["p"].append((p.flatten().double() * (1 - h["lr"] * h["weight_decay"]) - step).view(p.shape))
        if c["bits"] == 8:
            random = _mix(torch.arange(n, device="cuda") ^ _mix(_key(h["seed"], t, i)))
            for name, x, lowest, digits, above, u in (("m", mean, -6, 3, 7, random % 65536), ("v", square, -14, 2, 14, random // 65536)):
                largest = x.reshape(-1, 256).abs().max(1).values.clamp(min=SMALL).float()      # the exponent is that of the fp32 value
                unit = torch.ldexp(torch.ones_like(largest, dtype=torch.float64), torch.frexp(largest).exponent - 1 - above)
                x = (x.reshape(-1, 256) / unit[:, None]).reshape(-1)[:n]
                quantum = torch.ldexp(torch.ones_like(x), (torch.frexp(x).exponent - 1).clamp(min=lowest) - digits)
                code = torch.floor(x.abs() / quantum + u / 65536.0) * quantum * torch.sign(x)
                if name == "v":
                    code = torch.where(x > 0, torch.clamp(code, min=2.0 ** (lowest - digits)), code)
                out[name].append(torch.nn.functional.pad(code, (0, end - begin - n)))
                out[name + "_scales"].append(unit)
        else:
            out["m"].append(mean)
            out["v"].append(square)
        begin = end
    out = {k: x if k in ("p", "steps") else torch.cat(x) if x else None for k, x in out.items()}
    return out if c["bits"] == 8 else {k: out[k] for k in ("p", "m", "v", "steps")}
