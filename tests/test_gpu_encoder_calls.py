"""Calls of the encoder's operators that are allowed and unusual: a process's first calls inside a capture, recomputed segments and hooks on saved tensors, calls on
two streams at once, inference mode, tracing and transforms (refused)."""
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

FIRST = """
import torch
from spion_b200 import _lib
from spion_b200.optim import adamw_step
from spion_b200.quant import linear_e4m3, quantize_rows
from spion_b200.rmsnorm import rms_norm
torch.zeros(1, device="cuda")
shapes = ((5, 64, 128), (8192, 1024, 1024), (40000, 64, 128), (300, 512, 96))
xs = [torch.randn(T, K, device="cuda", requires_grad=True) for T, K, N in shapes] + [torch.randn(600, 2048, device="cuda", requires_grad=True)]
ws = [torch.randn(N, K, device="cuda") for T, K, N in shapes]
g = torch.ones(2048, device="cuda", requires_grad=True)
p, d = torch.randn(16_000_000, device="cuda"), torch.randn(16_000_000, device="cuda")
m, v = torch.zeros(16_000_000, device="cuda").to(torch.float8_e4m3fn), torch.zeros(16_000_000, device="cuda").to(torch.float8_e5m2)
scales, steps = (torch.ones(62500, device="cuda"), torch.ones(62500, device="cuda")), torch.zeros(1, device="cuda")
dy = torch.randn(600, 2048, device="cuda")

def all_of_them():
    out = [linear_e4m3(x.detach(), quantize_rows(w), out_dtype=torch.bfloat16) for x, w in zip(xs, ws)]
    y = rms_norm(xs[-1], g)
    out += [y.detach(), *torch.autograd.grad(y, (xs[-1], g), dy)]
    adamw_step([p], [d], m, v, steps, scales=scales)
    return out

graph = torch.cuda.CUDAGraph()
start = p.clone()
with torch.cuda.graph(graph):
    got = all_of_them()
graph.replay()
torch.cuda.synchronize()
p_graph = p.clone()
p.copy_(start)
m.view(torch.uint8).zero_(); v.view(torch.uint8).zero_(); steps.zero_()
scales[0].fill_(1); scales[1].fill_(1)
for a, b in zip(got, all_of_them()):
    assert torch.equal(a, b)
assert torch.equal(p, p_graph) and not torch.equal(p, start)
_lib.check(_lib.lib.spion_linear_status(0))
print("same")
"""


def test_first_calls_of_a_process_inside_a_capture():
    r = subprocess.run([sys.executable, "-c", FIRST], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def test_recomputed_segments_and_hooks_on_saved_tensors():
    from torch.utils.checkpoint import checkpoint

    from spion_b200.rmsnorm import rms_norm
    x, r = torch.randn(50, 192, device="cuda", requires_grad=True), torch.randn(50, 192, device="cuda", requires_grad=True)
    w = torch.randn(192, device="cuda", requires_grad=True)

    def f(x, r, w):
        s, y = rms_norm(x, w, res=r)
        return s * 0.5 + rms_norm(y, w)

    want = torch.autograd.grad(f(x, r, w).square().sum(), (x, r, w))
    got = torch.autograd.grad(checkpoint(f, x, r, w, use_reentrant=False).square().sum(), (x, r, w))
    with torch.autograd.graph.save_on_cpu():
        loss = f(x, r, w).square().sum()
    hooked = torch.autograd.grad(loss, (x, r, w))
    for a, b, c in zip(want, got, hooked):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_the_same_tensor_as_stream_and_residual():
    from spion_b200.rmsnorm import rms_norm
    for dtype in (torch.float32, torch.bfloat16):
        x, w = torch.randn(30, 128, device="cuda", dtype=dtype, requires_grad=True), torch.ones(128, device="cuda", requires_grad=True)
        z = x.detach().clone().requires_grad_()
        s, y = rms_norm(x, w, res=x)
        t, u = rms_norm(z, w, res=z.detach())
        assert torch.equal(s, t) and torch.equal(y, u)
        ds, dy = torch.randn_like(s), torch.randn_like(y)
        one, = torch.autograd.grad((t, u), z, (ds, dy))
        both, = torch.autograd.grad((s, y), x, (ds, dy))
        assert torch.equal(both, one + one)


def test_two_streams_at_once():
    from spion_b200.optim import adamw_step
    from spion_b200.quant import linear_e4m3, quantize_rows
    from spion_b200.rmsnorm import rms_norm
    x = torch.randn(8192, 1024, device="cuda")
    q, w, g = quantize_rows(x), quantize_rows(torch.randn(2048, 1024, device="cuda")), torch.ones(1024, device="cuda")
    n = 16_000_000

    def state():
        return (torch.ones(n, device="cuda"), torch.full((n,), 0.5, device="cuda"), torch.zeros(-(-n // 256) * 256, device="cuda"),
                torch.zeros(-(-n // 256) * 256, device="cuda"), torch.zeros(1, device="cuda"))

    want_y, want_n = linear_e4m3(q, w), rms_norm(x, g)
    states = [state() for _ in range(3)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k] += [linear_e4m3(q, w), rms_norm(x, g)]
                p, d, m, v, steps = states[k]
                adamw_step([p], [d], m, v, steps)
    torch.cuda.synchronize()
    p, d, m, v, steps = states[2]
    for _ in range(5):
        adamw_step([p], [d], m, v, steps)
    for k in range(2):
        for i, t in enumerate(got[k]):
            assert torch.equal(t, want_n if i % 2 else want_y)
        assert torch.equal(states[k][0], p) and float(states[k][4]) == 5


def test_inference_mode_and_what_is_refused():
    from spion_b200._lib import SpionError
    from spion_b200.quant import quantize_rows
    from spion_b200.rmsnorm import rms_norm, rms_norm_e4m3
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    with torch.inference_mode():
        a, b = rms_norm(x, w), rms_norm_e4m3(x.clone(), w)
    assert torch.equal(a, rms_norm(x, w)) and b.scales.shape == (4,)

    def refused(call, match):
        with pytest.raises(SpionError, match=match):
            call()

    refused(lambda: torch.func.vmap(lambda t: rms_norm(t, w))(x), "ordinary")
    refused(lambda: torch.jit.trace(lambda t: rms_norm(t, w), (x,)), "ordinary")
    refused(lambda: rms_norm_e4m3(x.clone().requires_grad_(), w), "gradient")
    refused(lambda: rms_norm(x, w[:32]), "weight")
    refused(lambda: rms_norm(x, w.double()), "weight")
    refused(lambda: rms_norm(x.double(), w), "type")
    refused(lambda: rms_norm(x, w, res=x[:2]), "res")
    refused(lambda: rms_norm(x.half(), w, res=x), "res")
    refused(lambda: rms_norm(x.half(), w, out_dtype=torch.float32), "output")
    refused(lambda: rms_norm(x, w.cpu()), "CUDA")
    refused(lambda: quantize_rows(x.to(torch.float8_e4m3fn)), "type")
    refused(lambda: quantize_rows(torch.tensor(1.0, device="cuda")), "shape")
    refused(lambda: quantize_rows(torch.empty(3, 0, device="cuda")), "shape")
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        refused(lambda: rms_norm(dual, w), "ordinary")


def test_the_rings_on_two_streams_at_once():
    """The norm's backward that copies its rows ahead, and the optimizer on many 8-bit moments."""
    from spion_b200.optim import adamw_step
    from spion_b200.rmsnorm import rms_norm
    x, g = torch.randn(4096, 2048, device="cuda", requires_grad=True), torch.rand(2048, device="cuda", requires_grad=True)
    dy, n = torch.randn(4096, 2048, device="cuda"), 16_000_000
    start, d = torch.randn(n, device="cuda"), torch.randn(n, device="cuda")

    def state():
        return (start.clone(), torch.zeros(n, device="cuda").to(torch.float8_e4m3fn), torch.zeros(n, device="cuda").to(torch.float8_e5m2),
                (torch.ones(n // 256, device="cuda"), torch.ones(n // 256, device="cuda")), torch.zeros(1, device="cuda"))

    def step(s):
        adamw_step([s[0]], [d], s[1], s[2], s[4], scales=s[3])

    want = torch.autograd.grad(rms_norm(x, g), (x, g), dy)
    states, streams, got = [state() for _ in range(3)], [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for _ in range(4):
        for s, stream in zip(states, streams):
            with torch.cuda.stream(stream):
                step(s)
                got.append(torch.autograd.grad(rms_norm(x, g), (x, g), dy))
    torch.cuda.synchronize()
    for _ in range(4):
        step(states[2])
    for pair in got:
        assert all(torch.equal(a, b) for a, b in zip(pair, want))
    p, m, v, scales, _ = states[2]
    for q, m1, v1, scales1, steps in states[:2]:
        assert torch.equal(p, q) and torch.equal(m.view(torch.uint8), m1.view(torch.uint8)) and torch.equal(v.view(torch.uint8), v1.view(torch.uint8))
        assert all(torch.equal(a, b) for a, b in zip(scales, scales1)) and float(steps) == 4


def test_a_wait_that_gave_up_leaves_nothing_half_done():
    """The words that a bounded wait sets are set by the self-test of a short one.  Until they have been reported the optimizer leaves parameters, moments and counts
    as they are and the 8-bit linear layer returns; after that all is as before."""
    from spion_b200 import _lib
    from spion_b200.optim import adamw_step
    from spion_b200.quant import linear_e4m3, quantize_rows
    g = torch.Generator(device="cuda").manual_seed(2)

    def moments(n, bits):
        at = -(-n // 256) * 256
        m, v = torch.zeros(at, device="cuda"), torch.zeros(at, device="cuda")
        if bits == 32:
            return [m, v], None
        return [m.to(torch.float8_e4m3fn), v.to(torch.float8_e5m2)], (torch.ones(at // 256, device="cuda"), torch.ones(at // 256, device="cuda"))

    cases = []
    for n, bits in ((16_000_001, 8), (5000, 8), (5000, 32)):
        p, d = torch.randn(n, generator=g, device="cuda"), torch.randn(n, generator=g, device="cuda")
        cases.append((p, d, *moments(n, bits), torch.zeros(1, device="cuda")))

    def step():
        for p, d, (m, v), scales, steps in cases:
            adamw_step([p], [d], m, v, steps, scales=scales)

    def state():
        torch.cuda.synchronize()
        return [t.clone().view(torch.uint8) for p, _, (m, v), scales, steps in cases for t in (p, m, v, steps, *(scales or ()))]

    operands = [(quantize_rows(torch.randn(T, 512, generator=g, device="cuda")), quantize_rows(torch.randn(N, 512, generator=g, device="cuda")))
                for T, N in ((4, 100), (700, 100), (20000, 1024))]
    linears = lambda: [linear_e4m3(x, w) for x, w in operands]      # noqa: E731
    step()
    before, want = state(), linears()
    assert _lib.lib.spion_linear_status(0) == 0
    _lib.check(_lib.lib.spion_linear_selftest_bounded_wait(1000, torch.cuda.current_stream().cuda_stream))
    try:
        assert _lib.lib.spion_linear_status(0) != 0
        step()
        assert all(torch.equal(a, b) for a, b in zip(before, state()))
        linears()
        torch.cuda.synchronize()
    finally:
        assert _lib.lib.spion_linear_status(1) != 0 and _lib.lib.spion_linear_status(0) == 0
    assert all(torch.equal(a, b) for a, b in zip(linears(), want))
    step()
    for (p, d, (m, v), scales, steps), first in zip(cases, (0, 6, 12)):
        assert float(steps) == 2 and not torch.equal(p.view(torch.uint8), before[first])
