"""The root-mean-square norm (csrc/rmsnorm.cu) against its formula in fp64: outputs, sums, gradients and rows in e4m3, for widths around every change of
kernel, types, strides, rows that are empty, zero or not finite, captured calls and calls on another stream.

Bounds, with u = 2^-24 and h(t) = half a step of type t relative to the value (torch.finfo(t).eps / 2):
  K(N) = 64 + N / 512: more additions than any partial sum of a row takes one after another (32 in a thread, the rest in trees, wide rows N / 512).
  y: the mean has a relative error of K u, its root K u / 2, rsqrtf 4 u, three products 3 u.
  dx: terms of the row's mean carry 6 u each and K u from their sum; the other factors of dx 12 u.
  dw: a column is added in at most M / 32 + 100 steps, each term carries 8 u.
Each result is then rounded once: h of its type (fp16 also half of its smallest step, 2^-25)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
T = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return 2.0 ** -25 if t == torch.float16 else 2.0 ** -140


def K(N):
    return 64 + N / 512


def inputs(M, N, stream, branch, out, seed=0):
    g = torch.Generator(device="cuda").manual_seed(1000 * M + N + seed)
    x = (torch.randn(M, N, generator=g, device="cuda") * 2 + 0.3).to(T[stream])
    r = None if branch is None else torch.randn(M, N, generator=g, device="cuda").to(T[branch])
    w = 1 + 0.3 * torch.randn(N, generator=g, device="cuda")
    dy = torch.randn(M, N, generator=g, device="cuda").to(T[out or stream])
    ds = torch.randn(M, N, generator=g, device="cuda").to(T[stream])
    return x, r, w, dy, ds


def normed(s, w):
    S = s.double()
    return S * w.double() / torch.sqrt((S * S).mean(-1, keepdim=True) + EPS)


def check_rows8(q, y, rel):
    """q against the values y in fp64 of which the quantised ones are a relative error of rel off."""
    a, scales = y.abs().amax(-1), q.scales.double()
    assert bool(((scales * 448 - a).abs() <= a * (rel + 2 * U)).all())
    # half a step of a normal number, or of the smallest numbers (2^-9), and what the value itself is off
    off = (q.values.double() * scales[..., None] - y).abs()
    assert bool((off <= y.abs() * (2.0 ** -4 + rel + 4 * U) + scales[..., None] * 2.0 ** -10 * (1 + 1e-6)).all())


def check_forward(s, w, y):
    """s: the rows that were normalised, as they are kept."""
    want, N = normed(s, w), s.shape[-1]
    bound = want.abs() * ((K(N) / 2 + 8) * U + half(y.dtype)) + tiny(y.dtype)
    assert bool(((y.double() - want).abs() <= bound).all())


def check_backward(s, w, dy, ds, dx, dw):
    S, W, D, N, M = s.double(), w.double(), dy.double(), s.shape[-1], s.numel() // s.shape[-1]
    rho = 1 / torch.sqrt((S * S).mean(-1, keepdim=True) + EPS)
    n, g = S * rho, D * W
    gn = g * n
    skip = torch.zeros_like(S) if ds is None else ds.double()
    want = rho * (g - n * gn.mean(-1, keepdim=True)) + skip
    bound = U * (rho * (16 * g.abs() + (2 * K(N) + 24) * n.abs() * gn.abs().mean(-1, keepdim=True)) + 2 * skip.abs() + K(N) * rho * g.abs())
    bound = bound + want.abs() * half(dx.dtype) * 1.01 + tiny(dx.dtype)
    assert bool(((dx.double() - want).abs() <= bound).all())
    dn = (D * n).reshape(-1, N)
    off = (dw.double() - dn.sum(0)).abs()
    assert bool((off <= dn.abs().sum(0) * (M / 32 + 100 + K(N) + 8) * U + dn.sum(0).abs() * half(dw.dtype) + 1e-30).all())


WIDTHS = [1, 2, 7, 8, 63, 64, 72, 128, 136, 256, 264, 512, 520, 769, 1000, 1024, 1032, 4096, 8192, 8193, 8200, 16384, 16392, 20001]


@pytest.mark.parametrize("N", WIDTHS)
@pytest.mark.parametrize("stream,branch,out", [("fp32", "bf16", "bf16"), ("bf16", "bf16", "bf16"), ("fp32", None, "fp16")])
def test_both_directions(N, stream, branch, out):
    from spion_b200.rmsnorm import rms_norm
    M = 5 if N > 4096 else 37 if N > 300 else 203
    x, r, w, dy, ds = inputs(M, N, stream, branch, out)
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    if r is None:
        y = rms_norm(xs, ws, EPS, out_dtype=T[out])
        dx, dw = torch.autograd.grad(y, (xs, ws), dy)
        check_forward(x, w, y)
        check_backward(x, w, dy, None, dx, dw)
        return
    rs = r.clone().requires_grad_()
    s, y = rms_norm(xs, ws, EPS, res=rs, out_dtype=T[out])
    assert s.dtype == x.dtype and y.dtype == T[out]
    want = x.double() + r.double()
    assert bool(((s.double() - want).abs() <= want.abs() * (half(s.dtype) + 2 * U) + tiny(s.dtype)).all())
    check_forward(s, w, y)
    dx, dr, dw = torch.autograd.grad((s, y), (xs, rs, ws), (ds, dy))
    check_backward(s, w, dy, ds, dx, dw)
    assert dr.dtype == r.dtype and bool(((dr.double() - dx.double()).abs() <= dx.double().abs() * half(r.dtype) * 1.01 + tiny(r.dtype)).all())


@pytest.mark.parametrize("stream,branch,out", [(s, b, o) for s in T for b in [None, *T] for o in T if s == "fp32" or (b in (None, s) and o == s)])
@pytest.mark.parametrize("M,N", [(1, 64), (300, 64), (150, 1024), (149, 1280), (20, 333)])
def test_types(M, N, stream, branch, out):
    from spion_b200.rmsnorm import rms_norm
    x, r, w, dy, ds = inputs(M, N, stream, branch, out, 3)
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    rs = None if r is None else r.clone().requires_grad_()
    got = rms_norm(xs, ws, EPS, res=rs, out_dtype=T[out])
    s, y = (x, got) if r is None else got
    check_forward(s, w, y)
    if r is None:
        dx, dw = torch.autograd.grad(y, (xs, ws), dy)
        check_backward(s, w, dy, None, dx, dw)
    else:
        dx, dw, dr = torch.autograd.grad((s, y), (xs, ws, rs), (ds, dy))
        check_backward(s, w, dy, ds, dx, dw)


@pytest.mark.parametrize("M,N", [(1, 1), (4, 16), (1, 4096), (700, 64), (150, 512), (149, 4096), (33, 777), (3, 17000), (2, 9001)])
@pytest.mark.parametrize("stream,branch", [("fp32", "bf16"), ("bf16", "bf16"), ("fp16", None), ("fp32", None)])
def test_rows_in_e4m3(M, N, stream, branch):
    from spion_b200.quant import quantize_rows
    from spion_b200.rmsnorm import rms_norm_e4m3
    x, r, w, _, _ = inputs(M, N, stream, branch, None, 7)
    out = rms_norm_e4m3(x, w, EPS, res=r)
    s, q = (x, out) if r is None else out
    assert q.values.dtype == torch.float8_e4m3fn and q.values.shape == x.shape and q.scales.shape == (M,)
    assert q.values.stride(0) % 16 == 0 or M == 1

    check_rows8(q, normed(s, w), (K(N) / 2 + 8) * U)
    check_rows8(quantize_rows(x), x.double(), 0.0)
    # the same bits as the definition in fp32 (maximum, one division, one product, one rounding)
    a = x.float().abs().amax(1, keepdim=True).clamp_min(2.0 ** -100)
    plain = (x.float() * (448.0 / a)).to(torch.float8_e4m3fn)
    assert torch.equal(quantize_rows(x).values.view(torch.uint8), plain.view(torch.uint8))


def test_rows_that_are_zero_tiny_or_not_finite():
    from spion_b200.quant import quantize_rows
    from spion_b200.rmsnorm import rms_norm, rms_norm_e4m3
    for N in (64, 333, 2048, 17000):
        x = torch.randn(6, N, device="cuda")
        x[1] = 0
        x[2, 3] = float("nan")
        x[3, 5] = float("inf")
        x[4] *= 1e-30
        w = torch.ones(N, device="cuda")
        y = rms_norm(x, w, EPS)
        assert bool(torch.isfinite(y[[0, 1, 4, 5]]).all()) and bool((y[1] == 0).all())
        assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(y[3, 5]))
        for q in (rms_norm_e4m3(x, w, EPS), quantize_rows(x)):
            back = q.values.float() * q.scales[:, None]
            assert bool(torch.isfinite(back[[0, 1, 4, 5]]).all()) and bool((back[1] == 0).all())
            assert not bool(torch.isfinite(back[2]).any()) and not bool(torch.isfinite(back[3]).any())
        back = quantize_rows(x).values[4].float() * quantize_rows(x).scales[4]
        assert bool(((back - x[4]).abs() <= x[4].abs() * 2.0 ** -4 + x[4].abs().max() / 448 * 2.0 ** -9).all())


def test_strides_shapes_and_empty_calls():
    from spion_b200.quant import quantize_rows
    from spion_b200.rmsnorm import rms_norm, rms_norm_e4m3
    g = torch.Generator(device="cuda").manual_seed(2)
    big = torch.randn(40, 3, 200, generator=g, device="cuda")
    w = torch.randn(64, generator=g, device="cuda")
    for x in (big[:, 1, 8:72], big[:, 1, 7:71], big[:, :, :64], big.transpose(0, 1)[..., 100:164], big[:1, 0, :64].expand(9, 64), big[:, 0, :128:2], big[0, 0, :64]):
        # (views off the pieces' boundaries are read element by element, in another order than their copies: not the same bits)
        y = rms_norm(x, w, EPS)
        assert y.shape == x.shape
        check_forward(x, w, y)
        s, y = rms_norm(x, w, EPS, res=x.flip(0).contiguous())
        assert torch.equal(s, x + x.flip(0))
        check_forward(s, w, y)
        xs, ws = x.detach().requires_grad_(), w.clone().requires_grad_()
        dy = torch.randn(x.shape, generator=g, device="cuda")
        dx, dw = torch.autograd.grad(rms_norm(xs, ws, EPS), (xs, ws), dy)
        check_backward(x, w, dy, None, dx, dw)
        q = rms_norm_e4m3(x, w, EPS)
        assert q.scales.shape == x.shape[:-1] and q.values.shape == x.shape
        check_rows8(q, normed(x, w), (K(64) / 2 + 8) * U)
        check_rows8(quantize_rows(x), x.double(), 0.0)
    # gradients that are views
    x = torch.randn(30, 64, device="cuda", requires_grad=True)
    dx, dw = torch.autograd.grad(rms_norm(x, ws, EPS), (x, ws), torch.ones(1, 1, device="cuda").expand(30, 64))
    check_backward(x.detach(), w, torch.ones(30, 64, device="cuda"), None, dx, dw)
    # no rows
    x = torch.empty(0, 64, device="cuda", requires_grad=True)
    y = rms_norm(x, ws, EPS)
    dx, dw = torch.autograd.grad(y, (x, ws), torch.empty(0, 64, device="cuda"))
    assert y.shape == (0, 64) and dx.shape == (0, 64) and bool((dw == 0).all())
    q = quantize_rows(torch.empty(2, 0, 7, device="cuda"))
    assert q.values.shape == (2, 0, 7) and q.scales.shape == (2, 0)


def test_gradients_that_do_not_arrive_and_inputs_that_need_none():
    from spion_b200.rmsnorm import rms_norm
    x, r, w, dy, ds = inputs(50, 64, "fp32", "bf16", "bf16")
    xs, rs, ws = x.clone().requires_grad_(), r.clone().requires_grad_(), w.clone().requires_grad_()
    s, y = rms_norm(xs, ws, EPS, res=rs, out_dtype=torch.bfloat16)
    dx, dr = torch.autograd.grad(s, (xs, rs), ds, retain_graph=True)
    assert torch.equal(dx, ds) and torch.equal(dr, ds.to(torch.bfloat16))
    dx, dw = torch.autograd.grad(y, (xs, ws), dy)
    check_backward(s.detach(), w, dy, None, dx, dw)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, xs, dy)                                     # freed
    s, y = rms_norm(x, ws, EPS, res=rs)
    dr, = torch.autograd.grad(y, rs, torch.ones_like(y))
    assert dr.dtype == torch.bfloat16
    assert not rms_norm(x, w, EPS).requires_grad
    # a sum that the caller changes before the backward
    s, y = rms_norm(xs, ws, EPS, res=rs)
    with torch.no_grad():
        s.add_(1)
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_gradient_of_the_gradient():
    from spion_b200.rmsnorm import rms_norm
    x, r, w, dy, _ = inputs(6, 24, "fp32", "fp32", "fp32")

    def penalty(f):
        xs, rs, ws = (t.clone().requires_grad_() for t in (x, r, w))
        s, y = f(xs, rs, ws)
        loss = (y * dy).sum() + (s * s).sum()
        gs = torch.autograd.grad(loss, (xs, ws), create_graph=True)
        return torch.autograd.grad(sum((g * g).sum() for g in gs), (xs, rs, ws))

    def plain(xs, rs, ws):
        s = xs + rs
        return s, s * torch.rsqrt((s * s).mean(-1, keepdim=True) + EPS) * ws

    for a, b in zip(penalty(lambda xs, rs, ws: rms_norm(xs, ws, EPS, res=rs)), penalty(plain)):
        assert float((a - b).abs().max()) <= 2e-4 * float(b.abs().max())   # two fp32 chains of the same formula, some tens of roundings of sums of 24


def test_against_differences():
    from spion_b200.rmsnorm import rms_norm
    x, r, w, dy, ds = (t.double() for t in inputs(3, 40, "fp32", "fp32", "fp32"))
    xs, rs, ws = (t.float().requires_grad_() for t in (x, r, w))
    s, y = rms_norm(xs, ws, EPS, res=rs)
    got = torch.autograd.grad((s, y), (xs, ws), (ds.float(), dy.float()))

    def value(x, w):
        t = x + r
        return float((t * ds).sum() + (t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS) * w * dy).sum())

    h = 1e-4
    for k, at in ((0, (1, 7)), (0, (2, 39)), (1, (11,))):
        lo, hi = [x.clone(), w.clone()], [x.clone(), w.clone()]
        lo[k][at] -= h
        hi[k][at] += h
        want = (value(*hi) - value(*lo)) / (2 * h)
        # differences in fp64: h^2 times a third derivative of order one; the gradient in fp32
        assert abs(float(got[k][at]) - want) <= 1e-5 * max(1.0, abs(want))


def test_captured_and_on_another_stream():
    from spion_b200.rmsnorm import rms_norm, rms_norm_e4m3
    x, r, w, dy, ds = inputs(500, 256, "fp32", "bf16", "bf16")
    xs, rs, ws = x.clone().requires_grad_(), r.clone().requires_grad_(), w.clone().requires_grad_()

    def step():
        s, y = rms_norm(xs, ws, EPS, res=rs, out_dtype=torch.bfloat16)
        # (no eager graph of the leaves may live while another is captured: results without their history)
        return (s.detach(), y.detach(), *torch.autograd.grad((s, y), (xs, rs, ws), (ds, dy)), *rms_norm_e4m3(xs.detach(), ws.detach(), EPS))

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            other = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        xs.mul_(2)
    graph.replay()
    changed = [t.clone() for t in got]
    with torch.no_grad():
        xs.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c, d in zip(want, got, other, changed):
        assert torch.equal(a.float(), b.float()) and torch.equal(a.float(), c.float())
    assert not torch.equal(want[0], changed[0])


def test_module_beside_the_framework():
    from spion_b200.rmsnorm import FusedRMSNorm
    mod, ref = FusedRMSNorm(96).cuda(), torch.nn.RMSNorm(96, eps=1e-6).cuda()
    ref.load_state_dict(mod.state_dict())
    x = torch.randn(4, 50, 96, device="cuda")
    assert float((mod(x) - ref(x)).detach().abs().max()) <= 2e-6                    # values up to 5, a few units in the last place each
    mod = FusedRMSNorm(96, bf16_out=True).cuda()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        s, y = mod.add_norm(x, x.bfloat16())
        assert s.dtype == torch.float32 and y.dtype == torch.bfloat16
    assert mod(x).dtype == torch.float32
    assert mod.add_norm(x.half(), x)[1].dtype == torch.float16


@pytest.mark.parametrize("N", [1, 40, 64, 136, 333, 512, 1000, 2048, 4096, 5001, 16384, 17000, 20001])
def test_weights_that_are_not_finite(N):
    """A NaN of the weight, or an infinite weight times zero, is a NaN in every row: in 8 bits nothing of such a row comes back finite, in other types that
    column alone.  An infinite y has an infinite scale, NaN in its place and zeros in the others, as the definition gives."""
    from spion_b200.rmsnorm import rms_norm, rms_norm_e4m3
    for M in (3, 300):
        for bad in (float("nan"), float("inf"), -float("inf")):
            x = torch.randn(M, N, device="cuda") + 3
            w = torch.ones(N, device="cuda")
            x[1, N // 2], w[N // 2] = 0, bad
            for res in (None, torch.zeros_like(x)):
                out = rms_norm_e4m3(x, w, EPS, res=res)
                q = out if res is None else out[1]
                y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
                a = y.abs().amax(1)
                want = (y * (448.0 / a)[:, None]).to(torch.float8_e4m3fn).float()
                assert torch.equal(q.scales.isnan(), a.isnan()) and torch.equal(q.scales.isinf(), a.isinf()) and bool(a.isnan()[1])
                assert torch.equal(q.values.float().nan_to_num(7.0), want.nan_to_num(7.0))
                z = rms_norm(x, w, EPS, res=res)
                z = z if res is None else z[1]
                assert torch.equal(z.isnan(), y.isnan()) and torch.equal(z.isinf(), y.isinf())


def test_gradients_after_a_wait_that_gave_up_are_nan():
    """The word that a bounded wait of the backward's ring sets is set by the self-test of a short one: until it has been reported the gradients of that kernel are
    NaN, not what their memory held; after that they are as before.  (The other kernels wait for nothing.)"""
    from spion_b200 import _lib
    from spion_b200.rmsnorm import rms_norm
    g = torch.Generator(device="cuda").manual_seed(2)
    calls = []
    for M, N, stream, branch in ((600, 2048, "fp32", "bf16"), (3, 4096, "fp32", None), (200, 16384, "bf16", None), (5, 1024, "fp32", "fp16"), (300, 4000, "fp16", "fp16")):
        x = torch.randn(M, N, generator=g, device="cuda").to(T[stream]).requires_grad_()
        r = None if branch is None else torch.randn(M, N, generator=g, device="cuda").to(T[branch]).requires_grad_()
        calls.append((x, r, torch.rand(N, generator=g, device="cuda", requires_grad=True), torch.randn(M, N, generator=g, device="cuda").to(T[stream])))

    def gradients():
        out = []
        for x, r, w, dy in calls:
            y = rms_norm(x, w, EPS, res=r)
            out += torch.autograd.grad(y if r is None else y[1], (x, w) if r is None else (x, w, r), dy)
        return out

    want = gradients()
    torch.cuda.synchronize()
    assert all(bool(torch.isfinite(t).all()) for t in want) and _lib.lib.spion_linear_status(0) == 0
    _lib.check(_lib.lib.spion_linear_selftest_bounded_wait(1000, torch.cuda.current_stream().cuda_stream))
    try:
        assert all(bool(t.isnan().all()) for t in gradients())
    finally:
        assert _lib.lib.spion_linear_status(1) != 0 and _lib.lib.spion_linear_status(0) == 0
    assert all(torch.equal(a, b) for a, b in zip(gradients(), want))


class Guarded:
    """Tensors cut out of larger ones, `off` elements from a boundary, with 64 elements on either side that nothing may change."""

    def __init__(self):
        self.made = []

    def __call__(self, M, N, dtype, off=0, ld=None):
        ld = N if ld is None else ld
        size = torch.empty((), dtype=dtype).element_size()
        buf = torch.full(((64 + off + max(M, 1) * ld + 64) * size,), 0x5A, dtype=torch.uint8, device="cuda").view(dtype)
        self.made.append((buf, buf.clone(), off, M, N, ld))
        return buf[64 + off:].as_strided((M, N), (ld, 1))

    def check(self):
        for buf, was, off, M, N, ld in self.made:
            was[64 + off:].as_strided((M, N), (ld, 1)).copy_(buf[64 + off:].as_strided((M, N), (ld, 1)))
            assert torch.equal(buf.view(torch.uint8), was.view(torch.uint8))


CODE = {"fp32": 0, "bf16": 1, "fp16": 2, "e4m3": 3}


@pytest.mark.parametrize("M,N", [(1, 1), (3, 8), (5, 64), (37, 72), (130, 120), (9, 250), (300, 256), (7, 512), (150, 520), (11, 1000), (149, 2048), (2, 4096), (5, 4104), (3, 8192), (2, 16384), (3, 16400), (2, 17001)])
@pytest.mark.parametrize("stream,branch,out", [("fp32", "bf16", "fp16"), ("bf16", "bf16", "bf16"), ("fp32", None, "e4m3"), ("fp16", "fp16", "e4m3"), ("fp32", "fp32", "fp32")])
def test_nothing_is_written_beside_the_results(M, N, stream, branch, out):
    """Through the C entries: inputs with rows apart, outputs in the middle of other memory, on and off the boundaries of the wide accesses."""
    from spion_b200 import _lib
    from spion_b200.rmsnorm import rms_norm, rms_norm_e4m3
    st = torch.cuda.current_stream().cuda_stream
    x, r, w, dy, ds = inputs(M, N, stream, branch, None if out == "e4m3" else out, 5)
    types = {**T, "e4m3": torch.float8_e4m3fn}
    if out == "e4m3":
        want = rms_norm_e4m3(x, w, EPS, res=r)
        want = (None, *want) if r is None else (want[0], *want[1])
    else:
        want = rms_norm(x, w, EPS, res=r, out_dtype=T[out])
        want = (None, want) if r is None else want

    def p(t):
        return None if t is None else t.data_ptr()

    for off, apart in ((0, 0), (1, 0), (0, 32), (8, 8), (3, 5)):
        new = Guarded()
        X, R = new(M, N, T[stream], off, N + apart).copy_(x), None if r is None else new(M, N, T[branch], 0, N + 2 * apart).copy_(r)
        S = None if r is None else new(M, N, T[stream], off)
        Y = new(M, N, types[out], 0 if out == "e4m3" else off, -(-N // 32) * 32 + apart if out == "e4m3" else N + apart)
        scale, rho = new(1, M, torch.float32) if out == "e4m3" else None, new(1, M, torch.float32)
        _lib.check(_lib.lib.spion_rmsnorm_forward(p(X), N + apart, CODE[stream], p(R), N + 2 * apart if R is not None else 0, CODE[branch or stream], p(w), 0, p(S), p(Y),
                                                  Y.stride(0), CODE[out], p(scale), p(rho), M, N, EPS, 1, st))
        new.check()
        if S is not None:
            assert torch.equal(S, want[0])
        if out == "e4m3":
            check_rows8(type("Rows", (), {"values": Y, "scales": scale[0]}), normed(x if S is None else S, w), (K(N) / 2 + 8) * U)
            continue
        check_forward(x if S is None else S, w, Y)
        new = Guarded()
        kept, two = (x if S is None else S), branch == "bf16" and stream == "fp32"
        Sx, D, Ds = new(M, N, T[stream], off, N + apart).copy_(kept), new(M, N, T[out], off).copy_(dy), new(M, N, T[stream], off).copy_(ds)
        dx, dr, dw = new(M, N, T[stream], off), new(M, N, T[branch], off) if two else None, new(1, N, torch.float32, off)
        ws = new(1, int(_lib.lib.spion_rmsnorm_workspace_floats(M, N)), torch.float32)
        _lib.check(_lib.lib.spion_rmsnorm_backward(p(Sx), N + apart, CODE[stream], p(D), CODE[out], p(Ds), p(w), 0, p(rho), p(dx), p(dr), CODE[branch] if two else 0, p(dw),
                                                   p(ws), M, N, st))
        new.check()
        check_backward(kept, w, dy, ds, dx, dw[0])
        if two:
            assert bool(((dr.double() - dx.double()).abs() <= dx.double().abs() * half(dr.dtype) * 1.01 + tiny(dr.dtype)).all())
