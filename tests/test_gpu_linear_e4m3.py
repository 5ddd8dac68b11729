"""The linear layer on 8-bit operands (csrc/linear_e4m3.cu) against fp64 sums of the same operands: few tokens and many, odd sizes, strides, types, rows
that are not finite, captured calls.

Bound, u = 2^-24: products of two e4m3 numbers are exact.  Their sum in the tensor cores is truncated, 2 u of the partial sum for each of the K / 16 steps at
most that the hardware adds one after another, and the partial sums are below S = sum |x w|; two scales, bias and the sums of eight warps are 12 u more.  Then
one rounding to the result's type (fp16: half of its smallest step too)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def rows8(M, K, g, spread=1.0):
    from spion_b200.quant import quantize_rows
    return quantize_rows(torch.randn(M, K, generator=g, device="cuda") * spread * torch.exp(torch.randn(M, 1, generator=g, device="cuda")))


def check(y, x, w, bias):
    X, W = x.values.double() * x.scales.double()[..., None], w.values.double() * w.scales.double()[:, None]
    b = 0.0 if bias is None else bias.double()
    want, size = X @ W.t() + b, X.abs() @ W.abs().t() + (0.0 if bias is None else bias.double().abs())
    bound = size * U * (X.shape[-1] / 8 + 16) + want.abs() * torch.finfo(y.dtype).eps / 2 + (2.0 ** -25 if y.dtype == torch.float16 else 1e-38)
    off = (y.double() - want).abs()
    if y.dtype == torch.float16:                          # numbers of 65520 and more are infinite in fp16 (half a step above 65504, the largest)
        off = torch.where((y.double() == torch.inf * want.sign()) & (want.abs() + bound >= 65520), 0.0, off)
    assert bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.parametrize("T", [1, 2, 8, 9, 16, 17, 32, 33, 128, 129, 300, 1000])
@pytest.mark.parametrize("K,N", [(1, 1), (16, 8), (64, 128), (100, 77), (129, 300), (1000, 333), (4096, 256)])
def test_sizes(T, K, N):
    from spion_b200.quant import linear_e4m3
    g = torch.Generator(device="cuda").manual_seed(T * 7 + K + N)
    x, w = rows8(T, K, g), rows8(N, K, g)
    bias = torch.randn(N, generator=g, device="cuda")
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        y = linear_e4m3(x, w, bias, out_dtype=dtype)
        assert y.dtype == dtype and y.shape == (T, N)
        check(y, x, w, bias)
    check(linear_e4m3(x, w), x, w, None)


@pytest.mark.parametrize("T,K,N", [(20000, 64, 128), (5000, 320, 257), (33000, 48, 40), (4096, 1040, 4096), (2500, 128, 2056), (130, 8192, 512)])
def test_every_tile_width_and_many_tiles_per_cta(T, K, N):
    from spion_b200.quant import linear_e4m3
    g = torch.Generator(device="cuda").manual_seed(T)
    x, w = rows8(T, K, g), rows8(N, K, g)
    bias = torch.randn(N, generator=g, device="cuda").bfloat16()
    for dtype in (torch.float32, torch.bfloat16):
        check(linear_e4m3(x, w, bias, out_dtype=dtype), x, w, bias)


def test_rows_in_floating_point_shapes_and_strides():
    from spion_b200.quant import Rows8, linear_e4m3, quantize_rows
    g = torch.Generator(device="cuda").manual_seed(1)
    w = rows8(72, 200, g)
    for T in (5, 200):
        x = torch.randn(T, 3, 200, generator=g, device="cuda")
        for t in (x, x.bfloat16(), x.half(), x.transpose(0, 1), x[:, 1]):
            y = linear_e4m3(t, w)
            assert y.dtype == t.dtype and y.shape == (*t.shape[:-1], 72)
            q = quantize_rows(t)
            assert torch.equal(y, linear_e4m3(q, w, out_dtype=t.dtype))
            check(y, q, w, None)
        # operands that lie anywhere: the same bits as their copies
        q = quantize_rows(x[:, 0])
        want = linear_e4m3(q, w)
        off = torch.zeros(T * 201 + 1, dtype=torch.float8_e4m3fn, device="cuda")[1:].view(T, 201)[:, :200]
        off.copy_(q.values)
        assert torch.equal(linear_e4m3(Rows8(off, q.scales), w), want)
        assert torch.equal(linear_e4m3(Rows8(q.values.t().contiguous().t(), q.scales), w), want)
        scales = torch.zeros(T, 2, device="cuda")[:, 0]
        scales.copy_(q.scales)
        assert torch.equal(linear_e4m3(Rows8(q.values, scales), w), want)
        one = Rows8(q.values[:1].expand(T, 200), q.scales[:1].expand(T))
        assert torch.equal(linear_e4m3(one, w), want[:1].expand(T, 72))
    assert linear_e4m3(quantize_rows(x[0, 0]), w).shape == (72,)
    assert linear_e4m3(torch.empty(0, 200, device="cuda"), w).shape == (0, 72)


def test_what_lies_behind_a_row_is_not_read_and_rows_behind_the_last_are_left():
    from spion_b200.quant import Rows8, linear_e4m3
    g = torch.Generator(device="cuda").manual_seed(4)
    for T in (3, 200):
        for K in (40, 120, 136):
            x, w = rows8(T, K, g), rows8(50, K, g)
            want = linear_e4m3(x, w)
            for q in (x, w):                                              # NaN codes behind every row
                ld = q.values.stride(0)
                q.values.as_strided((q.values.shape[0], ld - K), (ld, 1), K).view(torch.uint8).fill_(0x7F)
            assert torch.equal(linear_e4m3(Rows8(*x), Rows8(*w)), want) and bool(torch.isfinite(want).all())


def test_rows_that_are_not_finite_stay_their_own():
    from spion_b200.quant import linear_e4m3, quantize_rows
    for T in (6, 200):
        x, w = torch.randn(T, 256, device="cuda"), quantize_rows(torch.randn(130, 256, device="cuda"))
        want = linear_e4m3(x, w)
        x[2, 3], x[4, 100] = float("nan"), float("inf")
        y = linear_e4m3(x, w)
        rest = [t for t in range(T) if t not in (2, 4)]
        assert torch.equal(y[rest], want[rest]) and not bool(torch.isfinite(y[[2, 4]]).any())


def test_captured_on_another_stream_and_status():
    from spion_b200 import _lib
    from spion_b200.quant import linear_e4m3
    g = torch.Generator(device="cuda").manual_seed(9)
    w = rows8(300, 160, g)
    for T in (4, 700):
        x = torch.randn(T, 160, generator=g, device="cuda")
        want = linear_e4m3(x, w)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = linear_e4m3(x, w)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = linear_e4m3(x, w)
            z = linear_e4m3(y[:, :160].contiguous(), w)
        graph.replay()
        assert torch.equal(y, want) and torch.equal(other, want) and torch.equal(z, linear_e4m3(want[:, :160].contiguous(), w))
        x.mul_(2)
        graph.replay()
        assert torch.equal(y, want * 2)                                   # a power of two moves the scales only
    _lib.check(_lib.lib.spion_linear_status(0), "spion_linear_status")


def test_module_and_norm_before_it():
    """What an encoder does: residual addition, norm to 8 bits, projection."""
    from spion_b200.quant import E4M3Linear, linear_e4m3
    from spion_b200.rmsnorm import rms_norm_e4m3
    g = torch.Generator(device="cuda").manual_seed(3)
    lin = torch.nn.Linear(96, 200).cuda()
    mod = E4M3Linear(lin)
    for T in (7, 500):
        x, r = torch.randn(T, 96, generator=g, device="cuda"), torch.randn(T, 96, generator=g, device="cuda").bfloat16()
        with torch.no_grad():
            s, q = rms_norm_e4m3(x, torch.ones(96, device="cuda"), 1e-6, r)
            y = mod(q)
        assert y.dtype == torch.bfloat16 and mod(x).dtype == torch.float32
        with torch.autocast("cuda", dtype=torch.bfloat16):
            assert mod(x).dtype == torch.bfloat16
        S = s.double()
        n = S / torch.sqrt((S * S).mean(-1, keepdim=True) + 1e-6)
        want = n @ lin.weight.detach().double().t() + lin.bias.detach().double()
        # each operand within 2^-4 of its value (and its row's smallest step, 2^-10 of 1/448 of the largest)
        bound = (n.abs() @ lin.weight.detach().double().abs().t()) * (2 * 2.0 ** -4 + 2.0 ** -8) + want.abs() * 2.0 ** -8 + 1e-3
        assert bool(((y.double() - want).abs() <= bound).all())
    state = mod.state_dict()
    assert set(state) == {"values", "scales", "bias"}


def test_what_it_refuses():
    from spion_b200._lib import SpionError
    from spion_b200.quant import Rows8, linear_e4m3
    g = torch.Generator(device="cuda").manual_seed(5)
    x, w = rows8(10, 64, g), rows8(20, 64, g)

    def refused(match, *args, **kw):
        with pytest.raises(SpionError, match=match):
            linear_e4m3(*args, **kw)

    refused("features", rows8(10, 65, g), w)
    refused("type", Rows8(x.values.float(), x.scales), w)
    refused("type", torch.randn(4, 64, device="cuda").double(), w)
    refused("scale", Rows8(x.values, x.scales[:9]), w)
    refused("scale", Rows8(x.values, x.scales.double()), w)
    refused("bias", x, w, torch.zeros(19, device="cuda"))
    refused("CUDA", x, Rows8(w.values.cpu(), w.scales.cpu()))
    refused("CUDA", torch.randn(4, 64), w)
    refused("output", x, w, out_dtype=torch.float64)
    refused("gradient", torch.randn(4, 64, device="cuda", requires_grad=True), w)
    refused("gradient", x, w, torch.zeros(20, device="cuda", requires_grad=True))
    refused("weights", x, Rows8(w.values[0], w.scales[0]))


@pytest.mark.parametrize("T", [1, 7, 8, 9, 100, 128, 129, 257])
@pytest.mark.parametrize("K,N", [(40, 50), (40, 64), (300, 130), (1000, 333), (512, 520)])
def test_nothing_is_written_outside_of_the_result(T, K, N):
    """Results into a larger matrix, rows further apart than they are long and from any element on: what lies around them stays."""
    from spion_b200 import _lib
    from spion_b200.quant import linear_e4m3
    g = torch.Generator(device="cuda").manual_seed(T + K + N)
    x, w = rows8(T, K, g), rows8(N, K, g)
    for dtype, code in ((torch.float32, _lib.F32), (torch.bfloat16, _lib.BF16), (torch.float16, _lib.F16)):
        want = linear_e4m3(x, w, out_dtype=dtype)
        for ld, first in ((-(-N // 8) * 8 + 16, 64), (N + 3, 64), (N, 65), (N + 1, 3)):
            buf = torch.full((first + (T + 2) * ld + 64,), 7.0, dtype=dtype, device="cuda")
            expect = buf.clone()
            expect[first:].as_strided((T, N), (ld, 1)).copy_(want)
            _lib.check(_lib.lib.spion_linear_e4m3(x.values.data_ptr(), x.values.stride(0) if T > 1 else -(-K // 32) * 32, x.scales.data_ptr(), w.values.data_ptr(),
                                                  w.values.stride(0), w.scales.data_ptr(), None, _lib.F32, buf[first:].data_ptr(), ld, code, T, K, N,
                                                  torch.cuda.current_stream().cuda_stream))
            assert torch.equal(buf, expect)


def test_a_module_keeps_its_codes_when_its_type_is_changed():
    from spion_b200.quant import E4M3Linear
    lin = torch.nn.Linear(96, 40).cuda()
    x = torch.randn(20, 96, device="cuda")
    want = E4M3Linear(lin)(x)
    for change in (lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double().float(), lambda m: m.cpu().cuda(), lambda m: m.half().cpu().cuda().float()):
        m = E4M3Linear(lin)
        bias = m.bias.clone()
        m = change(m)
        assert m.values.dtype == torch.float8_e4m3fn and m.scales.dtype == torch.float32
        m.bias = bias                                                      # (a type change of the bias is the caller's)
        assert torch.equal(m(x), want)


@pytest.mark.parametrize("T,K,N", [(5000, 600, 1001), (5001, 2049, 1000), (20001, 513, 300), (5000, 320, 1001), (9999, 512, 515), (20001, 257, 300)])
def test_pairs_and_their_line_at_odd_sizes(T, K, N):
    """Tiles of two CTAs that end inside the tokens, the features and a chunk, on both sides of the 512 inner features from which pairs are taken; results on 16-byte
    boundaries and off them, each with a NaN behind its rows."""
    from spion_b200.quant import linear_e4m3
    g = torch.Generator(device="cuda").manual_seed(T + K)
    x, w = rows8(T, K, g), rows8(N, K, g)
    bias = torch.randn(N, generator=g, device="cuda").half()
    for q in (x, w):
        ld = q.values.stride(0)
        if ld > K:
            q.values.as_strided((q.values.shape[0], ld - K), (ld, 1), K).view(torch.uint8).fill_(0x7F)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        y = linear_e4m3(x, w, bias, out_dtype=dtype)
        check(y, x, w, bias)
        assert torch.equal(y, linear_e4m3(x, w, bias, out_dtype=dtype))
