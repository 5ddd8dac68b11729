"""Rows of a token table and its gradient (csrc/token_rows.cu) against fp64: sizes on both sides of every limit, types, padding, runs of equal ids, strides, captured calls.

Bounds, u = 2^-24: a looked-up row is one product and one rounding.  A row of the gradient is a sum of n numbers in fp32, in the order of the tokens up to how it is cut into
pieces: n u of the sum of their magnitudes at most, a product with the scale and one rounding."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(t):
    return torch.finfo(t).eps / 2


def least(t):
    return 2.0 ** -25 if t == torch.float16 else 1e-38


def gradient(ids, g, V, scale, padding, dtype):
    """The gradient and its bound in fp64"""
    ids, g = ids.reshape(-1), g.reshape(-1, g.shape[-1]).double()
    keep = (ids >= 0) & (ids < V)
    if padding is not None:
        keep &= ids != padding % V
    n = torch.bincount(ids[keep], minlength=V).double()[:, None]
    want, size = (torch.zeros(V, g.shape[1], dtype=torch.float64, device="cuda").index_add_(0, ids[keep], v[keep]) for v in (g, g.abs()))
    s = float(torch.tensor(scale, dtype=torch.float32))
    return want * s, size * abs(s) * U * (n + 2) + (want * s).abs() * half_step(dtype) + least(dtype)


def check(ids, w, scale=1.0, padding=None, out_dtype=None, seed=0):
    from spion_b200.tokens import embed_tokens
    V, N = w.shape
    w = w.detach().requires_grad_()
    y = embed_tokens(ids, w, scale, padding, out_dtype)
    dt = out_dtype or w.dtype
    assert y.dtype == dt and y.shape == (*ids.shape, N)
    want = w.detach().double()[ids] * float(torch.tensor(scale, dtype=torch.float32))
    assert bool(((y.detach().double() - want).abs() <= want.abs() * (half_step(dt) + U) + least(dt)).all())
    g = torch.randn(y.shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dt)
    dw, = torch.autograd.grad(y, w, g, retain_graph=True)
    want, bound = gradient(ids, g, V, scale, padding, w.dtype)
    off = (dw.double() - want).abs()
    assert dw.dtype == w.dtype and bool((off <= bound).all()), float((off / bound).max())
    again, = torch.autograd.grad(y, w, g)
    assert torch.equal(dw, again)
    return dw


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,N", [(1, 1, 1), (1, 32000, 4096), (3, 2, 7), (31, 511, 8), (64, 512, 33), (2048, 513, 64), (2049, 1000, 72), (5000, 300000, 16), (4099, 10007, 769),
                                   (70000, 100, 32), (300000, 5000, 24), (9000, 1, 260), (8192, 300, 16),
                                   (8193, 300, 16), (5000, 262143, 4), (9000, 262144, 4), (10, 50, 20000), (100, 2000000, 3), (131073, 70, 1)])
def test_sizes(T, V, N, dtype):
    g = torch.Generator(device="cuda").manual_seed(T + V + N)
    w = torch.randn(V, N, generator=g, device="cuda").to(dtype)
    ids = torch.randint(0, V, (T,), generator=g, device="cuda")
    check(ids, w, 1.7)


@pytest.mark.parametrize("seed", range(24))
def test_drawn_calls(seed):
    """Sizes, types, frequencies, strides and padding at random."""
    import random
    rng = random.Random(seed)
    T, V, N = (int(2 ** rng.uniform(0, m)) for m in (16, 14, 9))
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(V, N, generator=g, device="cuda").to(rng.choice(TYPES))
    if rng.random() < 0.3:
        w = torch.nn.functional.pad(w, (1, 2))[:, 1:1 + N]
    skew = rng.choice([0.0, 1.0, 4.0])                     # how unequally frequent ids are
    ids = (torch.rand(T, generator=g, device="cuda") ** (1 + skew) * V).long().clamp(max=V - 1)
    ids = ids if rng.random() < 0.5 else ids.sort().values
    check(ids, w, rng.choice([1.0, 0.1, 7.0]), rng.choice([None, rng.randrange(V)]), rng.choice([None, *TYPES]), seed)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [5, 64, 520])
def test_runs_of_every_length(N, dtype):
    """Ids whose runs begin and end anywhere in the pieces of 64, from none to thousands."""
    lengths = [0, 1, 2, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 191, 192, 193, 0, 300, 5000, 1, 64, 64, 64, 0, 7]
    ids = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths)).cuda()
    w = torch.randn(len(lengths) + 2, N, device="cuda").to(dtype)
    for order in (torch.arange(len(ids)), torch.randperm(len(ids), generator=torch.Generator().manual_seed(1))):
        for padding in (None, 18, -2):
            check(ids[order.cuda()], w, 0.5, padding)


def test_padding_and_ids_outside():
    from spion_b200.tokens import embed_tokens
    w = torch.randn(50, 40, device="cuda", requires_grad=True)
    ids = torch.randint(0, 50, (4, 33), device="cuda")
    ids[0, :20] = 49
    dw = check(ids, w, padding=49)
    assert bool((dw[49] == 0).all()) and bool((check(ids, w, padding=-1) == dw).all())
    outside = ids.clone()
    outside[1, 1], outside[2, 2], outside[3, 3], outside[3, 4] = -1, 50, 2 ** 40, -2 ** 40
    bad = (outside < 0) | (outside >= 50)
    y = embed_tokens(outside, w)
    assert bool(y.detach()[bad].isnan().all()) and torch.equal(y.detach()[~bad], w.detach()[outside[~bad]])
    g = torch.randn(y.shape, device="cuda")
    dw, = torch.autograd.grad(y, w, g)
    want, bound = gradient(outside, g, 50, 1.0, None, torch.float32)
    assert bool(((dw.double() - want).abs() <= bound).all())
    assert embed_tokens(torch.empty(0, 3, dtype=torch.long, device="cuda"), w).shape == (0, 3, 40)
    y = embed_tokens(torch.empty(0, dtype=torch.long, device="cuda"), w)
    dw, = torch.autograd.grad(y, w, y.detach())
    assert bool((dw == 0).all()) and dw.shape == (50, 40)


def test_not_finite_gradients_stay_with_their_row():
    from spion_b200.tokens import embed_tokens
    w = torch.randn(20, 16, device="cuda", requires_grad=True)
    ids = torch.randint(0, 20, (500,), device="cuda")
    ids[100] = 3
    y = embed_tokens(ids, w, padding_idx=5)
    g = torch.randn(500, 16, device="cuda")
    g[100, 2] = float("nan")
    g[ids == 5] = float("inf")
    dw, = torch.autograd.grad(y, w, g)
    finite = dw.isfinite()
    assert not bool(finite[3, 2]) and int((~finite).sum()) == 1


@pytest.mark.parametrize("dtype", TYPES)
def test_types_strides_and_offsets(dtype):
    from spion_b200.tokens import embed_tokens
    g = torch.Generator(device="cuda").manual_seed(2)
    w = torch.randn(100, 48, generator=g, device="cuda").to(dtype)
    ids = torch.randint(0, 100, (6, 70), generator=g, device="cuda")
    for out in TYPES:
        check(ids, w, 3.0, None, out)
    want = embed_tokens(ids, w, 3.0)
    dy = torch.randn(6, 70, 48, generator=g, device="cuda").to(dtype)

    def run(ids, w, dy):
        w = w.detach().requires_grad_()
        y = embed_tokens(ids, w, 3.0)
        return y.detach(), torch.autograd.grad(y, w, dy)[0]

    plain = run(ids, w, dy)
    assert torch.equal(plain[0], want)
    off = torch.empty(100 * 51 + 1, dtype=dtype, device="cuda")[1:].view(100, 51)[:, 2:50]
    off.copy_(w)
    dyo = torch.empty(6, 70, 50, dtype=dtype, device="cuda")[..., 1:49]
    dyo.copy_(dy)
    for a in ((ids.int(), w, dy), (ids, off, dy), (ids, w.t().contiguous().t(), dyo), (ids.t().contiguous().t(), w, dy.transpose(0, 1).contiguous().transpose(0, 1))):
        assert all(torch.equal(p, q) for p, q in zip(plain, run(*a)))
    # a gradient that is one row for all tokens
    w2 = w.detach().requires_grad_()
    total = embed_tokens(ids, w2, 3.0).float().sum()
    dw, = torch.autograd.grad(total, w2)
    n = torch.bincount(ids.reshape(-1), minlength=100).double()[:, None] * 3
    assert bool(((dw.double() - n).abs() <= n * (half_step(dtype) + 64 * U)).all())
    rows = w[:1].expand(100, 48)
    assert torch.equal(embed_tokens(ids, rows), w[:1].expand(420, 48).view(6, 70, 48))


def test_a_recorded_backward_and_two_streams():
    from spion_b200.tokens import embed_tokens
    w = torch.randn(30, 12, device="cuda", requires_grad=True)
    ids = torch.randint(-1, 31, (80,), device="cuda")
    g = torch.randn(80, 12, device="cuda", requires_grad=True)
    y = embed_tokens(ids, w, 2.0, padding_idx=4)
    plain, = torch.autograd.grad(y, w, g.detach(), retain_graph=True)
    graph, = torch.autograd.grad(y, w, g, create_graph=True)
    torch.testing.assert_close(plain, graph, rtol=1e-5, atol=1e-5)
    dg, = torch.autograd.grad((graph * plain).sum(), g)
    inside = (ids >= 0) & (ids < 30) & (ids != 4)
    torch.testing.assert_close(dg[inside], 2.0 * plain[ids[inside]])
    assert bool((dg[~inside] == 0).all())
    w2 = torch.randn(5000, 64, device="cuda", requires_grad=True)
    ids2 = torch.randint(0, 5000, (30000,), device="cuda")
    g2 = torch.randn(30000, 64, device="cuda")
    want = torch.autograd.grad(embed_tokens(ids2, w2), w2, g2)[0]
    other = torch.cuda.Stream()
    for _ in range(5):
        other.wait_stream(torch.cuda.current_stream())
        a = torch.autograd.grad(embed_tokens(ids2, w2), w2, g2)[0]
        with torch.cuda.stream(other):
            b = torch.autograd.grad(embed_tokens(ids2, w2), w2, g2)[0]
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, want)


def test_captured_and_replayed():
    from spion_b200.tokens import embed_tokens
    w = torch.randn(3000, 96, device="cuda").bfloat16().requires_grad_()
    batches = [torch.randint(0, 3000, (8, 700), device="cuda") for _ in range(2)]
    g = torch.randn(8, 700, 96, device="cuda").bfloat16()

    def step(ids):
        y = embed_tokens(ids, w, 9.0, padding_idx=0)
        return y.detach(), torch.autograd.grad(y, w, g)[0]

    want = [step(b) for b in batches]
    ids = batches[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        step(ids)
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = step(ids)
            graphs.append((graph, out))
    torch.cuda.synchronize()
    for i in (1, 0):
        ids.copy_(batches[i])
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, want[i]))


def test_the_module_beside_torchs():
    from spion_b200.tokens import ScaledEmbedding
    m = ScaledEmbedding(200, 32, padding_idx=3).cuda()
    t = torch.nn.Embedding(200, 32, padding_idx=3).cuda()
    t.load_state_dict(m.state_dict())
    ids = torch.randint(0, 200, (10, 20), device="cuda")
    assert torch.equal(m(ids), t(ids))
    for e in (m, t):
        e(ids).square().sum().backward()
    torch.testing.assert_close(m.weight.grad, t.weight.grad)
    half = ScaledEmbedding(200, 32, scale=5.0, bf16_out=True).cuda()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(half(ids), (half.weight[ids] * 5.0).bfloat16())
    assert half(ids).dtype == torch.float32
    with pytest.raises(ValueError, match="max_norm"):
        ScaledEmbedding(10, 4, max_norm=1.0)


def test_refusals():
    from spion_b200._lib import SpionError
    from spion_b200.tokens import embed_tokens
    w, ids = torch.randn(10, 8, device="cuda"), torch.zeros(3, dtype=torch.long, device="cuda")
    for call in (lambda: embed_tokens(ids.float(), w), lambda: embed_tokens(ids.cpu(), w), lambda: embed_tokens(ids, w.double()), lambda: embed_tokens(ids, w[0]),
                 lambda: embed_tokens(ids, w, padding_idx=10), lambda: embed_tokens(ids, w, padding_idx=-11), lambda: embed_tokens(ids, w, out_dtype=torch.float64)):
        with pytest.raises(SpionError):
            call()
