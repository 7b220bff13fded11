"""The block-scaled 8-bit products against plain implementations in 64 bits.

Quantization: scales are one fp32 division; a value is the e4m3 number nearest to x / s (an fp32 quotient), so it equals the
plain rounding exactly.  Products: the 8-bit values and the scales are given, a product of two e4m3 values is exact in fp32,
and every sum is held in fp32 or better, but for the tensor cores' sum within an instruction of 32 products, whose terms may
be cut at 2^-13 of the largest of them (a fixed-point sum of at least 13 bits below the leading one).  So the error is at
most (2^-13 + (K + 4) 2^-24) of the sum of magnitudes, and half a unit of the output's type."""
import pytest
import torch

from ltq_research_b200 import fp8

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in TYPES}


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def round_e4m3(v):
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def plain_quant(x, br):
    """e4m3 values and scales of blocks of br x 128, 64 bits (scales rounded to fp32, in which they are held)."""
    R, K = x.shape
    x = torch.nn.functional.pad(x.double(), (0, -K % 128, 0, -R % br))
    b = x.reshape(x.shape[0] // br, br, x.shape[1] // 128, 128)
    s = (b.abs().amax((1, 3)) / 448).float().clamp(min=2.0 ** -126)
    q = round_e4m3((b / s.double()[:, None, :, None]).float().double())  # the fp32 quotient, correctly rounded
    return q.reshape(x.shape)[:R, :K], s


def expand(s, br, R, K):
    return s.double().repeat_interleave(br, 0)[:R].repeat_interleave(128, 1)[:, :K]


def spread(g, R, K, dtype):
    return (torch.randn(R, K, device="cuda", generator=g) * torch.exp(2 * torch.randn(R, 1, device="cuda", generator=g))).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,K", [(1, 1), (3, 128), (5, 130), (128, 127), (129, 1000), (300, 515), (2, 8192)])
def test_quantize(R, K, dtype):
    x = spread(gen(R + K), R, K, dtype)
    for f, br in ((fp8.quantize_rows, 1), (fp8.quantize_blocks, 128)):
        q, s = f(x)
        wq, ws = plain_quant(x, br)
        assert q.shape == (R, K) and torch.equal(s, ws)
        assert torch.equal(q.double(), wq)


def test_quantize_ties_and_extremes():
    """Halfway cases go to the even neighbour; zeros, subnormal inputs; the largest value is 448."""
    x = torch.zeros(4, 256, device="cuda")
    x[0, :6] = torch.tensor([448.0, 17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10, -448.0])
    x[1, 0] = 2.0 ** -140
    x[2, 200] = 3e38
    q, s = fp8.quantize_rows(x)
    assert q[0, :6].double().tolist() == [448.0, 16.0, 20.0, 0.0, 2.0 ** -8, -448.0]
    assert s[0].tolist() == [1.0, 2.0 ** -126] and s[1, 0] == 2.0 ** -126
    assert torch.equal(s[3], torch.full((2,), 2.0 ** -126, device="cuda")) and not q[3].float().any()
    assert torch.equal(q.double(), plain_quant(x, 1)[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_tiny_scales(dtype):
    """Rows of every magnitude down to the subnormal numbers: around the scales below which values and scale are taken larger."""
    g = gen(9)
    e = torch.arange(-149, -40, device="cuda", dtype=torch.float64)[:, None]
    x = (torch.randn(109, 300, device="cuda", generator=g).double() * torch.exp2(e)).float().to(dtype)
    q, s = fp8.quantize_rows(x)
    wq, ws = plain_quant(x, 1)
    assert torch.equal(s, ws) and torch.equal(q.double(), wq)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_non_finite_values_make_their_rows_nan(bad):
    g = gen(3)
    W = fp8.BlockWeight.quantize(torch.randn(200, 300, device="cuda", generator=g))
    x = torch.randn(5, 300, device="cuda", generator=g)
    x[2, 150] = bad
    y = fp8.linear(x, W)
    assert torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 3, 4]]).all()


@pytest.mark.parametrize("off,ld,K", [(0, 300, 256), (1, 259, 200), (2, 130, 129), (3, 200, 128)])
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_strides(dtype, off, ld, K):
    buf = spread(gen(4), 40, ld, dtype).reshape(-1)
    x = torch.cat([buf[:8], buf])[off:off + 40 * ld].view(40, ld)[:, :K]
    for f, br in ((fp8.quantize_rows, 1), (fp8.quantize_blocks, 128)):
        q, s = f(x)
        wq, ws = plain_quant(x, br)
        assert torch.equal(s, ws) and torch.equal(q.double(), wq)


def check(x, W, y, grad=False):
    xq, xs = plain_quant(x.reshape(-1, x.shape[-1]), 1)
    M, R = xq.shape
    a = xq * expand(xs, 1, M, R)
    N, K = W.shape
    w = W.q[:, :K].view(torch.float8_e4m3fn).double() * expand(W.s, 128, N, K)
    if grad:
        w = w.T
    want, mag = a @ w.T, a.abs() @ w.abs().T
    got = y.reshape(want.shape).double()
    tol = (2.0 ** -13 + (R + 4) * 2.0 ** -24) * mag + HALF_ULP[y.dtype] * want.abs() + torch.finfo(y.dtype).smallest_normal
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).max())


SHAPES = [(1, 1, 1), (1, 128, 128), (2, 16, 17), (1, 1000, 2048), (5, 130, 300), (16, 256, 128), (17, 300, 1000), (31, 2051, 640),
          (33, 127, 129), (64, 512, 4096), (65, 513, 255), (100, 64, 8192), (127, 4097, 130), (128, 256, 512), (129, 257, 384),
          (300, 1000, 700), (520, 2500, 1153), (1000, 96, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear(M, N, K, dtype):
    g = gen(M + N + K)
    W = fp8.BlockWeight.quantize(spread(g, N, K, torch.float32) * 0.05)
    x = torch.randn(M, K, device="cuda", generator=g).to(dtype)
    y = fp8.linear(x, W)
    assert y.shape == (M, N) and y.dtype == dtype
    check(x, W, y)
    assert torch.equal(y, fp8.linear(x, W))
    fp8.check_errors(x.device)


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (3, 300, 40), (20, 1000, 513), (64, 5000, 256), (129, 700, 130), (400, 3001, 640),
                                   (7, 40000, 128), (200, 30000, 250)])
def test_linear_grad(M, N, K):
    g = gen(M + N + K)
    W = fp8.BlockWeight.quantize(spread(g, N, K, torch.bfloat16) * 0.05, backward=True)
    dy = (torch.randn(M, N, device="cuda", generator=g) * 1e-3).bfloat16()
    dx = fp8.linear_grad(dy, W)
    assert dx.shape == (M, K)
    check(dy, W, dx, grad=True)
    assert torch.equal(dx, fp8.linear_grad(dy, W))
    fp8.check_errors(dy.device)


@pytest.mark.parametrize("out", TYPES)
def test_output_types_and_leading_dimensions(out):
    g = gen(6)
    W = fp8.BlockWeight.quantize(torch.randn(136, 200, device="cuda", generator=g))
    x = torch.randn(2, 3, 7, 200, device="cuda", generator=g).bfloat16()
    y = fp8.linear(x, W, dtype=out)
    assert y.shape == (2, 3, 7, 136) and y.dtype == out
    check(x, W, y)
    check(x[:, 1], W, fp8.linear(x[:, 1], W))
    t = torch.randn(200, 9, device="cuda", generator=g)
    check(t.t(), W, fp8.linear(t.t(), W))
    assert fp8.linear(x[:0], W).shape == (0, 3, 7, 136)


def test_weights_of_other_layouts():
    """Values as a slice, transposed, of rows that are no multiple of 16 bytes."""
    g = gen(7)
    q, s = fp8.quantize_blocks(torch.randn(260, 333, device="cuda", generator=g))
    x = torch.randn(40, 333, device="cuda", generator=g)
    want = fp8.linear(x, fp8.BlockWeight(q, s))
    dense = q.view(torch.uint8).contiguous().view(torch.float8_e4m3fn)
    col = q.view(torch.uint8).t().contiguous().t().view(torch.float8_e4m3fn)
    for v in (dense, col):
        W = fp8.BlockWeight(v, s.t().contiguous().t())
        assert torch.equal(fp8.linear(x, W), want)
        assert torch.equal(W.dequantize(), fp8.BlockWeight(q, s).dequantize())


def test_long_reduction_and_scales_far_apart():
    """Blocks whose scales differ by many powers of two; K beyond a thousand blocks."""
    g = gen(8)
    K = 131072 + 40
    w = torch.randn(150, K, device="cuda", generator=g) * torch.exp2(torch.randint(-30, 20, (1, K // 128 + 1), device="cuda", generator=g).float()).repeat_interleave(128, 1)[:, :K]
    W = fp8.BlockWeight.quantize(w)
    for M in (2, 70, 130):
        x = torch.randn(M, K, device="cuda", generator=g)
        y = fp8.linear(x, W)
        check(x, W, y)
    fp8.check_errors(x.device)


def test_streams():
    g = gen(9)
    W = fp8.BlockWeight.quantize(torch.randn(1030, 500, device="cuda", generator=g), backward=True)
    x = torch.randn(77, 500, device="cuda", generator=g).bfloat16()
    want = fp8.linear(x, W)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = fp8.linear(x, W)
    s.synchronize()
    assert torch.equal(got, want)


def test_cuda_graph():
    g = gen(10)
    W = fp8.BlockWeight.quantize(torch.randn(1024, 512, device="cuda", generator=g))
    x = torch.randn(3, 512, device="cuda", generator=g).bfloat16()
    fp8.linear(x, W)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fp8.linear(x, W)
    x.copy_(torch.randn(3, 512, device="cuda", generator=g))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, fp8.linear(x, W))


@pytest.mark.parametrize("M,N,K", [(40, 100, 2900), (257, 257, 5300), (600, 1100, 9000), (1030, 2048, 11000), (2048, 2040, 20000),
                                   (1800, 2560, 17000)])
def test_long_sums(M, N, K):
    """Few tiles and a long K, cut among the GPU's SMs: slices that fill them, slices and a rest, one slice and a rest."""
    g = gen(K)
    W = fp8.BlockWeight.quantize(torch.randn(N, K, device="cuda", generator=g))
    x = torch.randn(M, K, device="cuda", generator=g).bfloat16()
    y = fp8.linear(x, W, dtype=torch.float32)
    check(x, W, y)
    assert torch.equal(y, fp8.linear(x, W, dtype=torch.float32))
    fp8.check_errors(x.device)


# one row tile of 128 and several, rows of both widths of the streaming kernel, K cut over 1, 2, 4 and 8 CTAs, odd numbers of
# blocks and widths; with 17 rows and more only weights of at least 18817 rows go there, and up to K = 4864
STREAMED = [(1, 19000, 300), (3, 5000, 1100), (9, 20001, 130), (16, 38000, 1000), (1, 128256, 256), (2, 300, 9000), (16, 2100, 3333),
            (17, 18817, 128), (17, 19072, 129), (20, 18950, 1000), (24, 25000, 2048), (31, 40009, 515), (32, 18944, 4864),
            (32, 20000, 4000), (19, 18820, 4865), (33, 19000, 300)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", STREAMED)
def test_streamed_weights(M, N, K, dtype):
    g = gen(M + N + K)
    W = fp8.BlockWeight.quantize(spread(g, N, K, torch.bfloat16) * 0.05)
    x = torch.randn(M, K, device="cuda", generator=g).to(dtype)
    y = fp8.linear(x, W)
    check(x, W, y)
    assert torch.equal(y, fp8.linear(x, W))
    fp8.check_errors(x.device)


@pytest.mark.parametrize("M", [1, 17, 32])
def test_streamed_rows_of_any_stride_and_bad_values(M):
    g = gen(15)
    W = fp8.BlockWeight.quantize(torch.randn(19000, 400, device="cuda", generator=g))
    x = torch.randn(M, 411, device="cuda", generator=g).bfloat16()[:, 3:403]
    check(x, W, fp8.linear(x, W))
    x[M // 2, 390] = float("nan")
    y = fp8.linear(x, W)
    bad = torch.arange(M, device="cuda") == M // 2
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()


@pytest.mark.parametrize("kind", ["random", "positive", "one large"])
@pytest.mark.parametrize("M,N,K", [(8, 512, 128), (8, 512, 4096), (24, 20000, 128), (24, 20000, 4096), (200, 512, 1024), (200, 512, 16384)])
def test_sums_are_those_of_fp32(M, N, K, kind):
    """The tensor cores' sums of 32 products and what was summed before lose at most 2^-24 of the largest term for each of the 33, and
    a block more is one rounding more: (33 + K / 128 + 4) 2^-24 of the sum of magnitudes.  (Measured: 8 at K = 128 and one product far
    above the others, 14 at K = 16384 and all of one sign.)"""
    g = gen(M + K)
    w, x = torch.randn(N, K, device="cuda", generator=g), torch.randn(M, K, device="cuda", generator=g)
    if kind == "positive":
        w, x = w.abs(), x.abs()
    if kind == "one large":
        x[:, ::128] *= 300
        w[:, ::128] *= 30
    W = fp8.BlockWeight.quantize(w)
    xq, xs = plain_quant(x, 1)
    a, b = xq * expand(xs, 1, M, K), W.q[:, :K].view(torch.float8_e4m3fn).double() * expand(W.s, 128, N, K)
    err = (fp8.linear(x, W, dtype=torch.float32).double() - a @ b.T).abs()
    assert bool((err <= (33 + K // 128 + 4) * 2.0 ** -24 * (a.abs() @ b.abs().T)).all())


@pytest.mark.parametrize("M,N,K", [(60, 512, 640), (300, 256, 4000), (700, 1100, 256)])
def test_calls_one_after_another(M, N, K):
    """Calls without a pause between them, in buffers that pass from one to the next, alone and from a graph: each has the
    result that it has by itself."""
    g = gen(M)
    W = fp8.BlockWeight.quantize(torch.randn(N, K, device="cuda", generator=g))
    xs = [torch.randn(M, K, device="cuda", generator=g).bfloat16() for _ in range(6)]
    want = []
    for x in xs:
        want.append(fp8.linear(x, W))
        torch.cuda.synchronize()
    for _ in range(10):
        got = [fp8.linear(x, W) for x in xs]
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    x = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fp8.linear(x, W)
        z = fp8.linear(x * 2, W)
    for k in range(6):
        x.copy_(xs[k])
        graph.replay()
        assert torch.equal(y, want[k]) and torch.equal(z, want[k] * 2)
    fp8.check_errors(x.device)


def test_gradient_against_differences():
    """linear is linear in its quantized input, and inputs that are e4m3 values under a power of two quantize to themselves
    when their block holds 448 of it: so the difference quotient is exact but for the sums' rounding."""
    g = gen(11)
    W = fp8.BlockWeight.quantize(torch.randn(256, 128, device="cuda", generator=g), backward=True)
    grid = lambda *shape: round_e4m3(torch.randn(*shape, device="cuda", generator=g).double() * 60).float()
    x, v, dy = grid(6, 128), torch.zeros(6, 128, device="cuda"), grid(6, 256)
    x[:, 0], dy[:, 0], dy[:, 128] = 448.0, 448.0, 448.0
    x[:, 1:] = x[:, 1:].sign() * 32.0 * torch.randint(8, 15, (6, 127), device="cuda", generator=g)
    v[:, 1:] = 32.0 * torch.randint(-1, 2, (6, 127), device="cuda", generator=g)
    x = torch.where(x.abs() > 448, torch.full_like(x, 448.0), x)
    up, dn = (x + v).clamp(-448, 448), (x - v).clamp(-448, 448)
    f = lambda t: (fp8.linear(t, W).double() * dy.double()).sum()
    d = fp8.linear_grad(dy, W)
    want = (d.double() * (up - dn).double()).sum()
    mag = (up.abs().double() @ W.dequantize().abs().double().T * dy.abs().double()).sum()
    assert abs(float(f(up) - f(dn) - want)) <= 3 * (2.0 ** -13 + 300 * 2.0 ** -24) * float(mag)


def test_autograd():
    g = gen(12)
    W = fp8.BlockWeight.quantize(torch.randn(140, 96, device="cuda", generator=g), backward=True)
    x = torch.randn(4, 5, 96, device="cuda", generator=g).requires_grad_()
    dy = torch.randn(4, 5, 140, device="cuda", generator=g)
    fp8.block_linear(x, W).backward(dy)
    check(dy, W, x.grad, grad=True)


@pytest.mark.parametrize("M", [3, 40])
def test_first_product_in_a_graph(M):
    """No call before the capture: what a first product needs once is there with the weight."""
    from ltq_research_b200 import liqk_v2
    torch.cuda.synchronize()
    fp8._FLAGS.clear()
    liqk_v2._GEMM_ERR.clear()
    g = gen(14)
    W = fp8.BlockWeight.quantize(torch.randn(300, 512, device="cuda", generator=g), backward=True)
    x, dy = torch.randn(M, 512, device="cuda", generator=g), torch.randn(M, 300, device="cuda", generator=g)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = fp8.linear(x, W), fp8.linear_grad(dy, W)
    graph.replay()
    assert torch.equal(y, fp8.linear(x, W)) and torch.equal(dx, fp8.linear_grad(dy, W))
    fp8.check_errors(x.device)


@pytest.mark.parametrize("device", ["cuda", "cuda:0"])
def test_errors_are_found_however_the_device_is_named(device):
    W = fp8.BlockWeight.quantize(torch.randn(64, 64, device="cuda:0"))
    fp8.check_errors("cuda:0")
    fp8._error_flag(W.device).fill_(1)  # as a wait that ran out does
    with pytest.raises(RuntimeError, match="ltq_fp8_gemm"):
        fp8.check_errors(device)
    fp8.check_errors(device)  # reported once


def test_second_derivatives_are_refused():
    g = gen(13)
    W = fp8.BlockWeight.quantize(torch.randn(40, 96, device="cuda", generator=g), backward=True)
    x = torch.randn(3, 96, device="cuda", generator=g).requires_grad_()
    d, = torch.autograd.grad(fp8.block_linear(x, W).pow(3).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(d.square().sum() + x.square().sum(), x)


def test_refusals():
    w = torch.randn(130, 200, device="cuda")
    q, s = fp8.quantize_blocks(w)
    W = fp8.BlockWeight(q, s)
    x = torch.randn(3, 200, device="cuda")
    for f in (lambda: fp8.linear(x.double(), W), lambda: fp8.linear(x, W, dtype=torch.float64), lambda: fp8.quantize_rows(x.int()),
              lambda: fp8.quantize_blocks(w.double())):
        with pytest.raises(TypeError):
            f()
    for f in (lambda: fp8.linear(x[:, :199], W), lambda: fp8.linear_grad(torch.randn(3, 130, device="cuda"), W),
              lambda: fp8.BlockWeight(q.float(), s), lambda: fp8.BlockWeight(q, s[:1]), lambda: fp8.BlockWeight(q, s.double()),
              lambda: fp8.quantize_rows(x.t()), lambda: fp8.quantize_rows(x[0]), lambda: fp8.quantize_rows(x[:1].expand(3, 200))):
        with pytest.raises(ValueError):
            f()
    for f in (lambda: fp8.linear(x.cpu(), W), lambda: fp8.BlockWeight(q.cpu(), s.cpu())):
        with pytest.raises(RuntimeError, match="CUDA"):
            f()
