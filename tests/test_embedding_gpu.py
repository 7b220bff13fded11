"""Token lookup and its gradient against plain implementations in 64 bits.

Tolerances: a looked-up value is one fp32 product of two numbers, rounded once more to the table's type; a gradient is an
fp32 sum of n terms (n - 1 roundings, each at most 2^-24 of the sum of magnitudes), times the scale (one rounding), rounded
once to the output's type."""
import pytest
import torch

from ltq_research_b200 import embedding

pytestmark = pytest.mark.gpu
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,D,shape", [(1, 1, (1,)), (10, 3, (2, 3)), (100, 64, (7,)), (333, 1000, (5, 2)), (50, 2560, (16,)),
                                       (1000, 2047, (31,)), (77, 130, (1000,)), (64, 8192, (3,)), (5, 12, (0,))])
def test_lookup(V, D, shape, dtype):
    g = gen(D)
    table = torch.randn(V, D, device="cuda", generator=g).to(dtype)
    tok = torch.randint(0, V, shape, device="cuda", generator=g)
    for t in (tok, tok.int()):
        got = embedding.lookup(table, t, scale=1.7)
        assert got.shape == (*shape, D) and got.dtype == dtype
        want = table.double()[tok] * float(torch.tensor(1.7, dtype=torch.float32))
        tol = (HALF_ULP[dtype] + 2.0 ** -24) * want.abs() * 1.01 + TINY[dtype]
        assert bool(((got.double() - want).abs() <= tol).all())
    assert torch.equal(embedding.lookup(table, tok), table[tok])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("off,ld,D", [(0, 72, 64), (1, 67, 64), (2, 66, 64), (0, 65, 65), (4, 100, 60)])
def test_lookup_strides(dtype, off, ld, D):
    buf = torch.randn(40 * ld + 8, device="cuda", generator=gen(1)).to(dtype)
    table = buf[off:off + 40 * ld].view(40, ld)[:, :D]
    tok = torch.randint(0, 40, (6, 50), device="cuda", generator=gen(2))
    assert torch.equal(embedding.lookup(table, tok.t()), table[tok.t()])
    out = torch.empty(6, 50, D, dtype=dtype, device="cuda")
    assert embedding.lookup(table, tok, out=out) is out and torch.equal(out, table[tok])


def test_lookup_outside():
    table = torch.ones(10, 40, device="cuda")
    got = embedding.lookup(table, torch.tensor([-1, 3, 10, 2 ** 40], device="cuda"))
    assert torch.equal(got[:, 0], torch.tensor([0.0, 1.0, 0.0, 0.0], device="cuda"))


def test_lookup_beyond_32_bits():
    """Element offsets above 2^32."""
    V, D = 2 ** 20 + 5, 4096 + 64
    table = torch.empty(V, D, dtype=torch.bfloat16, device="cuda")
    table[-1] = torch.arange(D, device="cuda") % 100
    table[7] = 3.0
    got = embedding.lookup(table, torch.tensor([V - 1, 7], device="cuda"))
    assert torch.equal(got[0], table[-1]) and torch.equal(got[1], table[7])
    tok = torch.tensor([V - 1, 7, V - 1], device="cuda")
    embedding.lookup_grad(tok, got[[0, 1, 0]], V, out=table)
    assert torch.equal(table[-1], 2 * got[0]) and torch.equal(table[7], got[1])
    assert not table[8:1000].any() and not table[-1000:-1].any()


def plain_grad(tok, dout, V, scale, pad=None):
    D = dout.shape[-1]
    t, d = tok.reshape(-1), dout.reshape(-1, D).double()
    ok = (t >= 0) & (t < V)
    if pad is not None:
        ok &= t != pad
    t, d = t[ok].long(), d[ok]
    z = torch.zeros(V, D, dtype=torch.float64, device=d.device)
    n = torch.zeros(V, dtype=torch.float64, device=d.device).index_add_(0, t, torch.ones_like(t, dtype=torch.float64))
    return z.clone().index_add_(0, t, d) * scale, z.index_add_(0, t, d.abs()) * abs(scale), n


def check_grad(tok, dout, V, scale=1.0, pad=None, dtype=torch.float32, base=None, got=None):
    want, mag, n = plain_grad(tok, dout, V, scale, pad)
    if got is None:
        out = None if base is None else base.clone()
        got = embedding.lookup_grad(tok, dout, V, scale, pad, out=out, accumulate=base is not None, dtype=dtype)
    if base is not None:
        want, mag = want + base.double(), mag + base.double().abs()
    tol = ((n + 1)[:, None] * 2.0 ** -24 * mag + HALF_ULP[got.dtype] * want.abs()) * 1.01 + TINY[got.dtype]
    assert bool(((got.double() - want).abs() <= tol).all())
    return got


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (1, 2000, 64), (5, 3, 7), (8, 1500, 40), (9, 1500, 40), (63, 1023, 1000),
                                   (700, 1024, 65), (1000, 20, 256), (5000, 70000, 96), (12345, 999, 130)])
def test_grad(n, V, D, dtype, out_dtype):
    g = gen(n + D)
    tok = torch.randint(0, V, (n,), device="cuda", generator=g)
    dout = torch.randn(n, D, device="cuda", generator=g).to(dtype)
    a = check_grad(tok, dout, V, scale=0.5, dtype=out_dtype)
    b = embedding.lookup_grad(tok.int(), dout, V, 0.5, dtype=out_dtype)
    assert torch.equal(a, b)  # deterministic, whatever the tokens' type
    assert not a[torch.bincount(tok, minlength=V) == 0].any()


@pytest.mark.parametrize("n", [31, 8192, 8193, 40000])
@pytest.mark.parametrize("hot", [1.0, 0.5, 0.1])
def test_grad_of_frequent_tokens(n, hot):
    """Runs over many chunks, that begin and end anywhere in them."""
    g = gen(n)
    V, D = 300000, 72
    tok = torch.randint(0, V, (n,), device="cuda", generator=g)
    is_hot = torch.rand(n, device="cuda", generator=g) < hot
    tok = torch.where(is_hot, torch.randint(0, 3, (n,), device="cuda", generator=g) * (V - 1) // 2, tok)
    dout = torch.randn(n, D, device="cuda", generator=g).bfloat16()
    check_grad(tok, dout, V)
    check_grad(torch.full_like(tok, V - 1), dout, V)


def test_grad_million_rows_of_tokens():
    g = gen(3)
    tok = torch.randint(0, 1 << 21, (300001,), device="cuda", generator=g)  # three sort passes
    check_grad(tok, torch.randn(300001, 16, device="cuda", generator=g), 1 << 21)


@pytest.mark.parametrize("n", [1, 300, 9001])
@pytest.mark.parametrize("D", [1032, 1031])
def test_grad_zeros_of_a_large_table(n, D):
    """Rows that no token names, more than are written beside the sort; some tokens in runs of neighbours, some at the ends."""
    g = gen(n + D)
    V = 70001
    tok = (torch.rand(n, device="cuda", generator=g) ** 4 * V).long()
    tok[n // 2:] = V - 1 - tok[n // 2:] // 64
    dout = torch.randn(n, D, device="cuda", generator=g)
    out = torch.full((V, D + 9), float("nan"), device="cuda")
    got = embedding.lookup_grad(tok, dout, V, out=out[:, :D])
    check_grad(tok, dout, V, got=got)
    assert not got[torch.bincount(tok, minlength=V) == 0].any()
    assert out[:, D:].isnan().all()


def test_grad_without_positions():
    for V, D in ((1, 1), (70001, 40)):
        out = torch.ones(V, D, device="cuda")
        embedding.lookup_grad(torch.empty(0, dtype=torch.int64, device="cuda"), torch.empty(0, D, device="cuda"), V, out=out)
        assert not out.any()


def test_grad_order_is_that_of_the_positions():
    """Equal tokens are summed in the order of their positions: a sum whose value depends on it."""
    tok = torch.zeros(8, dtype=torch.int64, device="cuda")
    d = torch.tensor([2.0 ** 24, 1.0, -2.0 ** 24, 1.0, 0, 0, 0, 0], device="cuda")[:, None].repeat(1, 5)
    assert (embedding.lookup_grad(tok, d, 2)[0] == 1.0).all()


def grouped_sums(tok, d, V, chunk=8):
    """The documented grouping, in fp32: chunks of the sorted list summed in order, a row's chunks joined in order, of nine chunks or
    more in eight stretches of equally many."""
    key, pos = torch.sort(tok, stable=True)
    parts = {}
    for at in range(len(tok)):
        row = parts.setdefault(int(key[at]), {})
        row[at // chunk] = row.get(at // chunk, torch.zeros(d.shape[1])) + d[pos[at]]

    def total(xs):
        s = torch.zeros(d.shape[1])
        for x in xs:
            s = s + x
        return s
    out = torch.zeros(V, d.shape[1])
    for v, row in parts.items():
        p = [row[c] for c in sorted(row)]
        if len(p) > 8:
            each = (len(p) + 7) // 8
            p = [total(p[w * each:(w + 1) * each]) for w in range(8)]
        out[v] = total(p)
    return out


@pytest.mark.parametrize("before", [0, 5, 6, 7])
@pytest.mark.parametrize("n", [12, 64, 71, 72, 73, 200])
def test_grad_grouping(before, n):
    """Rows of one to many chunks that begin anywhere in a chunk, with values whose sum depends on the grouping."""
    g = torch.Generator().manual_seed(n + before)
    tok = torch.cat([torch.zeros(before, dtype=torch.int64), torch.ones(n, dtype=torch.int64), torch.full((3,), 2)])
    tok = tok[torch.randperm(len(tok), generator=g)]
    d = torch.randn(len(tok), 5, generator=g) * torch.exp2(torch.randint(-10, 25, (len(tok), 5), generator=g).float())
    got = embedding.lookup_grad(tok.cuda(), d.cuda(), 3).cpu()
    assert torch.equal(got, grouped_sums(tok, d, 3))


def test_grad_padding_and_outside():
    g = gen(4)
    tok = torch.randint(-3, 55, (4, 100), device="cuda", generator=g)
    dout = torch.randn(4, 100, 48, device="cuda", generator=g)
    dout[(tok < 0) | (tok >= 50) | (tok == 7)] = float("nan")
    got = check_grad(tok, torch.nan_to_num(dout), 50, pad=7, got=embedding.lookup_grad(tok, dout, 50, padding_idx=7))
    assert not got[7].any()
    none = embedding.lookup_grad(torch.full((9,), 7, device="cuda"), torch.ones(9, 48, device="cuda"), 50, padding_idx=7)
    assert none.shape == (50, 48) and not none.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_grad_accumulates(dtype):
    g = gen(5)
    V, D, n = 400, 88, 900
    base = torch.randn(V, D, device="cuda", generator=g).to(dtype)
    tok = torch.randint(0, V // 2, (n,), device="cuda", generator=g)
    dout = torch.randn(n, D, device="cuda", generator=g).to(dtype)
    got = check_grad(tok, dout, V, scale=2.0, base=base, dtype=dtype)
    assert torch.equal(got[V // 2:], base[V // 2:])
    same = embedding.lookup_grad(tok[:0], dout[:0], V, out=base.clone(), accumulate=True)
    assert torch.equal(same, base)
    assert not embedding.lookup_grad(tok[:0], dout[:0], V).any()


@pytest.mark.parametrize("n,V,D", [(8193, 500, 40), (20000, 30000, 264), (30000, 70, 130), (9000, 100000, 1040)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_grad_accumulates_many_positions(n, V, D, dtype):
    """Beyond 8192 positions, with rows of one position and of many chunks, and rows that no token names."""
    g = gen(n)
    base = torch.randn(V, D, device="cuda", generator=g).to(dtype)
    tok = (torch.rand(n, device="cuda", generator=g) ** 4 * V * 0.9).long()
    dout = torch.randn(n, D, device="cuda", generator=g).to(dtype)
    got = check_grad(tok, dout, V, scale=0.5, pad=3, base=base, dtype=dtype)
    unnamed = torch.bincount(tok, minlength=V) == 0
    unnamed[3] = True
    assert bool((torch.bincount(tok, minlength=V) > 64).any()) and torch.equal(got[unnamed], base[unnamed])
    assert torch.equal(got, embedding.lookup_grad(tok, dout, V, 0.5, 3, out=base.clone(), accumulate=True))


@pytest.mark.parametrize("D,ld_d,ld_o,off", [(64, 72, 80, 0), (64, 65, 64, 0), (33, 40, 35, 1), (16, 16, 24, 3), (66, 68, 70, 2)])
@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.float32), (torch.float32, torch.float16)])
def test_grad_strides(D, ld_d, ld_o, off, dtype, out_dtype):
    g = gen(6)
    n, V = 200, 120
    tok = torch.randint(0, V, (n,), device="cuda", generator=g)
    dout = torch.randn(n * ld_d + off, device="cuda", generator=g).to(dtype)[off:].view(n, ld_d)[:, :D]
    buf = torch.full((V * ld_o + off,), 9.0, dtype=out_dtype, device="cuda")
    out = buf[off:].view(V, ld_o)[:, :D]
    check_grad(tok, dout, V, got=embedding.lookup_grad(tok, dout, V, out=out))
    out.fill_(9.0)
    assert (buf == 9.0).all()


def test_grad_of_an_expanded_gradient():
    tok = torch.randint(0, 30, (40,), device="cuda", generator=gen(7))
    check_grad(tok, torch.ones(1, 1, device="cuda").expand(40, 24), 30)


def test_grad_against_differences():
    """The lookup is linear in the table, so a difference quotient along a direction is exact up to rounding: sums of 900
    products of magnitude 1, 1e-4 of them at most."""
    g = gen(8)
    table, step = (torch.randn(60, 30, device="cuda", generator=g) for _ in range(2))
    tok = torch.randint(0, 60, (30,), device="cuda", generator=g)
    dout = torch.randn(30, 30, device="cuda", generator=g)
    f = lambda t: (embedding.lookup(t, tok, 3.0).double() * dout.double()).sum()
    d = embedding.lookup_grad(tok, dout, 60, 3.0)
    want = (f(table + step) - f(table - step)) / 2
    assert abs(float(want - (d.double() * step.double()).sum())) < 1e-2 * 1e-2 * 30


def test_autograd_and_streams():
    g = gen(9)
    table = torch.randn(90, 32, device="cuda", generator=g).requires_grad_()
    tok = torch.randint(0, 90, (3, 11), device="cuda", generator=g)
    dout = torch.randn(3, 11, 32, device="cuda", generator=g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        embedding.embed(table, tok, 2.0, padding_idx=1).backward(dout)
    s.synchronize()
    check_grad(tok, dout, 90, 2.0, 1, got=table.grad)


@pytest.mark.parametrize("n,V,D", [(700, 5000, 264), (9000, 40000, 1040)])
def test_grad_calls_one_after_another(n, V, D):
    """Calls without a pause between them, into one output, alone and from a graph: each has the result that it has by itself."""
    g = gen(n)
    toks = [(torch.rand(n, device="cuda", generator=g) ** 3 * V).long() for _ in range(4)]
    d = torch.randn(n, D, device="cuda", generator=g).bfloat16()
    want = []
    for t in toks:
        want.append(embedding.lookup_grad(t, d, V))
        torch.cuda.synchronize()
    out = torch.empty(V, D, device="cuda")
    tok = toks[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        embedding.lookup_grad(tok, d, V, out=out)
    for k in range(12):
        embedding.lookup_grad(toks[(k + 1) % 4], d, V, out=out)
        embedding.lookup_grad(toks[k % 4], d, V, out=out)
        assert torch.equal(out, want[k % 4])
        tok.copy_(toks[(k + 2) % 4])
        graph.replay()
        assert torch.equal(out, want[(k + 2) % 4])


@pytest.mark.parametrize("n,V", [(8193, 900), (20001, 70000), (100000, 1 << 21)])
def test_grad_of_many_positions_again_and_again(n, V):
    """One, two and three digit passes in a cluster, beside CTAs of the call before that still write: the same bits each time."""
    g = gen(n)
    tok = torch.randint(0, V, (n,), device="cuda", generator=g)
    dout = torch.randn(n, 8, device="cuda", generator=g)
    want = check_grad(tok, dout, V)
    for _ in range(30):
        assert torch.equal(embedding.lookup_grad(tok, dout, V), want)


@pytest.mark.parametrize("form", ["lookup", "gradient", "accumulated"])
def test_outputs_written_in_place_tell_autograd(form):
    a = torch.randn(6, 16, device="cuda", generator=gen(11)).requires_grad_()
    y = a.exp()  # keeps its result for the backward pass
    table, tok = torch.randn(20, 16, device="cuda", generator=gen(12)), torch.arange(6, device="cuda")
    if form == "lookup":
        embedding.lookup(table, tok, out=y.detach())
    else:
        embedding.lookup_grad(tok, table[:6], 6, out=y.detach(), accumulate=form == "accumulated")
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_second_derivatives_are_refused():
    table = torch.randn(20, 16, device="cuda", generator=gen(10)).requires_grad_()
    y = embedding.embed(table, torch.arange(9, device="cuda"))
    g, = torch.autograd.grad(y.pow(3).sum(), table, create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(g.square().sum() + table.square().sum(), table)


def test_outputs_that_overlap_an_input_are_refused():
    """Rows are written while others are still read: a table or a gradient that the output overlaps would be read half written."""
    buf = torch.randn(40, 24, device="cuda", generator=gen(13))
    keep, tok = buf.clone(), torch.arange(10, device="cuda")
    for f in (lambda: embedding.lookup(buf, tok, out=buf[:10]), lambda: embedding.lookup(buf[5:], tok, out=buf[2:12]),
              lambda: embedding.lookup_grad(tok, buf[:10], 20, out=buf[5:25]),
              lambda: embedding.lookup_grad(tok, buf[:10, :12], 10, out=buf[:10, 4:16], accumulate=True)):
        with pytest.raises(ValueError, match="overlap"):
            f()
    assert torch.equal(buf, keep)
    got = embedding.lookup_grad(tok, buf[:10, :12], 10, out=buf[:10, 12:])  # beside each other
    check_grad(tok, keep[:10, :12], 10, got=got)
    assert torch.equal(buf[:, :12], keep[:, :12])
    embedding.lookup(buf[:5], torch.zeros(0, dtype=torch.int64, device="cuda"), out=buf[:0])


def test_refusals():
    table = torch.zeros(10, 8, device="cuda")
    tok = torch.zeros(3, dtype=torch.int64, device="cuda")
    d = torch.zeros(3, 8, device="cuda")
    for f in (lambda: embedding.lookup(table.double(), tok), lambda: embedding.lookup(table, tok.float()),
              lambda: embedding.lookup_grad(tok.short(), d, 10), lambda: embedding.lookup_grad(tok, d.double(), 10),
              lambda: embedding.lookup_grad(tok, d, 10, dtype=torch.float64)):
        with pytest.raises(TypeError):
            f()
    for f in (lambda: embedding.lookup(table.t(), tok), lambda: embedding.lookup(table[0], tok),
              lambda: embedding.lookup(table[:1].expand(10, 8), tok), lambda: embedding.lookup(table[:0], tok),
              lambda: embedding.lookup(table, tok, out=torch.zeros(3, 7, device="cuda")),
              lambda: embedding.lookup_grad(tok, d[:2], 10), lambda: embedding.lookup_grad(tok, d, 0),
              lambda: embedding.lookup_grad(tok, d, 10, padding_idx=10), lambda: embedding.lookup_grad(tok, d, 10, padding_idx=-1),
              lambda: embedding.lookup_grad(tok, d, 10, accumulate=True),
              lambda: embedding.lookup_grad(tok, d, 10, out=torch.zeros(9, 8, device="cuda"))):
        with pytest.raises(ValueError):
            f()
    for f in (lambda: embedding.lookup(table.cpu(), tok), lambda: embedding.lookup_grad(tok.cpu(), d, 10)):
        with pytest.raises(RuntimeError, match="CUDA"):
            f()
