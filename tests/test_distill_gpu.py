"""The divergence from a teacher's top logits and its gradient against their formulas in 64 bits.

Tolerances.  z / tau in units of log2 is at most 64 here, so one fp32 rounding of it is 64 * 2^-24 = 4e-6, which is the
relative error of an exponential; a sum of V / 512 positive terms adds less.  A logarithm of a probability is then good to
1e-5, the teacher's p to 1e-5 of itself, and a loss (probabilities that sum to 1 times logarithms of at most 30) to 4e-4 at
worst where every p errs the same way; they are normalised by the same sum, so 1e-4 stands.  The gradient is w / tau
(q P - p): 4e-5 w / tau, and half a unit of the logits' type."""
import math

import pytest
import torch

from ltq_research_b200 import distill

pytestmark = pytest.mark.gpu
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def plain(logits, idx, teacher, lse=None, weight=None, tau=1.0):
    """Loss and gradient, 64 bits, row by row from the definition."""
    T, V = logits.shape
    z = logits.double().cpu() / tau
    loss, grad = torch.zeros(T, dtype=torch.float64), torch.zeros(T, V, dtype=torch.float64)
    for t in range(T):
        w = 1.0 if weight is None else float(weight[t])
        if w == 0.0:
            continue
        slots = [(int(i), float(u) / tau) for i, u in zip(idx[t].cpu(), teacher[t].double().cpu()) if 0 <= int(i) < V]
        m = float(z[t].max())
        e = torch.exp(z[t] - m) if m > -math.inf else torch.zeros(V, dtype=torch.float64)
        S = float(e.sum())
        q = e / S if S > 0 else e
        if lse is not None:
            p = [math.exp(u - float(lse[t])) for _, u in slots]
        else:
            um = max([u for _, u in slots], default=0.0)
            p = [math.exp(u - um) if u > -math.inf else 0.0 for _, u in slots]
            n = sum(p)
            p = [x / n for x in p] if n > 0 else p
        top = torch.zeros(V, dtype=torch.bool)
        target = torch.zeros(V, dtype=torch.float64)
        for (i, _), pk in zip(slots, p):
            top[i] = True
            target[i] += pk
            if pk > 0:
                loss[t] += w * pk * (math.log(pk) - (math.log(float(q[i])) if q[i] > 0 else -math.inf))
        rest = max(0.0, 1.0 - sum(p)) if lse is not None and not bool(top.all()) else 0.0
        qr = float(q[~top].sum())
        if rest > 0:
            loss[t] += w * rest * (math.log(rest) - (math.log(qr) if qr > 0 else -math.inf))
        P = sum(p) + rest
        g = q * P - target
        if rest > 0 and qr > 0:
            g = g - torch.where(top, torch.zeros_like(q), q * (rest / qr))
        grad[t] = w / tau * g
    return loss, grad


def make(T, V, K, dtype, seed=0, rest=True, pad=0, tau=1.0):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(T, V, generator=g) * 2
    z.scatter_add_(1, torch.randint(0, V, (T, 4), generator=g), 4 + 4 * torch.rand(T, 4, generator=g))
    u_all = z + 0.5 * torch.randn(T, V, generator=g)
    u, idx = torch.topk(u_all, K, dim=1)
    lse = torch.logsumexp(u_all / tau, 1) if rest else None
    buf = torch.zeros(T, V + pad, dtype=dtype, device="cuda")
    logits = buf[:, :V]
    logits.copy_(z)
    return logits, idx.cuda(), u.cuda(), None if lse is None else lse.cuda()


def check(logits, idx, teacher, lse=None, weight=None, tau=1.0, got=None):
    want_l, want_d = plain(logits, idx, teacher, lse, weight, tau)
    kw = dict(teacher_lse=lse, weight=weight, temperature=tau)
    loss, d = got if got is not None else distill.topk_loss_grad(logits, idx, teacher, **kw)
    w = (torch.ones(logits.shape[0]) if weight is None else weight.cpu()).double().abs()
    fin = torch.isfinite(want_l)
    assert torch.equal(torch.isfinite(loss.cpu()), fin)
    assert torch.equal(loss.cpu()[~fin].double(), want_l[~fin])
    assert bool(((loss.cpu().double() - want_l).abs()[fin] <= 1e-4 * w[fin]).all())
    err = (d.double().cpu() - want_d).abs()
    tol = 4e-5 * (w / tau)[:, None] + HALF_ULP[logits.dtype] * 1.01 * want_d.abs() + (2.0 ** -25 if logits.dtype == torch.float16 else 0)
    assert bool((err <= tol).all()), float((err - tol).max())
    return loss, d


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("T,V,K,pad", [(1, 1, 1, 0), (3, 5, 2, 0), (2, 31, 31, 1), (5, 1000, 17, 0), (3, 1003, 64, 0),
                                       (4, 4099, 128, 5), (2, 20000, 300, 8), (1, 3000, 1024, 0)])
def test_loss_and_gradient(T, V, K, pad, rest, dtype):
    logits, idx, u, lse = make(T, V, K, dtype, seed=V + K, rest=rest, pad=pad)
    loss, d = check(logits, idx, u, lse)
    loss0, stats = distill.topk_loss(logits, idx, u, teacher_lse=lse)
    assert torch.equal(loss, loss0)  # one code path
    g = torch.linspace(-1.0, 2.0, T, device="cuda")
    d2 = distill.topk_grad(logits, idx, u, stats, grad=g, teacher_lse=lse)
    check(logits, idx, u, lse, weight=g, got=(loss * g, d2))


@pytest.mark.parametrize("V", [128256, 262144])
def test_long_rows(V):
    logits, idx, u, lse = make(2, V, 64, torch.bfloat16, seed=V)
    check(logits, idx, u, lse)
    logits, idx, u, lse = make(2, V, 20, torch.float32, seed=V + 1, rest=False)
    check(logits, idx, u, lse)


@pytest.mark.parametrize("T", [40, 200, 700, 2500])
def test_row_counts(T):
    """Row counts on both sides of every choice of CTAs per row."""
    logits, idx, u, lse = make(T, 2048 + 13, 9, torch.bfloat16, seed=T)
    check(logits, idx, u, lse)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("T,V,ctas", [(50, 70000, 3), (38, 100003, 4), (30, 128256, 5), (25, 150001, 6), (22, 180000, 7), (19, 250000, 8)])
def test_ctas_of_a_row(T, V, ctas, rest):
    """Every number of CTAs that long 16-bit rows are cut into, beside the whole rows of the tests above, in place too."""
    logits, idx, u, lse = make(T, V, 12, torch.bfloat16, seed=V, rest=rest)
    loss, d = check(logits, idx, u, lse)
    again = logits.clone()
    distill.topk_loss_grad(again, idx, u, teacher_lse=lse, out=again)
    assert torch.equal(again, d)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,off", [(400003, 0), (1 << 20, 0), ((1 << 20) - 3, 1)])
def test_rows_longer_than_shared_memory(V, off, dtype):
    """Slices that are held in part only (fp32 beyond about 390000 tokens), up to the longest rows; in place too."""
    logits, idx, u, lse = make(3, V, 40, dtype, seed=V, pad=5)
    buf = torch.zeros(3 * (V + 5) + 8, dtype=dtype, device="cuda")[off:off + 3 * (V + 5)].view(3, V + 5)[:, :V]
    buf.copy_(logits)
    idx[0, 0], idx[1, 0], idx[2, 1] = 0, V - 1, V // 2
    loss, d = check(buf, idx, u, lse + 1.0)
    d2 = distill.topk_grad(buf, idx, u, distill.topk_loss(buf, idx, u, teacher_lse=lse + 1.0)[1], teacher_lse=lse + 1.0)
    check(buf, idx, u, lse + 1.0, got=(loss, d2))
    distill.topk_loss_grad(buf, idx, u, teacher_lse=lse + 1.0, out=buf)
    assert torch.equal(buf, d)


@pytest.mark.parametrize("tau", [0.5, 2.0])
def test_temperature_and_teacher_types(tau):
    logits, idx, u, lse = make(6, 777, 12, torch.bfloat16, seed=5, tau=tau)
    check(logits, idx, u, lse, tau=tau)
    for dt in (torch.bfloat16, torch.float16):
        ub = u.to(dt)
        check(logits, idx.int(), ub, None, tau=tau)


def test_empty_slots_and_rows():
    logits, idx, u, lse = make(6, 500, 8, torch.float32, seed=7)
    idx[0, 3:] = -1
    idx[1] = -5                        # no live slot
    idx[2, 0] = 500                    # beyond the vocabulary: empty
    idx[3, 2] = 2 ** 40
    u[4, 1] = -math.inf                # a slot of probability 0
    u[5] = -math.inf
    loss, d = check(logits, idx, u, None)
    assert loss[1] == 0 and not d[1].any() and loss[5] == 0 and not d[5].any()
    loss, d = check(logits[:5], idx[:5], u[:5], lse[:5])
    assert loss[1].abs() < 1e-6


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_weights_and_masked_rows(dtype):
    logits, idx, u, lse = make(5, 1003, 6, dtype, seed=8)
    w = torch.tensor([0.0, 1.0, 0.25, 0.0, 3.0], device="cuda")
    logits[0] = float("nan")
    logits[3] = -math.inf
    clean = logits.clone()
    clean[0] = 0
    want = plain(clean, idx, u, lse, w)
    loss, d = distill.topk_loss_grad(logits, idx, u, teacher_lse=lse, weight=w)
    assert loss[0] == 0 and loss[3] == 0 and not d[0].any() and not d[3].any()
    assert bool(((loss.cpu().double() - want[0]).abs() <= 3e-4).all())
    assert torch.isfinite(d).all()


@pytest.mark.parametrize("rest", [False, True])
def test_masked_vocabulary(rest):
    """Tokens the student excludes: no share of the gradient; a kept one among them makes the loss infinite."""
    logits, idx, u, lse = make(4, 900, 5, torch.float32, seed=9, rest=rest)
    keep = torch.zeros(4, 900, dtype=torch.bool, device="cuda").scatter_(1, idx, True)
    keep[:, ::3] = True
    logits[~keep] = -math.inf
    logits[1, idx[1, 0]] = -math.inf
    logits[2] = -math.inf               # nothing left
    logits[3] = torch.where(keep[3], logits[3], torch.finfo(torch.float32).min)
    loss, d = check(logits, idx, u, lse)
    assert loss[1] == math.inf and loss[2] == math.inf and torch.isfinite(d).all()
    assert not d[0][~keep[0]].any()


def test_student_gives_the_rest_nothing():
    logits, idx, u, lse = make(1, 300, 4, torch.float32, seed=10)
    rest = torch.ones(300, dtype=torch.bool, device="cuda")
    rest[idx[0]] = False
    logits[0, rest] = -math.inf
    loss, d = distill.topk_loss_grad(logits, idx, u, teacher_lse=lse)
    assert loss[0] == math.inf and torch.isfinite(d).all() and not d[0, rest].any()

def in_logs(logits, idx, teacher, lse=None, weight=None, tau=1.0):
    """Loss and gradient from the definition in 64 bits and in logarithms of probabilities, so that no mass of the student is too
    small; and the gradient's parts (q_j P, p_j and the rest's spread), of which each is rounded by itself."""
    T, V = logits.shape
    z = logits.double().cpu() / tau
    idx, u = idx.cpu().long(), teacher.double().cpu() / tau
    live = (idx >= 0) & (idx < V)
    at = torch.where(live, idx, torch.zeros_like(idx))
    p = torch.exp(u - lse.double().cpu()[:, None]) if lse is not None else torch.softmax(u.masked_fill(~live, -math.inf), 1)
    p = torch.where(live, p, torch.zeros_like(p))
    rest = (1 - p.sum(1)).clamp(min=0) if lse is not None else torch.zeros(T, dtype=torch.float64)
    top = torch.zeros(T, V, dtype=torch.float64).scatter_add_(1, at, live.double()) > 0
    first = z.amax(1, keepdim=True)  # differences before anything else: z may be 1e30
    log_s = torch.log(torch.exp(z - first).sum(1, keepdim=True))
    log_q = z - first - log_s
    z_r = z.masked_fill(top, -math.inf)
    first_r = z_r.amax(1, keepdim=True)
    e_r = torch.exp(z_r - torch.where(first_r > -math.inf, first_r, torch.zeros_like(first_r)))
    s_r = e_r.sum(1, keepdim=True)
    log_r = (first_r - first + torch.log(s_r) - log_s)[:, 0]
    w = torch.ones(T, dtype=torch.float64) if weight is None else weight.double().cpu()
    row = torch.where(p > 0, p * (torch.log(p) - log_q.gather(1, at)), torch.zeros_like(p)).sum(1)
    row += torch.where(rest > 0, rest * (torch.log(rest) - log_r), torch.zeros_like(rest))
    target = torch.zeros(T, V, dtype=torch.float64).scatter_add_(1, at, p)
    spread = torch.where((s_r == 0) | (rest == 0)[:, None], torch.zeros_like(z), e_r / s_r * rest[:, None])
    own = log_q.exp() * (p.sum(1) + rest)[:, None]
    return w * row, (own - target - spread) * (w / tau)[:, None], (own + target + spread) * (w / tau)[:, None].abs(), top


def check_logs(logits, idx, teacher, lse=None, tau=1.0):
    """The fused form, the loss alone and the gradient alone against in_logs.  An exponent of at most 126 in fp32 is good to 126
    2^-24 = 7.5e-6, so an exponential, a sum of them and a part of the gradient to 2e-5 of itself (what is below 2^-100 counts as
    0: exponentials end at 2^-126); a loss to 4e-7 of itself besides the 1e-4 above."""
    want_l, want_d, parts, _ = in_logs(logits, idx, teacher, lse, None, tau)
    kw = dict(teacher_lse=lse, temperature=tau)
    loss, d = distill.topk_loss_grad(logits, idx, teacher, **kw)
    loss0, stats = distill.topk_loss(logits, idx, teacher, **kw)
    assert torch.equal(loss, loss0)
    limit = torch.finfo(torch.float32).max
    inf = want_l.abs() > limit
    assert torch.equal(torch.isinf(loss.cpu()), inf) and not torch.isnan(loss).any()
    assert bool(((loss.double().cpu() - want_l).abs() <= 1e-4 + 4e-7 * want_l.abs())[~inf].all())
    out = torch.empty_like(logits)
    for g in (d, distill.topk_grad(logits, idx, teacher, stats, **kw),
              distill.topk_loss_grad(logits, idx, teacher, out=out.copy_(logits), **kw)[1],
              distill.topk_grad(out.copy_(logits), idx, teacher, stats, out=out, **kw)):
        g = g.double().cpu()
        assert torch.isfinite(g).all()
        tol = 2e-5 * parts + HALF_ULP[logits.dtype] * 1.01 * want_d.abs() + 2.0 ** -100 / tau
        tol += 2.0 ** -25 if logits.dtype == torch.float16 else 0
        assert bool(((g - want_d).abs() <= tol).all()), float(((g - want_d).abs() / tol).max())


def far(T, V, K, dtype, at, seed, share=0.3, spread=1.0):
    """Rows whose tokens outside the slots all lie near `at`, while the teacher leaves them `share` of its mass."""
    g = torch.Generator().manual_seed(seed)
    idx = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(T)])
    z = at + spread * torch.randn(T, V, generator=g)
    z = z.clamp(min=torch.finfo(dtype).min).scatter_(1, idx, torch.randn(T, K, generator=g) * 3)
    u = torch.randn(T, K, generator=g) * 2
    lse = torch.logsumexp(u, 1) - math.log(1 - share)
    return z.to(dtype).cuda(), idx.cuda(), u.cuda(), lse.cuda()


FAR = [-40.0, -60.0, -85.0, -100.0, -1e4, -1e9, -1e10, -1e30, -3e38]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("at", FAR)
def test_rest_far_below_the_slots(at, dtype):
    """A vocabulary masked with a finite value, the slots' tokens alone allowed: the teacher's remaining mass is spread over the
    rest, however small the student's own mass there is."""
    if dtype == torch.float16 and at < -65000.0:
        at = -65504.0
    for share in (0.3, 2e-7):
        check_logs(*far(3, 301, 5, dtype, at, seed=21, share=share))
    check_logs(*far(2, 40003, 40, dtype, at, seed=22))


@pytest.mark.parametrize("at", [-85.0, -1e4, -1e30])
def test_rest_far_below_the_slots_in_long_rows(at):
    check_logs(*far(40, 128256, 20, torch.bfloat16, at, seed=23))


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("mask", [-1e4, -1e10, -1e30, -3.3e38])
def test_vocabulary_masked_with_a_large_number(mask, dtype, rest):
    """Most tokens masked, so that whole threads' and CTAs' shares of a row are; a few left, in the slots and beside them."""
    mask = max(mask, torch.finfo(dtype).min)
    for V, keep in ((3001, 12), (60000, 40)):
        logits, idx, u, lse = make(4, V, 6, dtype, seed=24, rest=rest)
        allowed = torch.zeros(4, V, dtype=torch.bool, device="cuda").scatter_(1, idx, True)
        allowed[:, torch.randperm(V, generator=torch.Generator().manual_seed(25))[:keep].cuda()] = True
        logits.copy_(torch.where(allowed, logits, torch.full_like(logits, mask)))
        check_logs(logits, idx, u, lse)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("at", [-3e38, -1e30, -4e9, 3e9, 1e30])
def test_rows_of_large_numbers(at, rest):
    """All logits far from 0, equal ones and ones that differ by units of their type."""
    logits, idx, u, lse = make(3, 2100, 9, torch.float32, seed=26, rest=rest)
    z = torch.full_like(logits, at)
    z[1] *= 1 + 2.0 ** -23 * torch.randint(0, 2, (2100,), device="cuda", generator=torch.Generator("cuda").manual_seed(27))
    z[2, idx[2, :3]] = 0.9 * at
    check_logs(z, idx, u, lse)


@pytest.mark.parametrize("rest", [False, True])
def test_low_temperature(rest):
    logits, idx, u, lse = make(4, 1500, 8, torch.float32, seed=28, rest=False)
    tau = 2.0 ** -30  # a value of fp32, in which the temperature is held
    if rest:
        lse = (torch.logsumexp(u.double() / tau, 1) + 0.4).float()
        lse = torch.where(lse.double() < u.double().amax(1) / tau, torch.nextafter(lse, torch.full_like(lse, math.inf)), lse)
    check_logs(logits, idx, u, lse, tau=tau)


@pytest.mark.parametrize("K", [2, 10, 100, 777, 1000])
@pytest.mark.parametrize("spread", [0.0, 3.0])
def test_student_that_equals_its_teacher(K, spread):
    """The loss is 0 but for the rounding of the student's sum to fp32 (twice half a unit, 2^-24) and that of p's sum."""
    z = spread * torch.randn(3, K, generator=torch.Generator().manual_seed(K))
    idx = torch.arange(K, device="cuda").repeat(3, 1)
    loss = distill.topk_loss(z.cuda(), idx, z.cuda())[0]
    assert float(loss.abs().max()) <= 2.0 ** -23


def test_student_that_equals_its_teacher_with_a_rest():
    """2^-22 from the exponentials of the rest and as much from their sums in fp32."""
    z = 2 * torch.randn(5, 5000, generator=torch.Generator().manual_seed(3))
    u, idx = z.topk(64, 1)
    loss = distill.topk_loss(z.cuda(), idx.cuda(), u.cuda(), teacher_lse=torch.logsumexp(z.double(), 1).float().cuda())[0]
    assert float(loss.abs().max()) <= 2.0 ** -21


def test_nan_reaches_its_row_only():
    logits, idx, u, lse = make(3, 700, 4, torch.bfloat16, seed=11)
    logits[1, 690] = float("nan")
    loss, d = distill.topk_loss_grad(logits, idx, u, teacher_lse=lse)
    assert torch.isnan(loss[1]) and torch.isnan(d[1]).all()
    assert torch.isfinite(loss[[0, 2]]).all() and torch.isfinite(d[[0, 2]]).all()


@pytest.mark.parametrize("rest", [False, True])
def test_slots_that_name_one_token(rest):
    logits, idx, u, lse = make(3, 640, 12, torch.float32, seed=12, rest=rest)
    idx[0, 5] = idx[0, 1]
    idx[0, 9] = idx[0, 1]
    idx[1, :] = 17
    if rest:
        lse += 1.5
    loss, d = check(logits, idx, u, lse)
    again = distill.topk_loss_grad(logits, idx, u, teacher_lse=lse)
    assert torch.equal(loss, again[0]) and torch.equal(d, again[1])


@pytest.mark.parametrize("V", [1, 7, 40])
def test_slots_hold_every_token(V):
    logits, idx, u, lse = make(3, V, V, torch.float32, seed=13)
    check(logits, idx, u, lse)
    idx2 = torch.cat([idx, idx[:, :1]], 1)
    idx2[:, -1] = -1
    check(logits, idx2, torch.cat([u, u[:, :1]], 1), lse)


@pytest.mark.parametrize("off_in,off_out", [(0, 0), (1, 1), (3, 3), (1, 0), (0, 5)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_alignments(dtype, off_in, off_out):
    T, V, K = 3, 1537, 7
    logits, idx, u, lse = make(T, V, K, dtype, seed=14)
    buf = torch.zeros(T * (V + 3) + 16, dtype=dtype, device="cuda")
    view = buf[off_in:off_in + T * (V + 3)].view(T, V + 3)[:, :V]
    view.copy_(logits)
    obuf = torch.full((T * (V + 3) + 16,), 7.0, dtype=dtype, device="cuda")
    out = obuf[off_out:off_out + T * (V + 3)].view(T, V + 3)[:, :V]
    loss, d = distill.topk_loss_grad(view, idx, u, teacher_lse=lse, out=out)
    assert d is out
    check(logits, idx, u, lse, got=(loss, out))
    rest = obuf.clone()
    rest[off_out:off_out + T * (V + 3)].view(T, V + 3)[:, :V] = 7.0
    assert (rest == 7.0).all()  # nothing is written beside the rows
    own = distill.topk_loss_grad(view, idx, u, teacher_lse=lse)[1]
    assert torch.equal(own, out)


@pytest.mark.parametrize("V", [1000, 128256])
def test_in_place(V):
    logits, idx, u, lse = make(9, V, 8, torch.bfloat16, seed=15)
    want = distill.topk_loss_grad(logits, idx, u, teacher_lse=lse)
    got = distill.topk_loss_grad(logits, idx, u, teacher_lse=lse, out=logits)
    assert got[1] is logits and torch.equal(got[0], want[0]) and torch.equal(logits, want[1])


def test_other_stream():
    logits, idx, u, lse = make(64, 5000, 8, torch.bfloat16, seed=16)
    want = distill.topk_loss_grad(logits, idx, u, teacher_lse=lse)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = distill.topk_loss_grad(logits, idx, u, teacher_lse=lse)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("rest", [False, True])
def test_gradient_against_differences(rest):
    """Central differences of the kernel's own loss: h = 0.05 along a random direction; the third derivative along a unit
    direction is below 1, so h^2 / 6 = 4e-4, and 1e-5 / h = 2e-4 from the losses' rounding."""
    logits, idx, u, lse = make(8, 400, 6, torch.float32, seed=17, rest=rest)
    v = torch.randn(8, 400, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    v[torch.arange(8), idx[:, 0]] += 5.0
    v = v / v.norm(dim=1, keepdim=True)
    d = distill.topk_loss_grad(logits, idx, u, teacher_lse=lse)[1]
    h = 0.05
    up = distill.topk_loss(logits + h * v, idx, u, teacher_lse=lse)[0]
    dn = distill.topk_loss(logits - h * v, idx, u, teacher_lse=lse)[0]
    assert ((up - dn) / (2 * h) - (d * v).sum(1)).abs().max() < 1e-3


def test_autograd():
    logits, idx, u, lse = make(7, 600, 5, torch.float32, seed=18)
    z = logits.clone().requires_grad_()
    w = torch.linspace(0, 2, 7, device="cuda")
    loss = distill.distill_loss(z, idx, u, teacher_lse=lse, weight=w)
    loss.mean().backward()
    want = distill.topk_loss_grad(logits, idx, u, teacher_lse=lse, weight=w / 7)[1]
    assert (z.grad - want).abs().max() < 1e-6


@pytest.mark.parametrize("form", ["both", "gradient"])
def test_outputs_written_in_place_tell_autograd(form):
    logits, idx, u, lse = make(3, 300, 4, torch.float32, seed=30)
    a = logits.clone().requires_grad_()
    z = a.exp()  # keeps its result for the backward pass
    stats = distill.topk_loss(z.detach(), idx, u, teacher_lse=lse)[1]
    if form == "both":
        distill.topk_loss_grad(z.detach(), idx, u, teacher_lse=lse, out=z.detach())
    else:
        distill.topk_grad(z.detach(), idx, u, stats, teacher_lse=lse, out=z.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()


@pytest.mark.parametrize("upstream", ["constant", "dependent"])
def test_second_derivatives_are_refused(upstream):
    logits, idx, u, lse = make(4, 200, 5, torch.float32, seed=29)
    a = logits.clone().requires_grad_()
    loss = distill.distill_loss(a * a.detach().abs(), idx, u, teacher_lse=lse)
    g, = torch.autograd.grad(loss.sum() if upstream == "constant" else loss.square().sum(), a, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(g.square().sum() + a.square().sum(), a)


@pytest.mark.parametrize("order", [0, 1])
def test_output_beside_the_logits(order):
    """Columns of one tensor: their rows alternate in memory and share nothing."""
    T, V = 5, 1000
    logits, idx, u, lse = make(T, V, 6, torch.bfloat16, seed=31)
    buf = torch.zeros(T, 2 * V + 3, dtype=torch.bfloat16, device="cuda")
    view, out = (buf[:, :V], buf[:, V:2 * V]) if order == 0 else (buf[:, V + 3:], buf[:, 3:V + 3])
    view.copy_(logits)
    got = distill.topk_loss_grad(view, idx, u, teacher_lse=lse, out=out)
    assert torch.equal(view, logits)
    check(logits, idx, u, lse, got=got)
    for bad in (buf[:, 1:V + 1], buf[:, V - 1:2 * V - 1], buf[:, V + 4:]):
        if bad.shape[1] == V and order == 0:
            with pytest.raises(ValueError):
                distill.topk_loss_grad(view, idx, u, teacher_lse=lse, out=bad)
    with pytest.raises(ValueError):
        distill.topk_loss_grad(view, idx, u, teacher_lse=lse, out=view[:1].expand(T, V))
    with pytest.raises(ValueError):
        distill.topk_loss_grad(view[:1], idx[:1], u[:1], out=buf[:1, 1:V + 1] if order == 0 else buf[:1, V:2 * V])


def test_no_rows():
    loss, d = distill.topk_loss_grad(torch.empty(0, 9, device="cuda"), torch.empty(0, 2, dtype=torch.int64, device="cuda"),
                                     torch.empty(0, 2, device="cuda"))
    assert loss.shape == (0,) and d.shape == (0, 9)


def test_refusals():
    logits, idx, u, lse = make(4, 100, 5, torch.float32, seed=19)
    f = distill.topk_loss_grad
    for bad in [dict(logits=logits.double()), dict(idx=idx.float()), dict(u=u.double())]:
        a = dict(logits=logits, idx=idx, u=u) | bad
        with pytest.raises(TypeError):
            f(a["logits"], a["idx"], a["u"])
    for bad in [dict(logits=logits[:3]), dict(idx=idx[:, :4]), dict(logits=logits.t()), dict(logits=logits[:1].expand(4, 100)),
                dict(logits=logits[0]), dict(idx=idx[:, :0], u=u[:, :0])]:
        a = dict(logits=logits, idx=idx, u=u) | bad
        with pytest.raises(ValueError):
            f(a["logits"], a["idx"], a["u"])
    for kw in [dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")), dict(weight=lse[:2]),
               dict(weight=lse.double()), dict(teacher_lse=lse[:, None]), dict(out=logits.half()), dict(out=logits[:, 1:])]:
        with pytest.raises(ValueError):
            f(logits, idx, u, **kw)
    wide = torch.zeros(5, 100, device="cuda")
    with pytest.raises(ValueError):  # overlaps the logits without being them
        f(wide[:4], idx, u, out=wide[1:])
    with pytest.raises(RuntimeError, match="CUDA"):
        f(logits.cpu(), idx, u)
    with pytest.raises(ValueError):
        f(torch.zeros(1, 1100, device="cuda"), torch.zeros(1, 1025, dtype=torch.int64, device="cuda"),
          torch.zeros(1, 1025, device="cuda"))
