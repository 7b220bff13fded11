"""The operators at the vocabulary's two ends of a quantized model, as cases that can be timed and compared.

Recovering a quantized model's quality by a few training steps, and judging it afterwards, takes three operators beside
the quantizer's own:

* ``distill``  the divergence from a teacher's top logits, and its gradient by the student's logits;
* ``embed``    the lookup of scaled token rows, and the table's gradient by sorted tokens;
* ``fp8``      the product with a weight held in 8-bit floating point (e4m3) with one scale per 128 x 128 block, the
               activations quantized in the call with one scale per row and 128 columns, and its gradient by the input.

``own = False`` runs them in plain torch operations in 32 bits; ``own = True`` through ``ltq_research_b200``.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
BLOCK = 128
E4M3_MAX = 448.0
TINY = 2.0 ** -126


# ---------------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # a few positions scored against a teacher while text is generated: latency
        _distill("distill_loss_few", rows=4, vocab=128256, k=20, dtype="bf16", grad=False, rest=False),
        # an evaluation batch: the divergence with the teacher's remaining mass as one more outcome
        _distill("distill_loss_eval", rows=2048, vocab=128256, k=64, dtype="bf16", grad=False, rest=True),
        # a recovery step's loss and gradient, a part of the rows masked out (prompt positions)
        _distill("distill_step", rows=4096, vocab=128256, k=64, dtype="bf16", grad=True, rest=True, masked=0.25),
        # an odd vocabulary inside padded rows, fp32 logits, a softened teacher with slots left empty
        _distill("distill_step_odd", rows=777, vocab=50003, k=17, dtype="fp32", grad=True, rest=False, pad=64, empty=0.2,
                 temperature=2.0, masked=0.1),
        # one decoding step of a batch of sequences: latency
        _embed("embed_decode", tokens=16, vocab=262144, dim=2560, dtype="bf16", scale=math.sqrt(2560.0)),
        # a batch of prompts
        _embed("embed_prompts", tokens=16384, vocab=262144, dim=2560, dtype="bf16", scale=math.sqrt(2560.0)),
        # a training step's table gradient, natural text: a few tokens take a large part of the positions
        _embed("embed_grad", tokens=16384, vocab=128256, dim=2048, dtype="bf16", out="fp32", grad=True, scale=1.0),
        # odd sizes, the gradient kept in the table's 16 bits, padding positions that take no gradient
        _embed("embed_grad_odd", tokens=4099, vocab=50003, dim=1000, dtype="bf16", out="bf16", grad=True,
               scale=math.sqrt(1000.0), padding=0.15),
        # one token through a projection
        _fp8("fp8_one_token", rows=1, n=8192, k=2048, dtype="bf16"),
        # the output head for a few tokens
        _fp8("fp8_head_few", rows=24, n=128256, k=2048, dtype="bf16"),
        # a projection over a batch of prompts
        _fp8("fp8_prompts", rows=8192, n=8192, k=4096, dtype="bf16"),
        # the gradient that reaches the hidden states through the frozen output head, odd row count
        _fp8("fp8_head_grad", rows=1003, n=128256, k=2048, dtype="bf16", grad=True),
    ]


def _distill(name, rows, vocab, k, dtype, grad, rest, pad=1, empty=0.0, temperature=1.0, masked=0.0):
    c = dict(op="distill", rows=rows, vocab=vocab, k=k, dtype=dtype, grad=grad, rest=rest, pad=pad, empty=empty,
             temperature=temperature, masked=masked)
    return dict(c, name=name) if name else c


def _embed(name, tokens, vocab, dim, dtype, scale, grad=False, out="", padding=0.0):
    c = dict(op="embed", tokens=tokens, vocab=vocab, dim=dim, dtype=dtype, scale=scale, grad=grad, out=out,
             padding=padding)
    return dict(c, name=name) if name else c


def _fp8(name, rows, n, k, dtype, grad=False):
    c = dict(op="fp8", rows=rows, n=n, k=k, dtype=dtype, grad=grad)
    return dict(c, name=name) if name else c


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm; about one in three a multiple of 64 where it can be."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v >= 128 and rng.random() < 1 / 3:
        v = v // 64 * 64
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["distill", "embed", "fp8"])
    if op == "distill":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        vocab = _log(rng, 1000, 262144)
        rows = _log(rng, 1, max(1, min(8192, 4096 * 128256 * 2 // (vocab * BYTES[dtype]))))
        return _distill(None, rows=rows, vocab=vocab, k=_log(rng, 1, 256), dtype=dtype, grad=rng.random() < 0.6,
                        rest=rng.random() < 0.5, pad=rng.choice([1, 8, 64]), empty=rng.choice([0.0, 0.0, 0.3]),
                        temperature=rng.choice([1.0, 1.0, 0.7, 2.0]), masked=rng.choice([0.0, 0.2, 0.6]))
    if op == "embed":
        grad = rng.random() < 0.6
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        vocab = _log(rng, 1000, 262144)
        dim = _log(rng, 64, min(8192, 128256 * 2048 // vocab))
        tokens = _log(rng, 1, min(65536, 2 ** 26 // dim))
        return _embed(None, tokens=tokens, vocab=vocab, dim=dim, dtype=dtype, scale=rng.choice([1.0, math.sqrt(dim)]),
                      grad=grad, out=rng.choice(["fp32", dtype]) if grad else "",
                      padding=rng.choice([0.0, 0.2]) if grad else 0.0)
    k = _log(rng, 64, 8192)
    n = _log(rng, 64, min(128256, 128256 * 2048 // k))
    rows = _log(rng, 1, max(1, min(8192, 8192 * 8192 * 4096 // (n * k))))
    return _fp8(None, rows=rows, n=n, k=k, dtype=rng.choice(["bf16", "bf16", "fp16"]), grad=rng.random() < 0.4)


def work(case):
    """Bytes and operations that one pass cannot do without: inputs read once, outputs written once."""
    if case["op"] == "distill":
        rows, live = case["rows"], case["rows"] - _masked_rows(case)  # rows without weight need not be read
        e = BYTES[case["dtype"]]
        b = live * (case["vocab"] * e + case["k"] * 8 + (4 if case["rest"] else 0)) + rows * 8
        f = live * case["vocab"] * 4
        if case["grad"]:
            b += rows * case["vocab"] * e
            f += live * case["vocab"] * 4
        return {"bytes": b, "flops": f}
    if case["op"] == "embed":
        n, d = case["tokens"], case["dim"]
        if case["grad"]:
            return {"bytes": n * 8 + n * d * BYTES[case["dtype"]] + case["vocab"] * d * BYTES[case["out"]], "flops": n * d}
        return {"bytes": n * 8 + 2 * n * d * BYTES[case["dtype"]], "flops": n * d}
    m, n, k = case["rows"], case["n"], case["k"]
    e = BYTES[case["dtype"]]
    blocks = math.ceil(n / BLOCK) * math.ceil(k / BLOCK)
    return {"bytes": e * m * k + n * k + 4 * blocks + e * m * n, "flops": 2 * m * n * k}


# --------------------------------------------------------------------------------------------------------- the inputs

def _masked_rows(case):
    return int(case["rows"] * case["masked"])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"distill": _prepare_distill, "embed": _prepare_embed, "fp8": _prepare_fp8}[case["op"]](case, g)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _prepare_distill(case, g):
    """Student logits with a few likely tokens in each row above a broad floor; a teacher that differs from them by a
    noise, its top k logits in falling order and the log-sum-exp of all of them at the same temperature."""
    rows, vocab, k = case["rows"], case["vocab"], case["k"]
    ld = (vocab + case["pad"] - 1) // case["pad"] * case["pad"]
    logits = torch.zeros(rows, ld, dtype=DT[case["dtype"]], device="cuda")[:, :vocab]
    idx = torch.empty(rows, k, dtype=torch.int64, device="cuda")
    teacher = torch.empty(rows, k, device="cuda")
    lse = torch.empty(rows, device="cuda")
    step = max(1, 2 ** 27 // vocab)
    for a in range(0, rows, step):
        b = min(rows, a + step)
        z = _randn(g, b - a, vocab) * 2
        hot = (_rand(g, b - a, 24) * vocab).long()
        z.scatter_add_(1, hot, 6 - 3 * torch.log(_rand(g, b - a, 24) + 1e-6))
        logits[a:b] = z.to(logits.dtype)
        z += _randn(g, b - a, vocab) * 0.5
        teacher[a:b], idx[a:b] = torch.topk(z, k, dim=1)
        lse[a:b] = torch.logsumexp(z / case["temperature"], 1)
    if case["empty"]:  # a teacher that kept fewer tokens for some rows: the slots behind them are empty
        kept = (_rand(g, rows) * k * 1.5 + (_rand(g, rows) > case["empty"] * 0.1)).long()
        slot = torch.arange(k, device="cuda")
        kept = torch.where(_rand(g, rows) < case["empty"], kept, torch.full_like(kept, k))
        idx = torch.where(slot[None] < kept[:, None], idx, torch.full_like(idx, -1))
    weight = torch.ones(rows, device="cuda")
    weight[torch.randperm(rows, generator=g, device="cuda")[:_masked_rows(case)]] = 0.0
    return dict(case=case, logits=logits, idx=idx, teacher=teacher, lse=lse if case["rest"] else None,
                weight=weight)


def _text_tokens(g, n, vocab):
    """Token ids as text has them: probability about 1 / (rank + 3), the ranks in a random order of ids."""
    p = 1.0 / (torch.arange(vocab, device="cuda", dtype=torch.float64) + 3.0)
    cdf = torch.cumsum(p / p.sum(), 0)
    rank = torch.searchsorted(cdf, _rand(g, n).double()).clamp_(max=vocab - 1)
    return torch.randperm(vocab, generator=g, device="cuda")[rank]


def _prepare_embed(case, g):
    n, vocab, dim = case["tokens"], case["vocab"], case["dim"]
    tokens = _text_tokens(g, n, vocab)
    if not case["grad"]:
        return dict(case=case, tokens=tokens, table=(_randn(g, vocab, dim) * 0.02).to(DT[case["dtype"]]))
    pad = -1
    if case["padding"]:  # the ends of shorter sequences in the batch
        pad = 0
        tokens[n - int(n * case["padding"]):] = pad
    return dict(case=case, tokens=tokens, pad=pad, dout=(_randn(g, n, dim) * 1e-3).to(DT[case["dtype"]]))


def _prepare_fp8(case, g):
    """Weights of a trained projection's spread, quantized as a checkpoint holds them; activations with a few channels
    far above the others.  The program keeps the weight's handle."""
    m, n, k = case["rows"], case["n"], case["k"]
    w = _randn(g, n, k) * (0.02 * torch.exp(_randn(g, n, 1) * 0.3))
    q, s = _plain_blocks(w)
    q = q.to(torch.float8_e4m3fn)
    cols = n if case["grad"] else k
    x = _randn(g, m, cols)
    if case["grad"]:  # softmax-minus-target gradients: small, with a few large entries in each row
        x = x * 1e-5 + (_rand(g, m, cols) < 3e-4) * _randn(g, m, cols) * 0.05
    else:
        x = x * (1 + 20 * (_rand(g, cols) < 0.005))
    state = dict(case=case, x=x.to(DT[case["dtype"]]), q=q, s=s)
    if own:
        from ltq_research_b200 import fp8
        state["weight"] = fp8.BlockWeight(q, s, backward=case["grad"])
    return state


# ------------------------------------------------------------------------------------------------------------ the pass

def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "distill":
        return _plain_distill(state, case["grad"])
    if case["op"] == "embed":
        return _plain_embed_grad(state) if case["grad"] else _plain_embed(state)
    return _plain_fp8(state)


def _run_own(case, state):
    if case["op"] == "distill":
        from ltq_research_b200 import distill
        kw = dict(teacher_lse=state["lse"], weight=state["weight"], temperature=case["temperature"])
        if case["grad"]:
            return distill.topk_loss_grad(state["logits"], state["idx"], state["teacher"], **kw)
        return distill.topk_loss(state["logits"], state["idx"], state["teacher"], **kw)[0]
    if case["op"] == "embed":
        from ltq_research_b200 import embedding
        if case["grad"]:
            return embedding.lookup_grad(state["tokens"], state["dout"], case["vocab"], scale=case["scale"],
                                         padding_idx=state["pad"] if state["pad"] >= 0 else None, dtype=DT[case["out"]])
        return embedding.lookup(state["table"], state["tokens"], scale=case["scale"])
    from ltq_research_b200 import fp8
    if case["grad"]:
        return fp8.linear_grad(state["x"], state["weight"])
    return fp8.linear(state["x"], state["weight"])


# ----------------------------------------------------------------------------- the plain forms: torch operations, 32 bits

def _plain_distill(state, grad):
    case, idx, w = state["case"], state["idx"], state["weight"]
    rows, vocab = state["logits"].shape
    z = state["logits"].float() / case["temperature"]
    live = (idx >= 0) & (idx < vocab)
    at = torch.where(live, idx, torch.zeros_like(idx))
    t = torch.where(live, state["teacher"] / case["temperature"], torch.full_like(state["teacher"], -math.inf))
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True)
    log_q = torch.gather(z, 1, at) - m - torch.log(total)
    if case["rest"]:
        p = torch.exp(t - state["lse"][:, None])
        rest = (1 - p.sum(1, keepdim=True)).clamp(min=0)
        top = torch.zeros(rows, vocab + 1, dtype=torch.bool, device=z.device)
        top = top.scatter_(1, torch.where(live, idx, torch.full_like(idx, vocab)), True)[:, :vocab]
        q_rest = torch.where(top, torch.zeros_like(e), e).sum(1, keepdim=True) / total
        tail = torch.where(rest > 0, rest * (torch.log(rest) - torch.log(q_rest)), torch.zeros_like(rest))
    else:
        tm = t.amax(1, keepdim=True)
        p = torch.where(live, torch.exp(t - torch.where(torch.isfinite(tm), tm, torch.zeros_like(tm))), torch.zeros_like(t))
        p = p / p.sum(1, keepdim=True).clamp(min=TINY)
        rest, tail = torch.zeros_like(m), torch.zeros_like(m)
    terms = torch.where(p > 0, p * (torch.log(p) - log_q), torch.zeros_like(p))
    used = w != 0
    loss = torch.where(used, w * (terms.sum(1) + tail[:, 0]), torch.zeros_like(w))
    if not grad:
        return loss
    mass = p.sum(1, keepdim=True) + rest
    d = e / total
    if case["rest"]:
        outside = torch.where(rest > 0, rest / q_rest, torch.zeros_like(rest))
        d = d * torch.where(top, mass, mass - outside)
    else:
        d = d * mass
    d.scatter_add_(1, at, -p)
    d = torch.where(used[:, None], d * (w[:, None] / case["temperature"]), torch.zeros_like(d))
    return loss, d.to(state["logits"].dtype)


def _plain_embed(state):
    rows = state["table"][state["tokens"]].float() * state["case"]["scale"]
    return rows.to(state["table"].dtype)


def _plain_embed_grad(state):
    case, tokens = state["case"], state["tokens"]
    out = torch.zeros(case["vocab"], case["dim"], device=tokens.device)
    d = state["dout"].float() * (tokens != state["pad"])[:, None]
    out.index_add_(0, tokens, d)
    return (out * case["scale"]).to(DT[case["out"]])


def _pad_to(x, r, c):
    """x with zero rows and columns behind it, to multiples of r and c."""
    return torch.nn.functional.pad(x, (0, -x.shape[1] % c, 0, -x.shape[0] % r))


def _e4m3(x):
    return x.to(torch.float8_e4m3fn).float()


def _plain_blocks(w):
    """The e4m3 values (in 32 bits) of w [n, k] and one scale per 128 x 128 block."""
    n, k = w.shape
    b = _pad_to(w, BLOCK, BLOCK)
    b = b.reshape(b.shape[0] // BLOCK, BLOCK, b.shape[1] // BLOCK, BLOCK)
    s = (b.abs().amax((1, 3)) / E4M3_MAX).clamp(min=TINY)
    q = _e4m3(b / s[:, None, :, None])
    return q.reshape(q.shape[0] * BLOCK, -1)[:n, :k].contiguous(), s


def _plain_rows(x):
    """x with each row's 128 columns rounded to e4m3 times their scale, in 32 bits."""
    m, k = x.shape
    b = _pad_to(x.float(), 1, BLOCK)
    b = b.reshape(m, -1, BLOCK)
    s = (b.abs().amax(2, keepdim=True) / E4M3_MAX).clamp(min=TINY)
    return (_e4m3(b / s) * s).reshape(m, -1)[:, :k]


def _plain_fp8(state):
    q, s = state["q"], state["s"]
    n, k = q.shape
    w = q.float() * s.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    x = _plain_rows(state["x"])
    y = x @ w if state["case"]["grad"] else x @ w.T
    return y.to(state["x"].dtype)


# ------------------------------------------------------------------------------- the definitions, in 64 bits, row by row

def exact(case, seed):
    state = prepare(case, seed)
    return {"distill": _exact_distill, "embed": _exact_embed, "fp8": _exact_fp8}[case["op"]](case, state)


def _exact_distill(case, state):
    """KL(p || q) of each row: q the student's softmax at the temperature; p the teacher's, over its live slots alone, or
    over these and one outcome for all other tokens."""
    logits, idx, w = state["logits"], state["idx"], state["weight"].double()
    rows, vocab = logits.shape
    tau = case["temperature"]
    loss = torch.zeros(rows, dtype=torch.float64, device=logits.device)
    d = torch.zeros(rows, vocab, dtype=torch.float64, device=logits.device) if case["grad"] else None
    step = max(1, 2 ** 26 // vocab)
    for a in range(0, rows, step):
        b = min(rows, a + step)
        log_q = torch.log_softmax(logits[a:b].double() / tau, 1)
        live = (idx[a:b] >= 0) & (idx[a:b] < vocab)
        t = (state["teacher"][a:b].double() / tau).masked_fill(~live, -math.inf)
        if case["rest"]:
            p = torch.exp(t - state["lse"][a:b, None].double())
        else:
            p = torch.nan_to_num(torch.softmax(t, 1), nan=0.0)
        target = torch.zeros_like(log_q)
        target.scatter_add_(1, idx[a:b].clamp(min=0), p)  # empty slots add exact zeros
        top = torch.zeros_like(log_q).scatter_add_(1, idx[a:b].clamp(min=0), live.double()) > 0
        rest = (1 - p.sum(1)).clamp(min=0) if case["rest"] else torch.zeros(b - a, dtype=torch.float64, device=p.device)
        row = torch.xlogy(p, p).sum(1) - torch.where(target > 0, target * log_q, torch.zeros_like(target)).sum(1)
        log_rest = torch.logsumexp(log_q.masked_fill(top, -math.inf), 1)
        row += torch.where(rest > 0, torch.xlogy(rest, rest) - rest * log_rest, torch.zeros_like(rest))
        loss[a:b] = row * w[a:b]
        if d is not None:
            q = log_q.exp()
            # outside the top tokens the rest's mass is spread as the student spreads its own
            spread = (log_q - log_rest[:, None]).exp() * rest[:, None]
            target += torch.where(top | (rest[:, None] == 0), torch.zeros_like(spread), spread)
            d[a:b] = (q * (p.sum(1) + rest)[:, None] - target) * (w[a:b, None] / tau)
    return (loss, d) if case["grad"] else loss


def _exact_embed(case, state):
    if not case["grad"]:
        return torch.index_select(state["table"], 0, state["tokens"]).double() * case["scale"]
    kept = state["tokens"] != state["pad"]
    out = torch.zeros(case["vocab"], case["dim"], dtype=torch.float64, device="cuda")
    return out.index_put_((state["tokens"][kept],), state["dout"][kept].double(), accumulate=True) * case["scale"]


def _round_e4m3(v):
    """v rounded to the nearest number of three significand bits after the leading one (ties to even), the spacing
    2^-9 below 2^-6, the magnitude at most 448."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_fp8(case, state):
    x, q, s = state["x"], state["q"], state["s"].double()
    n, k = q.shape
    y = torch.zeros(x.shape[0], k if case["grad"] else n, dtype=torch.float64, device=x.device)
    for c in range(0, x.shape[1], BLOCK):
        xb = x[:, c:c + BLOCK].double()
        # the scale is held in 32 bits
        sx = (xb.abs().amax(1, keepdim=True) / E4M3_MAX).float().clamp(min=TINY).double()
        xb = _round_e4m3(xb / sx) * sx
        if case["grad"]:
            wb = q[c:c + BLOCK].double() * s[c // BLOCK].repeat_interleave(BLOCK)[:k]
        else:
            wb = (q[:, c:c + BLOCK].double() * s[:, c // BLOCK].repeat_interleave(BLOCK)[:n, None]).T
        y += xb @ wb
    return y
