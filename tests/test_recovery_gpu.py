"""The vocabulary's two ends around a quantized body, run as one recovery step: the table's gradient against the same model
in plain torch operations, and a few steps that bring the student nearer to its teacher."""
import pytest
import torch

from ltq_research_b200 import fp8, recovery

pytestmark = pytest.mark.gpu


def setup(V=1003, D=256, T=64, K=16, seed=0):
    from ltq_research_b200.liqk_v2 import quantize_matrix_liqk_v2
    g = torch.Generator("cuda").manual_seed(seed)
    table = torch.randn(V, D, device="cuda", generator=g)
    W = torch.randn(D, D, device="cuda", generator=g) * D ** -0.5
    X = torch.randn(4 * D, D, device="cuda", generator=g)
    _, W_hat, _ = quantize_matrix_liqk_v2(W, X.T @ X / (4 * D), "TCQ25X")
    head_w = torch.randn(V, D, device="cuda", generator=g) * (2.0 * D ** -0.5)
    tokens = torch.randint(0, V, (4, T // 4), device="cuda", generator=g)
    z = torch.nn.functional.linear(torch.nn.functional.linear(table[tokens], W), head_w)
    u, idx = z.topk(K, -1)
    teacher = recovery.TeacherTop(idx, u, torch.logsumexp(z, -1))
    return table, recovery.QuantizedLinear(W_hat, torch.float32), head_w, tokens, teacher


def plain_rows(x):
    """x with each row's 128 columns rounded to e4m3 under their scale."""
    b = torch.nn.functional.pad(x, (0, -x.shape[-1] % 128)).reshape(*x.shape[:-1], -1, 128)
    s = (b.abs().amax(-1, keepdim=True) / 448).clamp(min=2.0 ** -126)
    return ((b / s).to(torch.float8_e4m3fn).float() * s).flatten(-2)[..., :x.shape[-1]]


class PlainHead(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, w):
        ctx.w = w
        return plain_rows(h) @ w.T

    @staticmethod
    def backward(ctx, dz):
        return plain_rows(dz) @ ctx.w, None


def test_step_gradient():
    """Against the same step in torch's own operators, the two 8-bit roundings among them.  What differs is fp32 rounding:
    1e-5 of the loss; in the gradient, of 64 x 1003 values rounded to e4m3 the one or two whose fp32 difference (1e-6) meets
    a tie (spacing 2^-3 of the value), which moves the gradient's norm by less than a hundredth."""
    table, body, head_w, tokens, teacher = setup()
    head = fp8.BlockWeight.quantize(head_w, backward=True)
    a = table.clone().requires_grad_()
    w = (torch.arange(tokens.numel(), device="cuda") % 4 != 0).float().view(tokens.shape)
    loss = recovery.step(a, tokens, body, head, teacher, weight=w)
    b = table.clone().requires_grad_()
    z = PlainHead.apply(body(b[tokens]), head.dequantize())
    logq = torch.log_softmax(z, -1)
    p = torch.exp(teacher.logits - teacher.lse[..., None])
    rest = 1 - p.sum(-1)
    top = torch.zeros_like(z, dtype=torch.bool).scatter_(-1, teacher.idx, True)
    kl = (p * (p.log() - logq.gather(-1, teacher.idx))).sum(-1)
    kl = kl + rest * (rest.log() - torch.logsumexp(logq.masked_fill(top, float("-inf")), -1))
    want = (kl * w).sum() / w.sum()
    want.backward()
    assert abs(float(loss) - float(want.detach())) < 1e-3 * float(want.detach())
    assert float((a.grad - b.grad).norm() / b.grad.norm()) < 0.01
    per = recovery.score(table, tokens, body, head, teacher, weight=w)
    assert per.shape == tokens.shape and abs(float(per.sum() / w.sum()) - float(loss)) < 1e-4 * float(loss) + 1e-5


def test_recovers():
    table, body, head_w, tokens, teacher = setup(seed=1)
    head = fp8.BlockWeight.quantize(head_w, backward=True)
    t = (table + 0.3 * torch.randn(table.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(5))).requires_grad_()
    opt = torch.optim.Adam([t], lr=0.02)
    first = float(recovery.score(t, tokens, body, head, teacher).mean())
    for _ in range(30):
        opt.zero_grad()
        recovery.step(t, tokens, body, head, teacher)
        opt.step()
    assert float(recovery.score(t, tokens, body, head, teacher).mean()) < 0.5 * first
    fp8.check_errors(t.device)


@pytest.mark.parametrize("dtype", [torch.bool, torch.int64, torch.bfloat16])
def test_weights_of_any_type(dtype):
    """A mask as data loaders give it, to the step and to the score."""
    table, body, head_w, tokens, teacher = setup(V=130, T=8)
    head = fp8.BlockWeight.quantize(head_w, backward=True)
    mask = (torch.arange(tokens.numel(), device="cuda") % 3 != 0).view(tokens.shape)
    want = recovery.score(table, tokens, body, head, teacher, weight=mask.float())
    got = recovery.score(table, tokens, body, head, teacher, weight=mask.to(dtype))
    assert torch.equal(got, want) and not got[~mask].any()
    loss = recovery.step(table.requires_grad_(), tokens, body, head, teacher, weight=mask.to(dtype))
    assert abs(float(loss) - float(want.sum() / mask.sum())) < 1e-5 * float(loss) + 1e-6


def test_table_must_train():
    table, body, head_w, tokens, teacher = setup(V=130, T=8)
    with pytest.raises(ValueError):
        recovery.step(table, tokens, body, fp8.BlockWeight.quantize(head_w, backward=True), teacher)
