"""The C entries of the token, logit and 8-bit operators refuse invalid sizes, types, strides and alignments with -1 before any
CUDA call (fake, never-dereferenced addresses); sizes of nothing succeed."""
import pytest

from ltq_research_b200 import _lib

A, B, C, D = 1 << 20, 1 << 21, 1 << 22, 1 << 23  # aligned stand-ins


def distill(**over):
    a = dict(logits=A, dtype=1, ld=1000, idx=B, idx64=1, ld_idx=8, teacher=C, tdt=0, ld_t=8, lse=None, weight=None, grad=None,
             gs=0, T=4, V=1000, K=8, temperature=1.0, mode=1, loss=D, stats=None, dlogits=A, ld_d=1000, stream=None)
    a.update(over)
    return _lib.lib().ltq_distill_topk(*a.values())


@pytest.mark.parametrize("over", [
    dict(dtype=3), dict(dtype=-1), dict(tdt=4), dict(T=-1), dict(V=0), dict(V=(1 << 20) + 1, ld=1 << 21, ld_d=1 << 21), dict(K=0),
    dict(K=1025, ld_idx=2000, ld_t=2000), dict(mode=3), dict(mode=-1), dict(temperature=0.0), dict(temperature=-1.0),
    dict(temperature=float("inf")), dict(temperature=float("nan")), dict(ld=999), dict(ld_idx=7), dict(ld_t=7), dict(ld_d=999),
    dict(logits=None), dict(idx=None), dict(teacher=None), dict(loss=None), dict(dlogits=None), dict(logits=A + 1),
    dict(dlogits=A + 1), dict(mode=2, stats=None), dict(T=1 << 30)])
def test_distill_refuses(over):
    assert distill(**over) == -1


def test_nothing_to_do():
    L = _lib.lib()
    assert distill(T=0) == 0
    assert L.ltq_embed_lookup(A, 1, 64, B, 1, 0, 10, 64, 1.0, C, 64, None) == 0
    assert L.ltq_embed_grad(B, 1, 0, 10, -1, A, 1, 64, 64, 1.0, C, 0, 64, 1, None, 0, None) == 0
    assert L.ltq_fp8_quant_rows(A, 1, 256, 0, 256, B, 256, C, 4, None) == 0
    assert L.ltq_fp8_gemm(A, 256, B, 4, C, 256, D, 2, A, 1, 128, 0, 128, 256, None, 0, None, None) == 0
    assert L.ltq_fp8_few(A, 1, 256, B, 256, C, 2, D, 1, 128, 0, 128, 256, None, None) == 0
    assert L.ltq_embed_grad_workspace_bytes(0, 64) == 0 and L.ltq_embed_grad_workspace_bytes(10, 0) == 0


def test_embed_refuses():
    L = _lib.lib()

    def lookup(**over):
        a = dict(table=A, dtype=1, ld=64, tokens=B, tok64=1, n=5, V=10, D=64, scale=1.0, out=C, ld_out=64, stream=None)
        a.update(over)
        return L.ltq_embed_lookup(*a.values())
    for over in (dict(dtype=7), dict(n=-1), dict(V=0), dict(D=0), dict(ld=63), dict(ld_out=63), dict(table=None), dict(tokens=None),
                 dict(out=None), dict(table=A + 1), dict(out=C + 1), dict(tokens=B + 4)):
        assert lookup(**over) == -1, over

    ws = L.ltq_embed_grad_workspace_bytes(5, 64)
    assert ws > 0

    def grad(**over):
        a = dict(tokens=B, tok64=1, n=5, V=10, padding=-1, dout=A, dtype=1, ld_d=64, D=64, scale=1.0, out=C, odt=0, ld_out=64,
                 acc=0, ws=D, bytes=ws, stream=None)
        a.update(over)
        return L.ltq_embed_grad(*a.values())
    for over in (dict(dtype=7), dict(odt=7), dict(n=-1), dict(n=(1 << 30) + 1), dict(V=0), dict(V=(1 << 30) + 1), dict(D=0),
                 dict(D=(1 << 20) + 1, ld_d=1 << 21, ld_out=1 << 21), dict(ld_d=63), dict(ld_out=63), dict(tokens=None),
                 dict(dout=None), dict(out=None), dict(ws=None), dict(ws=D + 16), dict(bytes=ws - 1), dict(out=C + 2),
                 dict(dout=A + 1), dict(tokens=B + 4)):
        assert grad(**over) == -1, over


def test_fp8_refuses():
    L = _lib.lib()
    for args in ((A, 9, 256, 4, 256, B, 256, C, 4), (A, 1, 255, 4, 256, B, 256, C, 4), (A, 1, 256, -1, 256, B, 256, C, 4),
                 (A, 1, 256, 4, 0, B, 256, C, 4), (A, 1, 256, 4, 256, B, 250, C, 4), (A, 1, 256, 4, 256, B + 8, 256, C, 4),
                 (A, 1, 256, 4, 256, B, 256, C, 3), (A + 1, 1, 256, 4, 256, B, 256, C, 4), (None, 1, 256, 4, 256, B, 256, C, 4),
                 (A, 1, 256, 4, 256, B, 256, None, 4)):
        assert L.ltq_fp8_quant_rows(*args, None) == -1, args
    for args in ((A, 9, 256, 200, 256, B, 256, C, 2), (A, 1, 256, 200, 256, B, 256, C, 1), (A, 1, 256, 200, 256, None, 256, C, 2),
                 (A, 1, 256, 200, 256, B, 248, C, 2)):
        assert L.ltq_fp8_quant_blocks(*args, None) == -1, args
    for args in ((A, 256, 0, 256, B, 16), (A, 255, 16, 256, B, 16), (A, 254, 16, 254, B, 16), (A + 1, 256, 16, 256, B, 16),
                 (A, 256, 16, 256, B, 8), (A, 256, 17, 256, B, 16), (A, 256, 16, 256, B, 80), (A, 256, 16, 256, None, 16)):
        assert L.ltq_fp8_transpose(*args, None) == -1, args

    def gemm(**over):
        a = dict(A=A, lda=256, sa=B, ld_sa=8, B=C, ldb=256, sb=D, ld_sb=2, C=A, dtype=1, ldc=128, M=8, N=128, K=256, ws=None, bytes=0,
                 err=None, stream=None)
        a.update(over)
        return L.ltq_fp8_gemm(*a.values())
    for over in (dict(dtype=5), dict(M=-1), dict(N=-1), dict(K=0), dict(ldc=127), dict(ld_sa=7), dict(ld_sa=10, M=9),
                 dict(ld_sb=1), dict(A=None), dict(A=A + 8), dict(lda=264), dict(lda=240), dict(B=None), dict(ldb=250), dict(sa=None),
                 dict(sa=B + 4), dict(sb=None), dict(sb=D + 2), dict(C=None), dict(C=A + 1)):
        assert gemm(**over) == -1, over

    def few(**over):
        a = dict(x=A, dtype=1, ldx=256, W=B, ldw=256, sw=C, ld_sw=2, y=D, odt=1, ldy=128, M=4, N=128, K=256, err=None, stream=None)
        a.update(over)
        return L.ltq_fp8_few(*a.values())
    for over in (dict(dtype=5), dict(odt=5), dict(M=-1), dict(M=33), dict(K=0), dict(ldx=255), dict(ldy=127), dict(ld_sw=1), dict(x=None),
                 dict(x=A + 1), dict(W=None), dict(W=B + 8), dict(ldw=250), dict(sw=None), dict(y=None), dict(y=D + 1)):
        assert few(**over) == -1, over


def test_operators_need_cuda():
    import torch
    from ltq_research_b200 import distill, embedding, fp8
    z, i, u = torch.zeros(2, 9), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    for f in (lambda: distill.topk_loss(z, i, u), lambda: embedding.lookup(z, i), lambda: embedding.lookup_grad(i[0], z[:1].expand(3, 9), 4),
              lambda: fp8.quantize_rows(z), lambda: fp8.quantize_blocks(z)):
        with pytest.raises(RuntimeError, match="CUDA"):
            f()
