"""Divergence of a quantized model from its teacher, and the gradient that recovers it, from the teacher's top logits
(the reference evaluates the same divergence on stored traces, src/eval_kld.py, over the whole vocabulary).

For a row of student logits z [V] and a teacher's K kept logits u_k of tokens id_k, with q = softmax(z / temperature):

* without ``teacher_lse`` the teacher is the softmax of its kept logits alone;
* with it (the log-sum-exp of ALL its logits / temperature) p_k = exp(u_k / temperature - lse), and the mass it did not
  keep is one more outcome, compared with the student's mass outside the kept tokens.

    loss = weight * ( sum_k p_k (log p_k - log q_{id_k})  +  p_r (log p_r - log q_r) )

A slot whose id is negative (or not below V) is empty.  Rows of weight 0 (prompt positions, padding) have loss and
gradient 0 and their logits are not read; a row without a live slot has loss and gradient 0; a kept token that the student
excludes (logit -inf) gives loss +inf and a finite gradient; NaN logits give NaN.  Finite logits of any size are taken as they
are: a vocabulary masked with -1e4, -1e30 or the type's lowest value has its share of the loss and of the gradient.
Exponentials and sums over the vocabulary are fp32; the teacher's probabilities, the slots' sums and the loss are formed in 64
bits from p rounded to fp32.

One entry (ltq_distill_topk): the loss reads the logits once, loss and gradient together read them once more from cache
or shared memory and write the gradient.  There is no CPU path.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import DTYPES, ptr

MAX_K = 1024
MAX_VOCAB = 1 << 20
LOSS, LOSS_AND_GRAD, GRAD = 0, 1, 2


def _rows(t: torch.Tensor, what: str) -> int:
    """Row stride of a 2-D tensor with unit column stride and rows that do not overlap."""
    if t.dim() != 2:
        raise ValueError(f"distill: {what} must be 2-D with unit column stride")
    rows, cols = t.shape
    ld, step = t.stride()
    if cols > 1 and step != 1:
        raise ValueError(f"distill: {what} must be 2-D with unit column stride")
    if rows <= 1:
        return max(cols, 1)
    if ld < cols:
        raise ValueError(f"distill: the rows of {what} overlap")
    return ld


def _vector(t: Optional[torch.Tensor], T: int, what: str) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.dtype is not torch.float32 or t.shape != (T,):
        raise ValueError(f"distill: {what} must be fp32 of shape [{T}]")
    return t if t.is_contiguous() else t.contiguous()


def _like(logits: torch.Tensor, ld: int) -> torch.Tensor:
    """An uninitialised [T, V] of the logits' type whose rows start at the same offset from a 16-byte boundary."""
    T, V = logits.shape
    es = logits.element_size()
    vec = 16 // es
    ld_out = V + (ld - V) % vec
    phase = (logits.data_ptr() & 15) // es
    buf = torch.empty(T * ld_out + phase, dtype=logits.dtype, device=logits.device)
    return buf.as_strided((T, V), (ld_out, 1), phase)


def _call(logits, idx, teacher, teacher_lse, weight, temperature, mode, stats=None, grad=None, out=None, want_stats=False):
    dev = _lib.require_cuda(logits, idx, teacher, teacher_lse, weight, stats, grad, out)
    code, tcode, itype = DTYPES.get(logits.dtype), DTYPES.get(teacher.dtype), idx.dtype
    if code is None or tcode is None:
        raise TypeError("distill: logits and teacher must be fp32, bf16 or fp16")
    if itype is not torch.int64 and itype is not torch.int32:
        raise TypeError("distill: idx must be int32 or int64")
    ld = _rows(logits, "logits")
    ld_i, ld_u = _rows(idx, "idx"), _rows(teacher, "teacher")
    (T, V), (Ti, K) = logits.shape, idx.shape
    if Ti != T or teacher.shape != idx.shape:
        raise ValueError(f"distill: idx and teacher must both be [{T}, K]")
    if not 1 <= K <= MAX_K or not 1 <= V <= MAX_VOCAB:
        raise ValueError(f"distill: between 1 and {MAX_K} slots and between 1 and {MAX_VOCAB} tokens are supported")
    if not 0.0 < temperature < float("inf"):
        raise ValueError("distill: the temperature must be positive and finite")
    if teacher_lse is not None:
        teacher_lse = _vector(teacher_lse, T, "teacher_lse")
    if weight is not None:
        weight = _vector(weight, T, "weight")
    loss = dlogits = None
    ld_d = s_grad = 0
    if mode != GRAD:
        loss = torch.empty(T, dtype=torch.float32, device=dev)
        if want_stats:
            stats = torch.empty((T, 3), dtype=torch.float32, device=dev)
    else:
        if stats.dtype != torch.float32 or stats.shape != (T, 3) or not stats.is_contiguous():
            raise ValueError(f"distill: stats must be the [{T}, 3] that topk_loss returned")
        if grad is not None:
            if grad.dtype != torch.float32 or grad.shape != (T,):
                raise ValueError(f"distill: grad must be fp32 of shape [{T}]")
            s_grad = grad.stride(0)
    if mode != LOSS:
        if out is None:
            dlogits = _like(logits, ld)
        elif out.dtype != logits.dtype or out.shape != logits.shape:
            raise ValueError("distill: out must have the logits' shape and type")
        else:
            dlogits = out
            same = out.data_ptr() == logits.data_ptr() and (T <= 1 or out.stride(0) == logits.stride(0))
            if not same and _lib.overlap(out, logits):
                raise ValueError("distill: out may be the logits themselves, but may not overlap them otherwise")
        ld_d = _rows(dlogits, "out")
    with _lib.on_device(dev):
        rc = _lib.lib().ltq_distill_topk(
            logits.data_ptr(), code, ld, idx.data_ptr(), itype is torch.int64, ld_i, teacher.data_ptr(), tcode, ld_u,
            ptr(teacher_lse), ptr(weight), ptr(grad), s_grad, T, V, K, temperature, mode, ptr(loss), ptr(stats),
            ptr(dlogits), ld_d, _lib.stream_ptr(dev))
    if rc != 0:
        raise RuntimeError(f"ltq_distill_topk: error code {rc}")
    if out is not None:
        _lib.written(out)
    return loss, stats, dlogits


def topk_loss(logits: torch.Tensor, idx: torch.Tensor, teacher: torch.Tensor, *,
              teacher_lse: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None,
              temperature: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss [T], stats [T, 3]) of logits [T, V] against teacher [T, K] at the tokens idx [T, K].  stats = (m, s, r), which
    topk_grad takes: the student's sum of exponentials is s 2^m, its mass outside the slots 2^r (m may round to an infinity in
    rows of logits beyond 2^29 temperature)."""
    loss, stats, _ = _call(logits, idx, teacher, teacher_lse, weight, temperature, LOSS, want_stats=True)
    return loss, stats


def topk_loss_grad(logits: torch.Tensor, idx: torch.Tensor, teacher: torch.Tensor, *,
                   teacher_lse: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None,
                   temperature: float = 1.0, out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss [T], d sum(loss) / d logits [T, V] in the logits' type), in one call.  A mean or any other weighting goes
    into `weight`.  out may be `logits` itself, which the gradient then replaces."""
    loss, _, d = _call(logits, idx, teacher, teacher_lse, weight, temperature, LOSS_AND_GRAD, out=out)
    return loss, d


def topk_grad(logits: torch.Tensor, idx: torch.Tensor, teacher: torch.Tensor, stats: torch.Tensor, *,
              grad: Optional[torch.Tensor] = None, teacher_lse: Optional[torch.Tensor] = None,
              weight: Optional[torch.Tensor] = None, temperature: float = 1.0,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient by the logits alone, from topk_loss's stats and the upstream gradient `grad` [T] of its losses."""
    return _call(logits, idx, teacher, teacher_lse, weight, temperature, GRAD, stats=stats, grad=grad, out=out)[2]


class _TopkGrad(torch.autograd.Function):
    """topk_grad within a backward pass.  It depends on the logits as well as on the upstream gradient, so the graph of a gradient
    (create_graph=True) ends in a node that refuses, whatever the upstream gradient is."""

    @staticmethod
    def forward(ctx, logits, idx, teacher, teacher_lse, weight, stats, grad, temperature):
        return topk_grad(logits, idx, teacher, stats, grad=grad, teacher_lse=teacher_lse, weight=weight, temperature=temperature)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("distill: the divergence has no second derivatives")


class _TopkLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, idx, teacher, teacher_lse, weight, temperature):
        loss, stats = topk_loss(logits, idx, teacher, teacher_lse=teacher_lse, weight=weight, temperature=temperature)
        ctx.save_for_backward(logits, idx, teacher, teacher_lse, weight, stats)
        ctx.temperature = temperature
        return loss

    @staticmethod
    def backward(ctx, grad):
        logits, idx, teacher, teacher_lse, weight, stats = ctx.saved_tensors
        d = _TopkGrad.apply(logits, idx, teacher, teacher_lse, weight, stats, grad, ctx.temperature)
        return d, None, None, None, None, None


def distill_loss(logits: torch.Tensor, idx: torch.Tensor, teacher: torch.Tensor, *,
                 teacher_lse: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None,
                 temperature: float = 1.0) -> torch.Tensor:
    """topk_loss as a node of torch's autograd graph: loss [T], differentiable by the logits (the teacher and the weights
    are constants).  The backward pass reads the logits again and runs topk_grad; a second derivative raises RuntimeError."""
    return _TopkLoss.apply(logits, idx, teacher, teacher_lse, weight, temperature)
