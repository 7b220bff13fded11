"""One step of recovering a quantized model from its teacher's top logits, with the vocabulary's two ends in this
package's kernels:

    tokens -> embedding.embed (scaled rows of the trainable table)
           -> body            (the quantized layers: any differentiable callable, its weights frozen)
           -> fp8.block_linear (the frozen output head, e4m3 blocks)
           -> distill.distill_loss against the teacher's top logits
    and back: logits' gradient -> head's input gradient (8-bit) -> body -> the table's gradient by sorted tokens.

QuantizedLinear is a frozen body layer made of a matrix that quantize_matrix_liqk_v2 or an .ltq file decoded.
"""
from __future__ import annotations

from typing import Callable, NamedTuple, Optional

import torch

from . import distill, embedding, fp8


class TeacherTop(NamedTuple):
    """A teacher's top logits at every position: ids and logits [*tokens.shape, K]; lse [*tokens.shape] the log-sum-exp of
    all of its logits at the temperature, or None to compare over the kept tokens alone."""
    idx: torch.Tensor
    logits: torch.Tensor
    lse: Optional[torch.Tensor] = None


class QuantizedLinear:
    """x -> x W_hat^T for a frozen decoded matrix W_hat [out, in]."""

    def __init__(self, W_hat: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
        self.W = W_hat.to(dtype)

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        return torch.nn.functional.linear(x, self.W)


def logits(table: torch.Tensor, tokens: torch.Tensor, body: Callable, head: fp8.BlockWeight, scale: float = 1.0,
           padding_idx: Optional[int] = None) -> torch.Tensor:
    """The student's logits [positions, V] for tokens of any shape."""
    h = body(embedding.embed(table, tokens, scale, padding_idx))
    return fp8.block_linear(h.reshape(-1, h.shape[-1]), head)


def score(table: torch.Tensor, tokens: torch.Tensor, body: Callable, head: fp8.BlockWeight, teacher: TeacherTop, *,
          scale: float = 1.0, temperature: float = 1.0, weight: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The divergence from the teacher at every position, of tokens' shape (evaluation: no gradient)."""
    with torch.no_grad():
        z = logits(table, tokens, body, head, scale)
        K = teacher.idx.shape[-1]
        loss, _ = distill.topk_loss(z, teacher.idx.reshape(-1, K), teacher.logits.reshape(-1, K),
                                    teacher_lse=None if teacher.lse is None else teacher.lse.reshape(-1),
                                    weight=None if weight is None else weight.reshape(-1).float(), temperature=temperature)
    return loss.view(tokens.shape)


def step(table: torch.Tensor, tokens: torch.Tensor, body: Callable, head: fp8.BlockWeight, teacher: TeacherTop, *,
         scale: float = 1.0, temperature: float = 1.0, weight: Optional[torch.Tensor] = None,
         padding_idx: Optional[int] = None) -> torch.Tensor:
    """Mean divergence over the weighted positions; leaves its gradient in table.grad (added to what is there) and in
    whatever of `body` asks for one.  The loss and the logits' gradient come from one call that writes the gradient over
    the logits."""
    if not table.requires_grad:
        raise ValueError("recovery.step: the table must require a gradient")
    w = torch.ones(tokens.numel(), device=tokens.device) if weight is None else weight.reshape(-1).float()
    w = w / w.sum().clamp(min=1e-20)
    z = logits(table, tokens, body, head, scale, padding_idx)
    K = teacher.idx.shape[-1]
    zd = z.detach()
    loss, dz = distill.topk_loss_grad(zd, teacher.idx.reshape(-1, K), teacher.logits.reshape(-1, K),
                                      teacher_lse=None if teacher.lse is None else teacher.lse.reshape(-1), weight=w,
                                      temperature=temperature, out=zd)
    z.backward(dz)
    return loss.sum()
