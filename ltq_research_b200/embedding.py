"""Token table lookup with scaling, and the table's gradient by sorted tokens.

* lookup       out[i] = scale * table[tokens[i]], rounded once to the table's type (one kernel, ltq_embed_lookup);
* lookup_grad  grad[v] = scale * sum of dout[i] over the positions i with tokens[i] = v: the positions are sorted by token
               and the runs summed in fp32, a run in groups that follow from its places in the sorted list (three launches,
               ltq_embed_grad).  The same bits at every call with the same tokens: no atomics on values.

A token outside [0, number of rows) reads as zeros and takes no gradient, as does the padding token in the gradient.
There is no CPU path.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._lib import DTYPES, ptr


def _tokens(tokens: torch.Tensor) -> torch.Tensor:
    if tokens.dtype not in (torch.int32, torch.int64):
        raise TypeError("embedding: tokens must be int32 or int64")
    return tokens if tokens.is_contiguous() else tokens.contiguous()


def _row_stride(t: torch.Tensor, what: str) -> int:
    if t.dim() != 2:
        raise ValueError(f"embedding: {what} must be 2-D with unit column stride")
    rows, cols = t.shape
    ld, step = t.stride()
    if cols < 1 or (cols > 1 and step != 1):
        raise ValueError(f"embedding: {what} must be 2-D with unit column stride")
    if rows <= 1:
        return cols
    if ld < cols:
        raise ValueError(f"embedding: the rows of {what} overlap")
    return ld


def lookup(table: torch.Tensor, tokens: torch.Tensor, scale: float = 1.0,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """scale * table[tokens]: table [V, D] fp32, bf16 or fp16, tokens of any shape -> [*tokens.shape, D]."""
    dev = _lib.require_cuda(table, tokens, out)
    code = DTYPES.get(table.dtype)
    if code is None:
        raise TypeError("embedding: the table must be fp32, bf16 or fp16")
    ld = _row_stride(table, "the table")
    V, D = table.shape
    if V < 1:
        raise ValueError("embedding: the table has no rows")
    tok = _tokens(tokens)
    given = out is not None
    if not given:
        out = torch.empty((*tokens.shape, D), dtype=table.dtype, device=dev)
    elif out.dtype != table.dtype or out.shape != (*tokens.shape, D) or not out.is_contiguous():
        raise ValueError("embedding: out must be contiguous, of the table's type and shape [*tokens.shape, D]")
    elif _lib.overlap(out.view(-1, D), table):
        raise ValueError("embedding: out may not overlap the table")
    with _lib.on_device(dev):
        rc = _lib.lib().ltq_embed_lookup(table.data_ptr(), code, ld, tok.data_ptr(), tok.dtype is torch.int64, tok.numel(), V, D,
                                         scale, out.data_ptr(), D, _lib.stream_ptr(dev))
    if rc != 0:
        raise RuntimeError(f"ltq_embed_lookup: error code {rc}")
    if given:
        _lib.written(out)
    return out


def lookup_grad(tokens: torch.Tensor, dout: torch.Tensor, num_rows: int, scale: float = 1.0,
                padding_idx: Optional[int] = None, out: Optional[torch.Tensor] = None, accumulate: bool = False,
                dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The gradient [num_rows, D] of a table by dout [*tokens.shape, D], the gradient of lookup(table, tokens, scale).
    out: written (accumulate=False) or added to (accumulate=True; rows that no token names are not touched), with its own
    type; without it a new tensor of `dtype`."""
    dev = _lib.require_cuda(tokens, dout, out)
    if dout.dtype not in DTYPES or (out.dtype if out is not None else dtype) not in DTYPES:
        raise TypeError("embedding: gradients must be fp32, bf16 or fp16")
    if dout.dim() < 1 or dout.shape[:-1] != tokens.shape:
        raise ValueError("embedding: dout must be [*tokens.shape, D]")
    num_rows = int(num_rows)
    if num_rows < 1 or num_rows > 1 << 30:
        raise ValueError("embedding: between 1 and 2^30 table rows are supported")
    if padding_idx is not None and not 0 <= padding_idx < num_rows:
        raise ValueError("embedding: padding_idx is not a row of the table")
    tok = _tokens(tokens)
    D = dout.shape[-1]
    d = dout if dout.dim() == 2 else dout.reshape(-1, D)
    if d.shape[0] > 1 and (d.stride(0) < D or (D > 1 and d.stride(1) != 1)) or (D > 1 and d.stride(1) != 1):
        d = d.contiguous()  # a gradient that autograd expanded
    ld_d = _row_stride(d, "dout")
    given = out is not None
    if not given:
        if accumulate:
            raise ValueError("embedding: accumulate needs the tensor to add to")
        out = torch.empty((num_rows, D), dtype=dtype, device=dev)
    elif out.shape != (num_rows, D):
        raise ValueError(f"embedding: out must be [{num_rows}, {D}]")
    ld_o = _row_stride(out, "out")
    if given and _lib.overlap(out, d):
        raise ValueError("embedding: out may not overlap dout")
    n = tok.numel()
    L = _lib.lib()
    ws = torch.empty(L.ltq_embed_grad_workspace_bytes(n, D), dtype=torch.uint8, device=dev)
    with _lib.on_device(dev):
        rc = L.ltq_embed_grad(ptr(tok), int(tok.dtype == torch.int64), n, num_rows,
                              -1 if padding_idx is None else padding_idx, ptr(d), DTYPES[d.dtype], ld_d, D, float(scale),
                              ptr(out), DTYPES[out.dtype], ld_o, int(accumulate), ptr(ws), ws.numel(),
                              _lib.stream_ptr(dev))
    if rc != 0:
        raise RuntimeError(f"ltq_embed_grad: error code {rc}")
    if given:
        _lib.written(out)
    return out


class _LookupGrad(torch.autograd.Function):
    """lookup_grad within a backward pass: in the graph of a gradient (create_graph=True) a node that refuses."""

    @staticmethod
    def forward(ctx, tokens, dout, rows, scale, padding_idx, dtype):
        return lookup_grad(tokens, dout, rows, scale, padding_idx, dtype=dtype)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("embedding: the lookup's gradient is not differentiable by dout")


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, tokens, scale, padding_idx):
        ctx.save_for_backward(tokens)
        ctx.args = (table.shape[0], scale, padding_idx, table.dtype)
        return lookup(table, tokens, scale)

    @staticmethod
    def backward(ctx, dout):
        return _LookupGrad.apply(ctx.saved_tensors[0], dout, *ctx.args), None, None, None


def embed(table: torch.Tensor, tokens: torch.Tensor, scale: float = 1.0,
          padding_idx: Optional[int] = None) -> torch.Tensor:
    """lookup as a node of torch's autograd graph: the table's gradient is lookup_grad's, in the table's type; a second
    derivative (a dout that depends on what is differentiated by) raises RuntimeError."""
    return _Lookup.apply(table, tokens, scale, padding_idx)
