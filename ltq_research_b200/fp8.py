"""Products with weights held in 8-bit floating point (e4m3) under one scale per 128 x 128 block, the form of 8-bit
checkpoints.

* quantize_blocks(w) / quantize_rows(x): e4m3 values and fp32 scales max|.| / 448 (at least 2^-126), per 128 x 128 block of a
  weight, per row and 128 columns of an activation; a block that holds a NaN or an infinity becomes NaN.
* BlockWeight: a weight's values and scales as the kernels read them (rows padded to 16 bytes; with backward=True also
  transposed, with the same 8-bit values and scales: the blocks are square).  Made once, kept by the program.
* linear(x, W) = x W^T and linear_grad(dy, W) = dy W: the activations are quantized in the call, the products of each block
  of 128 are summed on the tensor cores and joined under their scales in fp32, one rounding to the output's type.
  The weight is frozen: the gradient by the input alone.

There is no CPU path.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import DTYPES, ptr

BLOCK = 128
FEW = 32  # rows up to which one launch quantizes them and streams the weight (ltq_fp8_few)
E4M3 = torch.float8_e4m3fn


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _pad16(n: int) -> int:
    return (n + 15) // 16 * 16


_FLAGS = {}


def _error_flag(dev: torch.device) -> torch.Tensor:
    """The tensor-core products' common flag of a device."""
    flag = _FLAGS.get(dev)
    if flag is None:
        from .liqk_v2 import gemm_error_flag
        flag = _FLAGS[dev] = gemm_error_flag(dev)
    return flag


def _check(rc: int, what: str):
    if rc != 0:
        raise RuntimeError(f"{what}: error code {rc}")


def _rows(x: torch.Tensor, what: str) -> int:
    if x.dtype not in DTYPES:
        raise TypeError(f"fp8: {what} must be fp32, bf16 or fp16")
    if x.dim() != 2 or x.shape[1] < 1 or (x.shape[1] > 1 and x.stride(1) != 1):
        raise ValueError(f"fp8: {what} must be 2-D with unit column stride and at least one column")
    if x.shape[0] <= 1:
        return x.shape[1]
    if x.stride(0) < x.shape[1]:
        raise ValueError(f"fp8: the rows of {what} overlap")
    return x.stride(0)


def _quantize_rows(x: torch.Tensor, ld: int):
    """(values [M, pad16(K)] uint8, scales [blocks, pad4(M)] fp32) of x, the layout the product reads."""
    M, K = x.shape
    q = torch.empty((M, _pad16(K)), dtype=torch.uint8, device=x.device)
    s = torch.empty((_blocks(K), (M + 3) // 4 * 4), dtype=torch.float32, device=x.device)
    _check(_lib.lib().ltq_fp8_quant_rows(ptr(x), DTYPES[x.dtype], ld, M, K, ptr(q), q.shape[1], ptr(s), s.shape[1],
                                         _lib.stream_ptr(x.device)), "ltq_fp8_quant_rows")
    return q, s


@torch.no_grad()
def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(e4m3 values [M, K], scales [M, ceil(K / 128)]) of x [M, K], both views of buffers laid out for the product."""
    dev = _lib.require_cuda(x)
    ld = _rows(x, "x")
    with _lib.on_device(dev):
        q, s = _quantize_rows(x, ld)
    return q[:, :x.shape[1]].view(E4M3), s[:, :x.shape[0]].t()


@torch.no_grad()
def quantize_blocks(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(e4m3 values [N, K], scales [ceil(N / 128), ceil(K / 128)]) of w [N, K]."""
    dev = _lib.require_cuda(w)
    ld = _rows(w, "w")
    N, K = w.shape
    q = torch.empty((N, _pad16(K)), dtype=torch.uint8, device=dev)
    s = torch.empty((_blocks(N), _blocks(K)), dtype=torch.float32, device=dev)
    with _lib.on_device(dev):
        _check(_lib.lib().ltq_fp8_quant_blocks(ptr(w), DTYPES[w.dtype], ld, N, K, ptr(q), q.shape[1], ptr(s), s.shape[1],
                                               _lib.stream_ptr(dev)), "ltq_fp8_quant_blocks")
    return q[:, :K].view(E4M3), s


class BlockWeight:
    """A weight [N, K] in e4m3 with scales [ceil(N / 128), ceil(K / 128)], laid out once for the products.  backward=True
    also holds its transpose (as many bytes again), which linear_grad reads."""

    def __init__(self, q: torch.Tensor, s: torch.Tensor, backward: bool = False):
        self.device = _lib.require_cuda(q, s)
        if q.dtype != E4M3 or q.dim() != 2 or q.shape[0] < 1 or q.shape[1] < 1:
            raise ValueError("BlockWeight: the values must be a 2-D float8_e4m3fn tensor")
        N, K = self.shape = tuple(q.shape)
        if s.dtype != torch.float32 or tuple(s.shape) != (_blocks(N), _blocks(K)):
            raise ValueError(f"BlockWeight: the scales must be fp32 [{_blocks(N)}, {_blocks(K)}]")
        self.q, self.s = self._lay(q), s.contiguous()  # before the transpose, which reads them
        self.qt = self._transposed(N, K) if backward else None
        self.st = s.t().contiguous() if backward else None
        _error_flag(self.device)  # made (which synchronises) here, so that the first product may be captured into a graph

    @classmethod
    def quantize(cls, w: torch.Tensor, backward: bool = False) -> "BlockWeight":
        return cls(*quantize_blocks(w), backward=backward)

    @staticmethod
    def _lay(q: torch.Tensor) -> torch.Tensor:
        rows, cols = q.shape
        u = q.view(torch.uint8)
        if u.stride(1) == 1 and u.stride(0) % 16 == 0 and u.stride(0) >= cols and u.data_ptr() % 16 == 0:
            return u
        out = torch.zeros((rows, _pad16(cols)), dtype=torch.uint8, device=q.device)
        out[:, :cols] = u
        return out

    def _transposed(self, N: int, K: int) -> torch.Tensor:
        qt = torch.empty((K, _pad16(N)), dtype=torch.uint8, device=self.device)
        with _lib.on_device(self.device):
            _check(_lib.lib().ltq_fp8_transpose(ptr(self.q), self.q.stride(0), N, K, ptr(qt), qt.shape[1],
                                                _lib.stream_ptr(self.device)), "ltq_fp8_transpose")
        return qt

    def dequantize(self) -> torch.Tensor:
        """The weight's values in fp32."""
        N, K = self.shape
        s = self.s.repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]
        return self.q[:, :K].view(E4M3).float() * s


def _product(x: torch.Tensor, q: torch.Tensor, s: torch.Tensor, N: int, K: int, dtype: Optional[torch.dtype]) -> torch.Tensor:
    dtype = x.dtype if dtype is None else dtype
    code = DTYPES.get(dtype)
    if code is None:
        raise TypeError("fp8: the output must be fp32, bf16 or fp16")
    shape = x.shape
    if len(shape) < 1 or shape[-1] != K:
        raise ValueError(f"fp8: the last dimension must be {K}")
    dev = _lib.require_cuda(x, q)
    x2 = x if len(shape) == 2 else x.reshape(-1, K)
    M = x2.shape[0]
    ld, step = x2.stride()
    if (K > 1 and step != 1) or (M > 1 and ld < K):
        x2 = x2.contiguous()
        ld = K
    if M <= 1:
        ld = K
    xcode = DTYPES.get(x2.dtype)
    if xcode is None:
        raise TypeError("fp8: x must be fp32, bf16 or fp16")
    y = torch.empty((*shape[:-1], N), dtype=dtype, device=dev)
    if M == 0:
        return y
    L = _lib.lib()
    with _lib.on_device(dev):
        st, err = _lib.stream_ptr(dev), ptr(_error_flag(dev))
        if M <= FEW and L.ltq_fp8_few_supported(M, N, K):
            _check(L.ltq_fp8_few(x2.data_ptr(), xcode, ld, q.data_ptr(), q.stride(0), s.data_ptr(), s.shape[1], y.data_ptr(),
                                 code, N, M, N, K, err, st), "ltq_fp8_few")
            return y
        xq, xs = _quantize_rows(x2, ld)
        nws = L.ltq_fp8_gemm_workspace_bytes(M, N, K)
        ws = torch.empty(nws, dtype=torch.uint8, device=dev) if nws else None
        _check(L.ltq_fp8_gemm(ptr(xq), xq.shape[1], ptr(xs), xs.shape[1], ptr(q), q.stride(0), ptr(s), s.shape[1], ptr(y),
                              code, N, M, N, K, ptr(ws), nws, err, st), "ltq_fp8_gemm")
    return y


def linear(x: torch.Tensor, W: BlockWeight, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x W^T: x [..., K] fp32, bf16 or fp16 -> [..., N] in `dtype` (x's by default)."""
    N, K = W.shape
    return _product(x, W.q, W.s, N, K, dtype)


def linear_grad(dy: torch.Tensor, W: BlockWeight, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """dy W: the gradient [..., K] of linear's input by dy [..., N], dy quantized per row and 128 columns."""
    if W.qt is None:
        raise ValueError("fp8: linear_grad needs a BlockWeight made with backward=True")
    N, K = W.shape
    return _product(dy, W.qt, W.st, K, N, dtype)


def check_errors(device):
    """Raises if a product on `device` reported a timed-out pipeline wait since the last check (synchronises)."""
    from .liqk_v2 import check_gemm_errors
    check_gemm_errors(device)


class _LinearGrad(torch.autograd.Function):
    """linear_grad within a backward pass: in the graph of a gradient (create_graph=True) a node that refuses."""

    @staticmethod
    def forward(ctx, dy, W, dtype):
        return linear_grad(dy, W, dtype)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("fp8: the product's gradient is not differentiable by dy")


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, W):
        ctx.W = W
        ctx.dtype = x.dtype
        return linear(x, W)

    @staticmethod
    def backward(ctx, dy):
        return _LinearGrad.apply(dy, ctx.W, ctx.dtype), None


def block_linear(x: torch.Tensor, W: BlockWeight) -> torch.Tensor:
    """linear as a node of torch's autograd graph; the gradient by x is linear_grad's (W made with backward=True); a second
    derivative (a dy that depends on what is differentiated by) raises RuntimeError."""
    return _Linear.apply(x, W)
