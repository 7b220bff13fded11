"""Loader of the in-tree CUDA library ``libltq_b200.so`` (C ABI: include/ltq_b200.h).

There is no fallback: if the library is missing, or a call is made without a CUDA device, the call raises.
"""
from __future__ import annotations

import ctypes
import threading
from contextlib import nullcontext
from pathlib import Path

import torch

LIB_PATH = Path(__file__).resolve().parent / "libltq_b200.so"
_LIB = None
_LOCK = threading.Lock()

P = ctypes.c_void_p
I = ctypes.c_int
SZ = ctypes.c_size_t
LL = ctypes.c_longlong

# name -> (restype, argtypes); mirrors include/ltq_b200.h
SIGNATURES = {
    "ltq_b200_version": (ctypes.c_char_p, []),
    # reference ctypes binding, src/tcq_proto.py:529: 15 pointers, 18 ints, pointer, int, pointer
    "tcq_viterbi": (I, [P] * 15 + [I] * 18 + [P, I, P]),
    "ltq_viterbi_tb_workspace_bytes": (SZ, [I] * 8),
    "ltq_viterbi_tb": (I, [P, P, I, P, P, P, P, P, P] + [I] * 5 + [P] + [I] * 10 + [P, SZ, P]),
    # matrix-level kernels
    "ltq_fwht256": (I, [P, I, ctypes.c_longlong, P, ctypes.c_longlong, P, I, I, I, P]),
    "ltq_scale_fit": (I, [P, ctypes.c_longlong, I, I, ctypes.c_float, ctypes.c_float, I, P, P, P, P, P]),
    "ltq_ldlq_gather": (I, [P, ctypes.c_longlong, P, I, P, P]),
    "ltq_ldlq_feedback": (I, [P, ctypes.c_longlong, I, I, P, P, P, P, ctypes.c_longlong, P, ctypes.c_longlong, P,
                              ctypes.c_longlong, P, P, ctypes.c_longlong, P]),
    "ltq_ldlq_block_workspace_bytes": (SZ, [I] * 6),
    "ltq_ldlq_bcat_elems": (SZ, [I]),
    "ltq_bf16x6_split": (I, [P, LL, I, I, I, I, P, LL, P]),
    "ltq_bf16x6_split_batched": (I, [P, LL, LL, I, I, I, I, I, I, P, LL, LL, P]),
    "ltq_trtri256_lower": (I, [P, LL, I, P, LL, P]),
    "ltq_chol256_diag": (I, [P, LL, I, P, P, LL, P, P]),
    "lut_subs_quant": (I, [P, P, P, P, I, ctypes.c_float, ctypes.c_float, I, P]),
    "ltq_int8_rings": (I, [P, P, LL, I, P]),
    "ltq_matvec_slice": (I, [P, I, I, I, I, I, I, P, I, P, P, P, P, LL, P, P, P]),
    "ltq_ldlq_bcat": (I, [P, LL, I, P, P]),
    "ltq_ldlq_bcat_t": (I, [P, LL, I, P, P]),
    "ltq_gemm_bf16_tn": (I, [P, LL, P, LL, P, LL, I, I, I, ctypes.c_float, ctypes.c_float, P, P]),
    "ltq_gemm_bf16x6_tn": (I, [P, LL, P, LL, P, LL, I, I, I, ctypes.c_float, ctypes.c_float, P, P]),
    "ltq_gemm_wait_selftest": (I, [I, ctypes.c_uint, P, P, P]),
    "ltq_chol_solve": (I, [P, LL, I, P, P, P, P, P]),
    "ltq_gemm_bf16x3p_tn": (I, [P, LL, LL, P, LL, LL, P, LL, LL, I, I, I, I, I, ctypes.c_float, ctypes.c_float, P, P]),
    "ltq_bf16x3_split": (I, [P, LL, LL, I, I, I, I, I, I, P, LL, LL, P]),
    "ltq_ldlq_inter3": (I, [P, LL, P, LL, P, LL, P, LL, I, P, LL, P, LL, P, P]),
    "ltq_ldlq_inter": (I, [P, LL, P, LL, P, LL, P, LL, I, P, LL, P, LL, P, P]),
    "ltq_ldlq_block": (I, [P, LL, P, LL, P, P, LL, P, LL, P, LL, P, P, LL, I, P, P, I, I, P] + [I] * 6 + [P, SZ, P]),
    # .ltq packing and spec decode
    "ltq_slice_bytes": (SZ, [I] * 6),
    "ltq_pack_slice": (I, [P, P, LL] + [I] * 6 + [P, SZ, P]),
    "ltq_decode_slice": (I, [P] + [I] * 6 + [P, I, P, P, P, LL, P, LL, P, P]),
    # allocation-free variant (scratch inside the library): same arguments without the workspace
    "ltq_viterbi_tb_noalloc_capacity": (SZ, []),
    "ltq_viterbi_tb_noalloc": (I, [P, P, I, P, P, P, P, P, P] + [I] * 5 + [P] + [I] * 10 + [P]),
    # operators at the vocabulary's ends
    "ltq_distill_topk": (I, [P, I, LL, P, I, LL, P, I, LL, P, P, P, LL, I, I, I, ctypes.c_float, I, P, P, P, LL, P]),
    "ltq_embed_lookup": (I, [P, I, LL, P, I, LL, I, I, ctypes.c_float, P, LL, P]),
    "ltq_embed_grad_workspace_bytes": (SZ, [LL, I]),
    "ltq_embed_grad": (I, [P, I, LL, I, LL, P, I, LL, I, ctypes.c_float, P, I, LL, I, P, SZ, P]),
    "ltq_fp8_quant_rows": (I, [P, I, LL, I, I, P, LL, P, LL, P]),
    "ltq_fp8_quant_blocks": (I, [P, I, LL, I, I, P, LL, P, LL, P]),
    "ltq_fp8_transpose": (I, [P, LL, I, I, P, LL, P]),
    "ltq_fp8_gemm_workspace_bytes": (SZ, [I, I, I]),
    "ltq_fp8_few_supported": (I, [I, I, I]),
    "ltq_fp8_few": (I, [P, I, LL, P, LL, P, LL, P, I, LL, I, I, I, P, P]),
    "ltq_fp8_gemm": (I, [P, LL, P, LL, P, LL, P, LL, P, I, LL, I, I, I, P, SZ, P, P]),
}

# element type codes of the C ABI
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class LtqLibraryError(RuntimeError):
    pass


# kernels launched by one successful call (a constant, or a function of the call's arguments)
KERNELS_PER_CALL = {
    "tcq_viterbi": 2,
    "ltq_viterbi_tb": lambda a: 2 * int(a[22]),
    "ltq_viterbi_tb_noalloc": lambda a: 2 * int(a[22]),
    "ltq_fwht256": 1, "ltq_scale_fit": 1, "ltq_ldlq_gather": 1, "ltq_ldlq_feedback": 1, "ltq_ldlq_block": 2,
    "ltq_ldlq_bcat": 1, "ltq_ldlq_bcat_t": 1, "ltq_gemm_bf16_tn": 1, "ltq_gemm_bf16x6_tn": 1, "ltq_gemm_bf16x3p_tn": 1, "ltq_gemm_wait_selftest": 1, "ltq_chol_solve": lambda a: 2 * (int(a[2]) // 256), "ltq_bf16x3_split": 1,
    "ltq_ldlq_inter": 1, "ltq_ldlq_inter3": 1, "ltq_bf16x6_split": 1, "ltq_bf16x6_split_batched": 1,
    "ltq_trtri256_lower": 1, "ltq_chol256_diag": 1, "lut_subs_quant": 1, "ltq_int8_rings": 1, "ltq_matvec_slice": 1,
    "ltq_pack_slice": 1, "ltq_decode_slice": 1,
    "ltq_distill_topk": lambda a: int(a[13] > 0) * (2 if a[17] == 1 else 1),  # loss and gradient: also the rows out of range
    "ltq_embed_lookup": lambda a: int(a[5] > 0),
    "ltq_embed_grad": lambda a: 3 if a[2] > 8 else (2 if a[2] > 0 else int(not a[13])),
    "ltq_fp8_quant_rows": lambda a: int(a[3] > 0), "ltq_fp8_quant_blocks": lambda a: int(a[3] > 0),
    "ltq_fp8_transpose": 1,
    "ltq_fp8_few": lambda a: int(a[10] > 0 and a[11] > 0),
    "ltq_fp8_gemm": lambda a: int(a[11] > 0 and a[12] > 0) + int(a[15] > 0),  # with a workspace also the parts' join
}


class _CountingLib:
    """The ctypes library with a count of the kernels its calls launched (``kernels``), per process."""

    def __init__(self, cdll: ctypes.CDLL):
        self._cdll = cdll
        self.kernels = 0
        self._lock = threading.Lock()

    def __getattr__(self, name):
        fn = getattr(self._cdll, name)
        k = KERNELS_PER_CALL.get(name)
        if k is None:
            return fn

        lock, varies = self._lock, callable(k)

        def call(*a):
            rc = fn(*a)
            if rc == 0:
                n = k(a) if varies else k
                with lock:
                    self.kernels += n
            return rc
        call.__name__ = name
        self.__dict__[name] = call
        return call


def kernels_launched() -> int:
    """Kernels launched so far by this process through the library (successful calls only)."""
    return lib().kernels


def lib() -> "_CountingLib":
    """The loaded library (ctypes functions, plus a launch count); raises LtqLibraryError when it has not been
    built."""
    global _LIB
    if _LIB is None:
        with _LOCK:
            if _LIB is None:
                if not LIB_PATH.exists():
                    raise LtqLibraryError(f"{LIB_PATH} is missing: build it with `python -m ltq_research_b200.build`")
                L = ctypes.CDLL(str(LIB_PATH))
                for name, (res, args) in SIGNATURES.items():
                    fn = getattr(L, name)
                    fn.restype = res
                    fn.argtypes = args
                _LIB = _CountingLib(L)
    return _LIB


def exported_symbols() -> list[str]:
    return list(SIGNATURES)


def stream_ptr(device: torch.device) -> int:
    """The current stream's handle on `device`."""
    if device.index is None:
        return torch.cuda.current_stream(device).cuda_stream
    return torch._C._cuda_getCurrentRawStream(device.index)  # the same handle without a Stream object around it


def require_cuda(*tensors: torch.Tensor) -> torch.device:
    """Every tensor must live on one CUDA device; there is no CPU path."""
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("ltq_research_b200: inputs must be CUDA tensors (there is no CPU implementation)")
        d = t.device
        if dev is None:
            dev = d
        elif d != dev:
            raise RuntimeError("ltq_research_b200: all inputs must be on the same CUDA device")
    if dev is None:
        raise RuntimeError("ltq_research_b200: no CUDA tensor given")
    return dev


def written(t: torch.Tensor):
    """Tells autograd that a kernel has written a tensor of the caller's: whoever saved what it held before gets torch's error."""
    torch.autograd.graph.increment_version(t)


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two 2-D tensors, each with rows that do not overlap, share memory."""
    def span(t):
        n = sum((s - 1) * st for s, st in zip(t.shape, t.stride())) + 1 if t.numel() else 0
        return t.data_ptr(), t.data_ptr() + n * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    if a0 >= b1 or b0 >= a1:
        return False
    ld, cols_a, cols_b = a.stride(0) * a.element_size(), a.shape[1] * a.element_size(), b.shape[1] * b.element_size()
    if a.shape[0] <= 1 or b.shape[0] <= 1 or ld != b.stride(0) * b.element_size() or ld < cols_a or ld < cols_b:
        return True
    apart = (b0 - a0) % ld  # rows of one stride may lie beside each other: columns of a wider tensor
    return not cols_a <= apart <= ld - cols_b


def on_device(device: torch.device):
    """Context with `device` current, as a launch on its streams needs."""
    return _SAME if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


_SAME = nullcontext()


def ptr(t) -> int | None:
    return None if t is None else t.data_ptr()
