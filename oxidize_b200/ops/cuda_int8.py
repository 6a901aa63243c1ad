"""Products on 8-bit integers (``csrc/oxb_int8.cu``): weights with a scale per output channel (``QTensor`` of type "I8"), activations
with one per token.  CUDA tensors only; reached through :func:`oxidize_b200.ops.linear`."""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import cuda as C
from .cuda import _check, _p, _stream

_declared = False
MAX_K = 131072  # 127 * 127 * MAX_K < 2^31: the sums are whole 32-bit numbers


class Int8Rows(NamedTuple):
    codes: torch.Tensor  # [T, K] int8, rows on 16-byte boundaries
    scales: torch.Tensor  # [T] float32


def lib():
    global _declared
    L = C.lib()
    if not _declared:
        vp, i32 = ctypes.c_void_p, ctypes.c_int
        L.oxb_quantize_tokens.argtypes = [vp, i32, i32, vp, i32, vp, vp]
        L.oxb_gemm_int8.argtypes = [vp, i32, vp, vp, i32, vp, vp, vp, i32, i32, i32, i32, vp]
        _declared = True
    return L


def quantize_tokens(x: torch.Tensor) -> Int8Rows:
    """Rows of x [T, K] (bf16, contiguous) as 8-bit integers (see :func:`oxidize_b200.ops.ref.quantize_tokens`)."""
    T, K = x.shape
    codes = torch.empty(T, -(-K // 16) * 16, dtype=torch.int8, device=x.device)
    scales = torch.empty(T, dtype=torch.float32, device=x.device)
    _check(lib().oxb_quantize_tokens(x.data_ptr(), T, K, codes.data_ptr(), codes.stride(0), scales.data_ptr(), _stream()), "oxb_quantize_tokens")
    return Int8Rows(codes[:, :K], scales)


def linear(x: Int8Rows, p, out_view: torch.Tensor, bias: Optional[torch.Tensor], ld_out: int) -> torch.Tensor:
    n, k = p.shape
    w = p.data
    if x.codes.shape[1] != k or k > MAX_K:
        raise ValueError(f"8-bit product of {x.codes.shape[1]} values a token with a [{n}, {k}] matrix (at most {MAX_K} columns)")
    if w.dtype != torch.int8 or w.stride(1) != 1 or w.stride(0) % 16 or w.data_ptr() % 16 or p.scales.dtype != torch.float32:
        raise ValueError("8-bit weights are int8 rows on 16-byte boundaries with float32 scales (quant.torch_quant.int8_rows)")
    _check(lib().oxb_gemm_int8(x.codes.data_ptr(), x.codes.stride(0), x.scales.data_ptr(), w.data_ptr(), w.stride(0), p.scales.data_ptr(),
                               _p(bias), out_view.data_ptr(), ld_out, x.codes.shape[0], n, k, _stream()), "oxb_gemm_int8")
    return out_view
