"""Products on 8-bit integers (``csrc/oxb_int8.cu``): weights with a scale per output channel (``QTensor`` of type "I8"), activations
with one per token.  CUDA tensors only; reached through :func:`oxidize_b200.ops.linear`."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import cuda as C
from .cuda import _check, _p, _stream

_declared = False
MAX_STRIDE = 2 ** 31 - 1  # values from row to row, a 32-bit number for the kernels
MAX_K = 131072  # 127 * 127 * MAX_K < 2^31: the sums are whole 32-bit numbers


def lib():
    global _declared
    L = C.lib()
    if not _declared:
        vp, i32 = ctypes.c_void_p, ctypes.c_int
        L.oxb_int8_needs_rows.argtypes = [i32, i32]
        L.oxb_linear_int8.argtypes = [vp, i32, i32, vp, i32, vp, i32, vp, vp, vp, i32, i32, vp]
        _declared = True
    return L


def linear(x: torch.Tensor, p, out_view: torch.Tensor, bias: Optional[torch.Tensor], ld_out: int,
           rows: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """out_view = x @ W^T (+ bias) for x [T, K] (bf16, contiguous).  Returns x's rows as 8-bit integers (see
    :func:`oxidize_b200.ops.ref.quantize_tokens`) for a further product of the same x (``rows``), or None where each makes its own."""
    n, k = p.shape
    w = p.data
    T = x.shape[0]
    if x.shape[1] != k or k > MAX_K:
        raise ValueError(f"8-bit product of {x.shape[1]} values a token with a [{n}, {k}] matrix (at most {MAX_K} columns)")
    ld, one = w.stride()
    if (w.dtype != torch.int8 or w.shape != (n, k) or one != 1 or ld % 16 or not k <= ld <= MAX_STRIDE or w.data_ptr() % 16 or p.scales.dtype != torch.float32
            or p.scales.shape != (n,) or not p.scales.is_contiguous()):
        raise ValueError("8-bit weights are int8 rows on 16-byte boundaries with float32 scales (quant.torch_quant.int8_rows)")
    device = torch._C._cuda_getDevice()
    if x.get_device() != device or w.get_device() != device or p.scales.get_device() != device or (bias is not None and bias.get_device() != device):
        raise ValueError(f"an 8-bit product's tensors lie on the current device, cuda:{device}")
    # (as for the other encodings, a bias may be longer and an output larger than what is used of them)
    if bias is not None and (bias.dim() == 0 or bias.shape[-1] < n or bias.numel() != bias.shape[-1]):
        raise ValueError(f"the bias of {n} outputs has as many values, not {tuple(bias.shape)}")
    if (out_view.dtype != torch.bfloat16 or out_view.get_device() != device or out_view.dim() != 2 or out_view.shape[0] < T or out_view.shape[1] < n
            or (out_view.stride(1) != 1 and n > 1) or (T > 1 and not n <= ld_out <= MAX_STRIDE)):
        raise ValueError(f"an 8-bit product's output is [{T}, {n}] in bfloat16 on the current device, columns side by side and rows at most {MAX_STRIDE} values "
                         f"apart, not {tuple(out_view.shape)} in {out_view.dtype} on {out_view.device} with strides {out_view.stride()}")
    if bias is not None and (bias.dtype != torch.float32 or not bias.is_contiguous()):
        bias = bias.float().contiguous()
    L = lib()
    made = rows is not None
    if not made and L.oxb_int8_needs_rows(T, k):
        rows = torch.empty(T * (-(-k // 16) * 16 + 4), dtype=torch.uint8, device=x.device)
    _check(L.oxb_linear_int8(x.data_ptr(), T, k, _p(rows), int(made), w.data_ptr(), ld, p.scales.data_ptr(), _p(bias),
                             out_view.data_ptr(), ld_out if T > 1 else n, n, _stream()), "oxb_linear_int8")
    return rows
