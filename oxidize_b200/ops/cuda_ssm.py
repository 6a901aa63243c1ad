"""Bindings of the kernels of state-space layers (``csrc/oxb_ssm.cu``).  CUDA tensors only; see
:func:`oxidize_b200.ops.causal_conv` and :func:`oxidize_b200.ops.selective_scan` for the operators' meaning."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import cuda as opcuda
from .cuda import _check, _p, _stream

_declared = False
DT = {torch.float32: 0, torch.bfloat16: 2}
MAX_STATES = 128


def lib():
    global _declared
    L = opcuda.lib()
    if not _declared:
        vp, i32, i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
        L.oxb_causal_conv.argtypes = [vp, i32, i32] + [vp] * 6 + [i64, i32, vp] + [i32] * 8 + [vp]
        L.oxb_selective_scan.argtypes = [vp, i32, i32] * 5 + [vp] * 7 + [i64, i32, vp] + [i32] * 7 + [vp]
        _declared = True
    return L


def _rows(x: torch.Tensor, what: str) -> torch.Tensor:
    """x with neighbouring columns, in a type that the kernels read."""
    if x.dtype not in DT:
        raise ValueError(f"{what} is float32 or bfloat16, not {x.dtype}")
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def _floats(v: Optional[torch.Tensor], what: str) -> Optional[torch.Tensor]:
    if v is None:
        return None
    if v.dtype != torch.float32:
        raise ValueError(f"{what} is float32, not {v.dtype}")
    return v.contiguous()


def _kept(v: torch.Tensor, what: str) -> torch.Tensor:
    """Slots that the kernels update in place: each one contiguous, any distance apart."""
    if v.stride(2) != 1 or v.stride(1) != v.shape[2]:
        raise ValueError(f"a slot of {what} is contiguous; strides are {v.stride()}")
    return v


def _out(out: Optional[torch.Tensor], T: int, C: int, dtype: torch.dtype, device) -> torch.Tensor:
    if dtype not in DT:
        raise ValueError(f"act_dtype is float32 or bfloat16, not {dtype}")
    if out is None:
        return torch.empty(T, C, dtype=dtype, device=device)
    if tuple(out.shape) != (T, C) or out.dtype != dtype or (out.stride(1) != 1 and C > 1):
        raise ValueError(f"out is [{T}, {C}] in {dtype} with neighbouring columns, not {tuple(out.shape)} in {out.dtype}")
    return out


def causal_conv(x, w, bias, meta, window, act, act_dtype, out=None):
    x, w, bias, window = _rows(x, "x"), _floats(w, "w"), _floats(bias, "bias"), _kept(window, "window")
    T, C = x.shape
    y = _out(out, T, C, act_dtype, x.device)
    _check(lib().oxb_causal_conv(x.data_ptr(), x.stride(0), DT[x.dtype], w.data_ptr(), _p(bias), meta.query_start.data_ptr(),
                                 meta.seq_lens.data_ptr(), meta.state_slots.data_ptr(), window.data_ptr(), window.stride(0), window.shape[0],
                                 y.data_ptr(), y.stride(0), DT[act_dtype], meta.seq_lens.shape[0], T, C, w.shape[1], int(act == "silu"),
                                 meta.max_query_len, _stream()), "oxb_causal_conv")
    return y


def selective_scan(u, dt, a, b, c, d, z, dt_bias, meta, state, act_dtype, out=None):
    T, C = u.shape
    N = a.shape[1]
    if not 1 <= N <= MAX_STATES:
        raise ValueError(f"the scan takes 1 to {MAX_STATES} states, not {N}")
    u, dt, b, c = _rows(u, "u"), _rows(dt, "dt"), _rows(b, "b"), _rows(c, "c")
    if u.dtype != dt.dtype:  # (the kernels read them as one type)
        u, dt = u.float(), dt.float()
    z = None if z is None else _rows(z, "z")
    a, d, dt_bias, state = _floats(a, "a"), _floats(d, "d"), _floats(dt_bias, "dt_bias"), _kept(state, "state")
    y = _out(out, T, C, act_dtype, u.device)
    at = lambda m: (m.data_ptr(), m.stride(0), DT[m.dtype])  # noqa: E731
    _check(lib().oxb_selective_scan(*at(u), *at(dt), *((None, 0, 0) if z is None else at(z)), *at(b), *at(c), a.data_ptr(), _p(d),
                                    _p(dt_bias), meta.query_start.data_ptr(), meta.seq_lens.data_ptr(), meta.state_slots.data_ptr(),
                                    state.data_ptr(), state.stride(0), state.shape[0], *at(y), meta.seq_lens.shape[0], T, C, N, meta.max_query_len, _stream()),
           "oxb_selective_scan")
    return y
