"""Bindings of the kernels of state-space layers (``csrc/oxb_conv.cu``, ``csrc/oxb_ssm.cu``).  CUDA tensors only; see
:func:`oxidize_b200.ops.causal_conv` and :func:`oxidize_b200.ops.selective_scan` for the operators' meaning."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import MAX_SCAN_STATES
from . import cuda as opcuda
from .cuda import _check, _p, _stream

_declared = False
DT = {torch.float32: 0, torch.bfloat16: 2}
MAX_STRIDE = 2 ** 31 - 1  # values from row to row: a 32-bit number for the kernels (offsets of rows are 64-bit ones)


def lib():
    global _declared
    L = opcuda.lib()
    if not _declared:
        vp, i32, i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
        L.oxb_causal_conv.argtypes = [vp, i32, i32] + [vp] * 6 + [i64, i32, vp] + [i32] * 8 + [vp]
        L.oxb_selective_scan.argtypes = [vp, i32, i32] * 5 + [vp] * 7 + [i64, i32, vp] + [i32] * 7 + [vp]
        _declared = True
    return L


def _elsewhere(here: int, **tensors: Optional[torch.Tensor]) -> ValueError:
    """What the kernels are given lies on the current device, in whose stream they run."""
    return ValueError(f"not on the current device, cuda:{here}: " + ", ".join(f"{k} on {v.device}" for k, v in tensors.items()
                                                                             if v is not None and v.get_device() != here))


def _rows(x: torch.Tensor, what: str):
    """(x with neighbouring columns, the three arguments that stand for it) in a type that the kernels read."""
    code = DT.get(x.dtype)
    if code is None:
        raise ValueError(f"{what} is float32 or bfloat16, not {x.dtype}")
    ld, one = x.stride()
    if (one != 1 and x.shape[1] != 1) or (ld > MAX_STRIDE and x.shape[0] > 1):
        x = x.contiguous()
        ld = x.stride(0)
    return x, (x.data_ptr(), ld, code)


def _floats(v: Optional[torch.Tensor], what: str) -> Optional[torch.Tensor]:
    if v is None:
        return None
    if v.dtype != torch.float32:
        raise ValueError(f"{what} is float32, not {v.dtype}")
    return v if v.is_contiguous() else v.contiguous()


def _kept(v: torch.Tensor, what: str):
    """Slots that the kernels update in place, each one contiguous, any distance apart: address, distance, count."""
    n, _, width = v.shape
    step, row, one = v.stride()
    if one != 1 or row != width:
        raise ValueError(f"a slot of {what} is contiguous; strides are {v.stride()}")
    return v.data_ptr(), step, n


def _sequences(meta, here: int):
    """Query starts, lengths with this step's rows, slots, and how many sequences there are."""
    starts, lens, slots = meta.query_start, meta.seq_lens, meta.state_slots
    n = lens.shape[0]
    if (starts.shape[0] <= n or slots.shape[0] < n or not starts.dtype == lens.dtype == slots.dtype == torch.int32
            or not (starts.is_contiguous() and lens.is_contiguous() and slots.is_contiguous())):
        raise ValueError(f"a step of {n} sequences has that many lengths and slots and a query start more, contiguous in int32, not {starts.dtype} "
                         f"{tuple(starts.shape)}, {lens.dtype} and {slots.dtype} {tuple(slots.shape)}")
    if not starts.get_device() == lens.get_device() == slots.get_device() == here:
        raise _elsewhere(here, query_start=starts, seq_lens=lens, state_slots=slots)
    return (starts.data_ptr(), lens.data_ptr(), slots.data_ptr()), n


def _out(out: Optional[torch.Tensor], T: int, C: int, dtype: torch.dtype, like: torch.Tensor) -> torch.Tensor:
    if dtype not in DT:
        raise ValueError(f"act_dtype is float32 or bfloat16, not {dtype}")
    if out is None:
        return like.new_empty((T, C), dtype=dtype)
    if out.shape != (T, C) or out.dtype != dtype or (out.stride(1) != 1 and C > 1):
        raise ValueError(f"out is [{T}, {C}] in {dtype} with neighbouring columns, not {tuple(out.shape)} in {out.dtype}")
    if out.stride(0) > MAX_STRIDE and T > 1:
        raise ValueError(f"rows of out are at most {MAX_STRIDE} values apart, not {out.stride(0)}")
    return out


def _extent(v: torch.Tensor):
    """First byte of a matrix, bytes of it whole and of a row."""
    (T, C), (ld, one), size = v.shape, v.stride(), v.element_size()
    row = ((C - 1) * one + 1) * size
    return v.data_ptr(), (T - 1) * ld * size + row, row


def _apart(v: Optional[torch.Tensor], out: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """v, or a copy of it where ``out`` shares memory with it: rows are read after others were written.  Columns side by side in rows of
    one length share none."""
    if v is None or out is None or out.dim() != 2 or v.numel() == 0 or out.numel() == 0:
        return v
    (at, size, row), (at_out, size_out, row_out) = _extent(v), _extent(out)
    if at + size <= at_out or at_out + size_out <= at:
        return v
    ld = v.stride(0) * v.element_size()
    if v.shape[0] > 1 and ld > 0 and ld == out.stride(0) * out.element_size() and row <= (at_out - at) % ld <= ld - row_out:
        return v
    return v.clone()


def causal_conv(x, w, bias, meta, window, act, act_dtype, out=None):
    T, C = x.shape
    here = torch._C._cuda_getDevice()
    if not (x.get_device() == w.get_device() == window.get_device() == here and (bias is None or bias.get_device() == here)
            and (out is None or out.get_device() == here)):
        raise _elsewhere(here, x=x, w=w, bias=bias, window=window, out=out)
    x, at_x = _rows(_apart(x, out), "x")
    w, bias = _floats(w, "w"), _floats(bias, "bias")
    seqs, B = _sequences(meta, here)
    y = _out(out, T, C, act_dtype, x)
    _check(lib().oxb_causal_conv(*at_x, w.data_ptr(), _p(bias), *seqs, *_kept(window, "window"), y.data_ptr(), y.stride(0), DT[act_dtype], B, T, C,
                                 w.shape[1], act == "silu", meta.max_query_len, _stream()), "oxb_causal_conv")
    return y


def selective_scan(u, dt, a, b, c, d, z, dt_bias, meta, state, act_dtype, out=None):
    T, C = u.shape
    N = a.shape[1]
    if not 1 <= N <= MAX_SCAN_STATES:
        raise ValueError(f"the scan takes 1 to {MAX_SCAN_STATES} states, not {N}")
    here = torch._C._cuda_getDevice()
    if not (u.get_device() == dt.get_device() == a.get_device() == b.get_device() == c.get_device() == state.get_device() == here
            and (z is None or z.get_device() == here) and (d is None or d.get_device() == here) and (dt_bias is None or dt_bias.get_device() == here)
            and (out is None or out.get_device() == here)):
        raise _elsewhere(here, u=u, dt=dt, a=a, b=b, c=c, d=d, z=z, dt_bias=dt_bias, state=state, out=out)
    if u.dtype != dt.dtype and u.dtype in DT and dt.dtype in DT:  # (the kernels read them as one type)
        u, dt = u.float(), dt.float()
    if out is not None:
        u, dt, b, c, z = (_apart(v, out) for v in (u, dt, b, c, z))
    (u, at_u), (dt, at_dt), (b, at_b), (c, at_c) = _rows(u, "u"), _rows(dt, "dt"), _rows(b, "b"), _rows(c, "c")
    z, at_z = (None, (None, 0, 0)) if z is None else _rows(z, "z")
    a, d, dt_bias = _floats(a, "a"), _floats(d, "d"), _floats(dt_bias, "dt_bias")
    seqs, B = _sequences(meta, here)
    y = _out(out, T, C, act_dtype, u)
    _check(lib().oxb_selective_scan(*at_u, *at_dt, *at_z, *at_b, *at_c, a.data_ptr(), _p(d), _p(dt_bias), *seqs, *_kept(state, "state"),
                                    y.data_ptr(), y.stride(0), DT[act_dtype], B, T, C, N, meta.max_query_len, _stream()), "oxb_selective_scan")
    return y
