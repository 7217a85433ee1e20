"""W8A8 operators on torch tensors: int8 codes with one fp32 scale per row, and their product.

    q, s = rmsnorm(x, w, eps, delta=d, resid_out=x)      # x += d; RMSNorm(x) * (1 + w) as codes
    q, s = quantize_act(act, lo=act_lo)                  # a mixer's or SwiGLU's planes as codes
    linear(q, s, quantize("int8", weight), out)          # out = codes @ codes.T * scales

Thin checks over `b200_rmsnorm_int8`, `b200_quantize_act_int8` and `b200_linear_int8` (the
contracts are in include/strands_b200.h). A model whose weights are in the "int8" format runs its
whole forward on the same entry points (runtime.DecisionModel).

Every tensor is 2-D with contiguous rows (any row stride of whole 16 bytes), on one CUDA device.
Calls go to that device's current stream, whichever device is current, and only enqueue work:
they can be captured in a CUDA graph. A tensor or shape an operator does not take raises
ValueError or _lib.B200Error before anything is launched.
"""

from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from .weights import PackedWeight

_EPILOGUE = {"store": _lib.EP_STORE, "residual": _lib.EP_RESID_ADD, "swiglu": _lib.EP_SWIGLU}
_ACT = {torch.float32: _lib.ACT_F32, torch.bfloat16: _lib.ACT_BF16}
_INT8 = _lib.FMT["int8"]
_LO_FORMAT = {torch.bfloat16: _lib.LO_BF16, torch.uint8: _lib.LO_E4M3, torch.float8_e4m3fn: _lib.LO_E4M3}


def _rows(name: str, t: torch.Tensor, dtype, device: int, rows: int, k: int) -> int:
    """The row stride of t in elements, after checking its type, place and shape."""
    if t.dtype is not dtype or t.get_device() != device or t.shape != (rows, k):
        raise ValueError(f"{name} must be {dtype} of shape {(rows, k)} on cuda:{device}, not {t.dtype} of "
                         f"{tuple(t.shape)} on {t.device}")
    if t.is_contiguous():
        return k
    ld, step = t.stride()
    if step != 1 and k > 1:
        raise ValueError(f"{name}'s rows must be contiguous")
    return ld if rows > 1 else k


def _vector(name: str, t: torch.Tensor, device: int, n: int) -> None:
    if t.dtype is not torch.float32 or t.get_device() != device or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous fp32 tensor of {n} on cuda:{device}")


def _place(name: str, t: torch.Tensor) -> tuple[int, int, int]:
    """(device index, rows, columns) of the tensor an operator goes by."""
    device = t.get_device()
    if device < 0:
        raise ValueError("b200 kernels take CUDA tensors only")
    shape = t.shape
    if len(shape) != 2:
        raise ValueError(f"{name} must be 2-D")
    return device, shape[0], shape[1]


def _call(device: int, name: str, *args) -> None:
    """One entry point on the device's current stream, with that device current."""
    f = getattr(_lib.load(), name)
    if torch._C._cuda_getDevice() == device:
        status = f(*args, _lib.raw_stream(device))
    else:
        with torch.cuda.device(device):
            status = f(*args, _lib.raw_stream(device))
    if status:
        _lib.check(status)


def _codes_out(out: torch.Tensor | None, scale: torch.Tensor | None, device: int, rows: int, k: int):
    if out is None:
        out, ldq = torch.empty(rows, k, dtype=torch.int8, device=device), k
    else:
        ldq = _rows("out", out, torch.int8, device, rows, k)
    if scale is None:
        scale = torch.empty(rows, dtype=torch.float32, device=device)
    else:
        _vector("scale", scale, device, rows)
    return out, ldq, scale


def quantize_act(x: torch.Tensor, lo: torch.Tensor | None = None, out: torch.Tensor | None = None,
                 scale: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """x fp32 or bf16 [rows, k] (bf16: optionally with its low plane, v = x + lo) -> (codes int8
    [rows, k], scales fp32 [rows]), written into out / scale when given."""
    dev, rows, k = _place("x", x)
    kind = _ACT.get(x.dtype)
    if kind is None:
        raise ValueError(f"x must be float32 or bfloat16, not {x.dtype}")
    ldx = _rows("x", x, x.dtype, dev, rows, k)
    if lo is not None:
        if kind != _lib.ACT_BF16:
            raise ValueError("a low plane belongs to bfloat16 activations")
        if _rows("lo", lo, torch.bfloat16, dev, rows, k) != ldx:
            raise ValueError("x and lo must have the same row stride")
    out, ldq, scale = _codes_out(out, scale, dev, rows, k)
    _call(dev, "b200_quantize_act_int8", x.data_ptr(), lo.data_ptr() if lo is not None else None, kind, rows, k, ldx,
          out.data_ptr(), ldq, scale.data_ptr())
    return out, scale


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float, delta: torch.Tensor | None = None,
            resid_out: torch.Tensor | None = None, out: torch.Tensor | None = None,
            scale: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """RMSNorm(x + delta) * (1 + w) as (codes int8 [rows, hidden], scales fp32 [rows]). x fp32;
    delta fp32 or bf16 or None; resid_out (with a delta) receives x + delta in fp32 and may be x."""
    dev, rows, hidden = _place("x", x)
    ldx = _rows("x", x, torch.float32, dev, rows, hidden)
    _vector("w", w, dev, hidden)
    kind, ldd, lds = _lib.ACT_F32, 0, 0
    if delta is not None:
        kind = _ACT.get(delta.dtype)
        if kind is None:
            raise ValueError(f"delta must be float32 or bfloat16, not {delta.dtype}")
        ldd = _rows("delta", delta, delta.dtype, dev, rows, hidden)
    if resid_out is not None:
        if delta is None:
            raise ValueError("resid_out needs a delta")
        lds = _rows("resid_out", resid_out, torch.float32, dev, rows, hidden)
    out, ldq, scale = _codes_out(out, scale, dev, rows, hidden)
    _call(dev, "b200_rmsnorm_int8", x.data_ptr(), ldx, delta.data_ptr() if delta is not None else None, kind, ldd,
          resid_out.data_ptr() if resid_out is not None else None, lds, rows, hidden, w.data_ptr(), eps,
          out.data_ptr(), ldq, scale.data_ptr())
    return out, scale


def linear(q: torch.Tensor, scale: torch.Tensor, weight: PackedWeight, out: torch.Tensor, epilogue: str = "store",
           lo: torch.Tensor | None = None, n_valid: int | None = None) -> torch.Tensor:
    """y = (q @ codes.T) * scale * channel scales into `out`: "store" (fp32 [rows, n_valid]),
    "residual" (fp32, out += y) or "swiglu" (bf16 [rows, n_valid / 2] from weight rows interleaved
    by weights.interleave_gate_up; `lo` optionally receives the low plane, bf16 or e4m3 bytes).
    n_valid: the outputs written, by default all of the weight's rows."""
    dev, rows, k = _place("q", q)
    if weight.fmt != "int8":
        raise ValueError(f"linear takes int8 weights, not {weight.fmt!r}")
    ep = _EPILOGUE.get(epilogue)
    if ep is None:
        raise ValueError(f"epilogue must be one of {sorted(_EPILOGUE)}, not {epilogue!r}")
    n = weight.n if n_valid is None else n_valid
    ldx = _rows("q", q, torch.int8, dev, rows, k)
    _vector("scale", scale, dev, rows)
    codes, ws = weight.data, weight.row_scale
    if ws is None or _rows("the weight", codes, torch.int8, dev, weight.n, weight.k) != weight.k:
        raise ValueError("the weight must hold contiguous int8 codes and their row scales")
    _vector("the weight's row scales", ws, dev, weight.n)
    swiglu = ep == _lib.EP_SWIGLU
    if swiglu and n % 2:
        raise ValueError("a SwiGLU has as many up as gate features")
    cols = n // 2 if swiglu else n
    ldo = _rows("out", out, torch.bfloat16 if swiglu else torch.float32, dev, rows, cols)
    lo_offset = lo_format = 0
    if lo is not None:
        if not swiglu or lo.dtype not in _LO_FORMAT:
            raise ValueError("a low plane belongs to the SwiGLU, in bfloat16 or e4m3 bytes")
        if _rows("lo", lo, lo.dtype, dev, rows, cols) != ldo:
            raise ValueError("out and lo must have the same row stride")
        gap = lo.data_ptr() - out.data_ptr()
        if gap == 0 or gap % 2:
            raise ValueError("lo must be a tensor of its own, a whole number of bf16 from out")
        lo_offset, lo_format = gap // 2, _LO_FORMAT[lo.dtype]
    qw = _lib.QWeight(_INT8, weight.n, weight.k, codes.data_ptr(), None, ws.data_ptr(), None, None)
    o = _lib.LinearOut(ep, n, out.data_ptr(), ldo, lo_offset, lo_format)
    _call(dev, "b200_linear_int8", q.data_ptr(), scale.data_ptr(), rows, k, ldx, C.byref(qw), C.byref(o))
    return out
