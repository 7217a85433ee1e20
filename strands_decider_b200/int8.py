"""W8A8 operators on torch tensors: int8 codes with one fp32 scale per row, and their product.

    q, s = rmsnorm(x, w, eps, delta=d, resid_out=x)      # x += d; RMSNorm(x) * (1 + w) as codes
    q, s = quantize_act(act, lo=act_lo)                  # a mixer's or SwiGLU's planes as codes
    linear(q, s, quantize("int8", weight), out)          # out = codes @ codes.T * scales

Thin checks (csrc/int8_torch.cpp) over `b200_quantize_act_int8`, `b200_rmsnorm_int8` and
`b200_linear_int8` (the contracts are in include/strands_b200.h). A model whose weights are in the
"int8" format runs its whole forward on the same entry points (runtime.DecisionModel).

Every tensor is 2-D with contiguous rows (any row stride of whole 16 bytes), on one CUDA device.
Calls go to that device's current stream, whichever device is current, and only enqueue work:
they can be captured in a CUDA graph. A tensor or shape an operator does not take raises
ValueError or _lib.B200Error before anything is launched.
"""

from __future__ import annotations

import torch

from . import _lib
from .weights import PackedWeight

_EPILOGUE = {"store": _lib.EP_STORE, "residual": _lib.EP_RESID_ADD, "swiglu": _lib.EP_SWIGLU}


def _call(name: str, device: int, *args) -> None:
    """One operator on the device's current stream, with that device current."""
    if device < 0:
        raise ValueError("b200 kernels take CUDA tensors only")
    op = getattr(_lib.int8_ops(), name)
    if torch._C._cuda_getDevice() == device:
        status = op(*args, _lib.raw_stream(device))
    else:
        with torch.cuda.device(device):
            status = op(*args, _lib.raw_stream(device))
    if status:
        _lib.check(status)


def quantize_act(x: torch.Tensor, lo: torch.Tensor | None = None, out: torch.Tensor | None = None,
                 scale: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """x fp32 or bf16 [rows, k] (bf16: optionally with its low plane, v = x + lo) -> (codes int8
    [rows, k], scales fp32 [rows]), written into out / scale when given."""
    if out is None:
        out = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    if scale is None:
        scale = torch.empty(x.shape[:1], dtype=torch.float32, device=x.device)
    _call("quantize_act", x.get_device(), x, lo, out, scale)
    return out, scale


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float, delta: torch.Tensor | None = None,
            resid_out: torch.Tensor | None = None, out: torch.Tensor | None = None,
            scale: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """RMSNorm(x + delta) * (1 + w) as (codes int8 [rows, hidden], scales fp32 [rows]). x fp32;
    delta fp32 or bf16 or None; resid_out (with a delta) receives x + delta in fp32 and may be x."""
    if out is None:
        out = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    if scale is None:
        scale = torch.empty(x.shape[:1], dtype=torch.float32, device=x.device)
    _call("rmsnorm", x.get_device(), x, w, eps, delta, resid_out, out, scale)
    return out, scale


def linear(q: torch.Tensor, scale: torch.Tensor, weight: PackedWeight, out: torch.Tensor, epilogue: str = "store",
           lo: torch.Tensor | None = None, n_valid: int | None = None) -> torch.Tensor:
    """y = (q @ codes.T) * scale * channel scales into `out`: "store" (fp32 [rows, n_valid]),
    "residual" (fp32, out += y) or "swiglu" (bf16 [rows, n_valid / 2] from weight rows interleaved
    by weights.interleave_gate_up; `lo` optionally receives the low plane, bf16 or e4m3 bytes).
    n_valid: the outputs written, by default all of the weight's rows."""
    if weight.fmt != "int8" or weight.row_scale is None:
        raise ValueError(f"linear takes int8 weights with their row scales, not {weight.fmt!r}")
    ep = _EPILOGUE.get(epilogue)
    if ep is None:
        raise ValueError(f"epilogue must be one of {sorted(_EPILOGUE)}, not {epilogue!r}")
    n = weight.n
    _call("linear", q.get_device(), q, scale, weight.data, weight.row_scale, out, lo, n, weight.k,
          n if n_valid is None else n_valid, ep)
    return out
