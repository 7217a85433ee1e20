"""What b200_linear and b200_linear_int8 would launch (host arithmetic, no GPU needed)."""

from __future__ import annotations

import ctypes as C

from strands_decider_b200 import _lib

EPILOGUE = {"store": _lib.EP_STORE, "residual": _lib.EP_RESID_ADD, "swiglu": _lib.EP_SWIGLU}
ADDRESS = 1 << 20   # stands for an aligned device pointer: a plan reads nothing


def int8_plan(m, n, k, ep="store", lo=0, sms=148, ldo=None, out=ADDRESS, n_valid=None):
    """The plan of an int8 product into rows of `ldo` elements at `out` (sms 0: the current device)."""
    nv = n if n_valid is None else n_valid
    plan, w = _lib.LaunchPlan(), _lib.QWeight(_lib.FMT["int8"], n, k, ADDRESS, None, ADDRESS, None, None)
    o = _lib.LinearOut(EPILOGUE[ep], nv, out, ldo or (nv // 2 if ep == "swiglu" else nv), lo, 0)
    _lib.call("b200_linear_int8_plan", ADDRESS, ADDRESS, m, k, k, C.byref(w), C.byref(o), sms, C.byref(plan))
    return plan


def bf16_plan(m, n, k, ep="store", planes=2, sms=148):
    plan, w = _lib.LaunchPlan(), _lib.QWeight(_lib.FMT["bf16"], n, k, ADDRESS, None, None, None, None)
    o = _lib.LinearOut(EPILOGUE[ep], n, ADDRESS, n // 2 if ep == "swiglu" else n, 0, 0)
    _lib.call("b200_linear_plan", ADDRESS, ADDRESS if planes == 2 else None, m, k, k, C.byref(w), C.byref(o), sms,
              C.byref(plan))
    return plan
