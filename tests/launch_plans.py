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


# (m, n, k, epilogue, CTAs per cluster, stages): products of the int8 split kernel on 148 SMs whose
# k-blocks pass an operand ring of 3 to 12 stages more than once. A ring of 2 is never passed twice.
# The first runs two CTAs to an SM.
RINGS = [(300, 12288, 2048, "swiglu", 1, 3), (300, 12288, 1040, "store", 1, 3), (200, 12288, 512, "residual", 1, 3),
         (129, 12288, 640, "swiglu", 1, 4), (37, 32768, 1152, "store", 1, 4), (33, 128, 2064, "store", 4, 4),
         (17, 128, 1536, "residual", 2, 5), (17, 4096, 3088, "swiglu", 4, 5), (1, 1280, 16384, "store", 8, 5),
         (600, 2048, 2048, "residual", 1, 6), (600, 1000, 3088, "store", 2, 6), (113, 128, 8208, "swiglu", 4, 6),
         (81, 12288, 2048, "store", 1, 7), (81, 6144, 4096, "swiglu", 2, 7), (81, 128, 8208, "residual", 4, 7),
         (129, 6144, 2064, "residual", 1, 8), (65, 6144, 6144, "store", 2, 8), (65, 128, 8208, "store", 4, 8),
         (49, 12288, 3088, "swiglu", 1, 9), (49, 6144, 6144, "residual", 2, 9), (49, 128, 16384, "store", 4, 9),
         (33, 12288, 3088, "store", 1, 10), (33, 6144, 6144, "swiglu", 2, 10), (33, 128, 16384, "residual", 4, 10),
         (17, 12288, 3088, "residual", 1, 11), (17, 6144, 6144, "store", 2, 11), (17, 4096, 16384, "store", 4, 11),
         (17, 128, 65536, "swiglu", 8, 11),
         (1, 12288, 3088, "store", 1, 12), (8, 6144, 8208, "residual", 2, 12), (16, 4096, 16384, "swiglu", 4, 12),
         (8, 1000, 65536, "store", 8, 12)]

# (m, n, k, tokens per tile): products of the int8 pair kernel whose weights are taken in several
# groups of output tiles, the last of them smaller, with more tiles than pairs
GROUPS = [(600, 12032, 8192, 256), (760, 6400, 16384, 192)]
