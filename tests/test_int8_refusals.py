"""The int8 (W8A8) entry points refuse what they do not take with a status and their own name in
the message, on the host, before anything touches a device (no GPU needed)."""

from __future__ import annotations

import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from strands_decider_b200 import _lib, build

    build.build()
    return _lib.load()


@pytest.fixture(scope="module")
def p16():
    buf = (C.c_uint8 * 4096)()
    p16.keep = buf
    return (C.cast(buf, C.c_void_p).value + 15) // 16 * 16


def _refused(lib, name, status, *args):
    assert getattr(lib, name)(*args) == status, lib.b200_last_error()
    assert lib.b200_last_error().decode().startswith(name + ":")


def test_quantize_act_int8(lib, p16):
    good = dict(x=p16, lo=None, type=0, rows=4, k=64, ldx=64, q=p16, ldq=64, scale=p16)

    def bad(status, **kw):
        a = {**good, **kw}
        _refused(lib, "b200_quantize_act_int8", status, a["x"], a["lo"], a["type"], a["rows"], a["k"], a["ldx"],
                 a["q"], a["ldq"], a["scale"], None)

    for name in ("x", "q", "scale"):
        bad(1, **{name: None})
    bad(1, type=2)
    bad(1, type=-1)
    bad(1, lo=p16)                       # a low plane of fp32 activations
    bad(2, rows=0)
    bad(2, rows=-3)
    bad(2, rows=(1 << 30) + 1)
    bad(2, k=0)
    bad(2, k=24, ldx=32, ldq=32)         # not a multiple of 16
    bad(2, k=65552, ldx=65552, ldq=65552)
    bad(2, ldx=48)                       # a row does not fit
    bad(2, ldx=66)
    bad(2, type=1, ldx=68)               # bf16 rows of 8 bytes past 16
    bad(2, ldq=48)
    bad(2, ldq=72)
    bad(2, x=p16 + 4)
    bad(2, q=p16 + 8)
    bad(2, type=1, lo=p16 + 2)
    bad(2, scale=p16 + 2)


def test_rmsnorm_int8(lib, p16):
    good = dict(x=p16, ldx=64, delta=p16, dt=0, ldd=64, sum=p16, lds=64, rows=2, k=64, w=p16, eps=1e-6, q=p16,
                ldq=64, scale=p16)

    def bad(status, **kw):
        a = {**good, **kw}
        _refused(lib, "b200_rmsnorm_int8", status, a["x"], a["ldx"], a["delta"], a["dt"], a["ldd"], a["sum"], a["lds"],
                 a["rows"], a["k"], a["w"], a["eps"], a["q"], a["ldq"], a["scale"], None)

    for name in ("x", "w", "q", "scale"):
        bad(1, **{name: None})
    bad(1, delta=None)                   # a sum of nothing
    bad(1, dt=3)
    bad(1, eps=-1e-6)
    bad(1, eps=0.0)
    bad(1, eps=float("nan"))
    bad(2, rows=0)
    bad(2, rows=(1 << 30) + 1)
    bad(2, k=0)
    bad(2, k=40, ldx=64)
    bad(2, k=65552, ldx=65552, ldd=65552, lds=65552, ldq=65552)
    for name in ("ldx", "ldd", "lds", "ldq"):
        bad(2, **{name: 48})
        bad(2, **{name: 66})
    bad(2, dt=1, ldd=68)
    for name in ("x", "delta", "sum", "w", "q"):
        bad(2, **{name: p16 + 4})


def test_linear_int8(lib, p16):
    from strands_decider_b200 import _lib

    def bad(status, q=p16, xs=p16, m=4, k=64, ldx=64, fmt=4, n=128, wk=64, data=p16, rs=p16, ep=0, nv=128, out=p16,
            ldo=128, lo=0, lof=0, w=True, o=True):
        qw = _lib.QWeight(fmt, n, wk, data, None, rs, None, None)
        lo_ = _lib.LinearOut(ep, nv, out, ldo, lo, lof)
        _refused(lib, "b200_linear_int8", status, q, xs, m, k, ldx, C.byref(qw) if w else None,
                 C.byref(lo_) if o else None, None)

    for kw in (dict(q=None), dict(xs=None), dict(data=None), dict(out=None), dict(rs=None), dict(w=False),
               dict(o=False), dict(ep=3), dict(ep=-1), dict(lof=2)):
        bad(1, **kw)
    for fmt in (0, 1, 2, 3, 5, -1):
        bad(3, fmt=fmt)
    for kw in (dict(m=0), dict(m=-1), dict(m=(1 << 30) + 1), dict(n=(1 << 30) + 1), dict(k=0, wk=0), dict(n=0), dict(wk=128), dict(k=40, wk=40),
               dict(k=65552, wk=65552, ldx=65552), dict(ldx=48), dict(ldx=72), dict(q=p16 + 8), dict(data=p16 + 4),
               dict(nv=0), dict(nv=129), dict(ldo=127), dict(out=p16 + 2), dict(ep=2, nv=64), dict(ep=2, ldo=63),
               dict(ep=2, out=p16 + 1), dict(xs=p16 + 2), dict(rs=p16 + 1)):
        bad(2, **kw)


def test_int8_weights_stay_with_their_linear(lib, p16):
    """The weight-only entry points refuse the format instead of reading it as another one."""
    from strands_decider_b200 import _lib

    qw = _lib.QWeight(4, 256, 128, p16, p16, p16, p16, p16)
    o = _lib.LinearOut(0, 256, p16, 256, 0, 0)
    nbytes = C.c_size_t()
    assert lib.b200_linear(p16, None, 4, 128, 128, C.byref(qw), C.byref(o), None) == 3
    assert lib.b200_linear_simt(p16, None, 4, 128, 128, C.byref(qw), C.byref(o), None) == 3
    assert lib.b200_dequantize(C.byref(qw), p16, None) == 3
    assert lib.b200_dequantize_lo8(C.byref(qw), p16, p16, None) == 3
    assert lib.b200_tile_bytes(4, 256, 128, C.byref(nbytes), C.byref(nbytes)) == 3
    assert lib.b200_tile_weights(C.byref(qw), p16, p16, None) == 3
    assert lib.b200_linear_nvfp4_native(p16, p16, 4, 256, C.byref(_lib.QWeight(4, 256, 256, p16, p16, p16, None, None)),
                                        p16, C.byref(o), None) == 3
    # the quantiser: row scales needed; the row rules of the activation quantiser, under its own name
    _refused(lib, "b200_quantize", 1, 4, p16, 256, 128, p16, None, None, None)
    _refused(lib, "b200_quantize", 2, 4, p16, 256, 120, p16, None, p16, None)
    _refused(lib, "b200_quantize", 2, 4, p16, 256, 128, p16 + 4, None, p16, None)


def test_python_operators_refuse_cpu_tensors_and_wrong_types():
    from strands_decider_b200 import int8
    from strands_decider_b200.weights import PackedWeight

    x = torch.zeros(2, 64)
    w = PackedWeight("int8", 128, 64, torch.zeros(128, 64, dtype=torch.int8), row_scale=torch.ones(128))
    with pytest.raises(ValueError, match="CUDA"):
        int8.quantize_act(x)
    with pytest.raises(ValueError, match="CUDA"):
        int8.rmsnorm(x, torch.zeros(64), 1e-6)
    with pytest.raises(ValueError, match="CUDA"):
        int8.linear(x.to(torch.int8), torch.ones(2), w, torch.zeros(2, 128))


def test_python_operators_refuse_what_is_not_a_cuda_tensor(lib):
    from strands_decider_b200 import _lib, int8
    from strands_decider_b200.weights import PackedWeight

    x, s, w = torch.zeros(2, 16), torch.zeros(2), torch.zeros(16)
    q, out = torch.zeros(2, 16, dtype=torch.int8), torch.zeros(2, 8)
    pw = PackedWeight("int8", 8, 16, torch.zeros(8, 16, dtype=torch.int8), row_scale=torch.zeros(8))
    for bad in (lambda: int8.quantize_act(x), lambda: int8.rmsnorm(x, w, 1e-6), lambda: int8.linear(q, s, pw, out),
                lambda: int8.linear(q, s, PackedWeight("int8", 8, 16, pw.data), out),
                lambda: int8.linear(q, s, pw, out, epilogue="gelu")):
        with pytest.raises(ValueError):
            bad()
    ops = _lib.int8_ops()
    for bad in (lambda: ops.quantize_act(x, None, q, s, 0), lambda: ops.rmsnorm(x, w, 1e-6, None, None, q, s, 0),
                lambda: ops.linear(q, s, pw.data, pw.row_scale, out, None, 8, 16, 8, 0, 0)):
        with pytest.raises(ValueError, match="CUDA tensors only"):
            bad()
    for bad in (lambda: ops.quantize_act(x.numpy(), None, q, s, 0), lambda: ops.linear(None, *[x] * 10),
                lambda: ops.rmsnorm(x), lambda: ops.bind(1, 2), lambda: ops.bind("a", 2, 3)):
        with pytest.raises(TypeError):
            bad()
