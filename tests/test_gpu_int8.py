"""The int8 (W8A8) operators against plain implementations in 64 bits.

* Codes and scales (b200_quantize_act_int8, b200_rmsnorm_int8, b200_quantize): equal to
  oracle.quant's, every step of which is one fp32 rounding.
* The product (b200_linear_int8): against the fp64 product of the codes. The int32 sum is exact,
  so a stored output has three roundings (sum to fp32, two scales): |y - ref| <= 3 * 2^-24 |ref|
  to first order, tested with 4 * 2^-24. A residual adds one rounding of the result.
* The SwiGLU: g, u as above; silu by the fast exponential and division. Relative errors: at most
  (2 + 1.2 |g|) * 2^-23 (exponential, its argument's rounding included), 2 * 2^-23 (division),
  3 * 2^-24 |g| (g's own error through the exponent) and 4 * 2^-24 (1 + e, the products), together
  6 * 2^-23 + 2.7 |g| * 2^-23, which 2^-17 + |g| * 2^-22 exceeds while |g| < 80; then a plane's
  rounding: 2^-8 for the hi plane alone, 2^-16 for hi + bf16 lo, and for an e4m3 lo plane 2^-4 of
  |h - hi| <= 2^-8 |h|, or half a step of its subnormals, 2^-10 / 2^6.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import quant as Q

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("the -m gpu tests need a CUDA device")
    from strands_decider_b200 import _lib

    _lib.load()
    yield
    torch.cuda.synchronize()
    assert _lib.read_fault() == 0


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _same_codes(q, scale, want_q, want_s):
    assert np.array_equal(scale.cpu().numpy(), want_s, equal_nan=True)
    assert np.array_equal(q.cpu().numpy(), want_q)


def _hard_rows(rows, k, seed):
    """Rows of varied size, with the ones a quantiser can get wrong in front."""
    x = torch.randn(rows, k, generator=_gen(seed)) * torch.exp(3 * torch.randn(rows, 1, generator=_gen(seed + 1)))
    hard = [torch.zeros(k), torch.full((k,), 3.0), torch.full((k,), 1e-45), torch.full((k,), 1.4e-36),
            torch.full((k,), 3e38), torch.arange(k).float() - k / 2]
    spike = torch.full((k,), 1e-30)
    spike[k - 1] = -1e30
    ties = torch.zeros(k)            # half codes: 0.5, 1.5, 2.5, ... of a scale of exactly 1
    ties[0] = 127.0
    ties[1:8] = torch.tensor([0.5, 1.5, 2.5, -0.5, -1.5, 63.5, -126.5])
    inf = torch.randn(k, generator=_gen(seed + 2))
    inf[k // 2] = float("-inf")
    nan = torch.randn(k, generator=_gen(seed + 3))
    nan[0] = float("nan")
    for i, h in enumerate(hard + [spike, ties, inf, nan]):
        if rows > 2 * i:
            x[2 * i] = h
    return x


ROW_SHAPES = [(1, 16), (1, 2048), (1, 6144), (3, 48), (5, 1040), (21, 2032), (33, 4096), (23, 8208), (4, 32784),
              (2, 65536), (1500, 144), (4099, 1152), (20011, 128), (10007, 16), (9601, 112), (40, 20000),
              (9000, 96), (2500, 272), (2500, 384), (3500, 704), (3001, 1392), (1500, 2400), (1200, 5648), (300, 12304),
              (70, 49168)]


@pytest.mark.parametrize("rows,k", ROW_SHAPES)
@pytest.mark.parametrize("kind", ["fp32", "bf16", "planes"])
def test_quantize_act_is_exact(rows, k, kind):
    from strands_decider_b200 import int8

    x = _hard_rows(rows, k, rows + k)
    lo = None
    if kind == "fp32":
        want = x
    else:
        hi = x.to(torch.bfloat16)
        want = hi.float()
        if kind == "planes":
            lo = (x - want).to(torch.bfloat16)
            want = want + lo.float()
        x = hi
    q, s = int8.quantize_act(x.cuda(), lo=lo.cuda() if lo is not None else None)
    _same_codes(q, s, *Q.quantize_int8_rows(want.numpy()))


@pytest.mark.parametrize("rows,k", ROW_SHAPES)
@pytest.mark.parametrize("delta", [None, torch.float32, torch.bfloat16])
def test_rmsnorm_is_exact(rows, k, delta):
    from strands_decider_b200 import int8

    x = _hard_rows(rows, k, rows + k + 1)
    w = torch.randn(k, generator=_gen(k)) * 0.2
    d = None if delta is None else torch.randn(rows, k, generator=_gen(7)).to(delta)
    want_q, want_s, want_t = Q.rmsnorm_int8(x.numpy(), w.numpy(), 1e-6, None if d is None else d.float().numpy())
    t = torch.empty(rows, k, device="cuda") if d is not None else None
    q, s = int8.rmsnorm(x.cuda(), w.cuda(), 1e-6, delta=d.cuda() if d is not None else None, resid_out=t)
    _same_codes(q, s, want_q, want_s)
    if t is not None:
        assert np.array_equal(t.cpu().numpy(), want_t, equal_nan=True)


def test_rmsnorm_in_place_and_without_a_sum():
    """The sum may land in x or in an fp32 delta, or nowhere; the codes are the same."""
    from strands_decider_b200 import int8

    x, d = torch.randn(37, 528).cuda(), torch.randn(37, 528).cuda()
    w = torch.randn(528).cuda()
    q0, s0 = int8.rmsnorm(x, w, 1e-5, delta=d)
    t = x + d
    x1, d1 = x.clone(), d.clone()
    q1, s1 = int8.rmsnorm(x1, w, 1e-5, delta=d, resid_out=x1)
    q2, s2 = int8.rmsnorm(x, w, 1e-5, delta=d1, resid_out=d1)
    for q, s in ((q1, s1), (q2, s2)):
        assert torch.equal(q, q0) and torch.equal(s, s0)
    assert torch.equal(x1, t) and torch.equal(d1, t)


def test_row_strides_and_what_lies_between_rows():
    """Views with a row stride read and write their own columns only."""
    from strands_decider_b200 import int8

    rows, k = 19, 272
    x = torch.full((rows, 400), float("nan")).cuda()
    x[:, 64:64 + k] = torch.randn(rows, k).cuda()
    q = torch.full((rows, 512), 99, dtype=torch.int8).cuda()
    s = torch.full((rows + 2,), -7.0).cuda()
    int8.quantize_act(x[:, 64:64 + k], out=q[:, 128:128 + k], scale=s[1:-1])
    _same_codes(q[:, 128:128 + k], s[1:-1], *Q.quantize_int8_rows(x[:, 64:64 + k].cpu().numpy()))
    assert (q[:, :128] == 99).all() and (q[:, 128 + k:] == 99).all() and s[0] == -7 and s[-1] == -7
    t = torch.full((rows, 300), 5.0).cuda()
    d = torch.randn(rows, 320).to(torch.bfloat16).cuda()
    w = torch.randn(k).cuda()
    int8.rmsnorm(x[:, 64:64 + k], w, 1e-6, delta=d[:, 16:16 + k], resid_out=t[:, 12:12 + k], out=q[:, 16:16 + k],
                 scale=s[:rows])
    wq, ws, wt = Q.rmsnorm_int8(x[:, 64:64 + k].cpu().numpy(), w.cpu().numpy(), 1e-6,
                                d[:, 16:16 + k].float().cpu().numpy())
    _same_codes(q[:, 16:16 + k], s[:rows], wq, ws)
    assert np.array_equal(t[:, 12:12 + k].cpu().numpy(), wt)
    assert (t[:, :12] == 5).all() and (t[:, 12 + k:] == 5).all()


@pytest.mark.parametrize("n,k", [(1, 16), (300, 2048), (129, 4112)])
def test_weight_quantiser_is_exact(n, k):
    from strands_decider_b200 import weights as W

    w = _hard_rows(n, k, 3) if n > 30 else torch.randn(n, k)
    pw = W.quantize("int8", w.cuda())
    parts = W.packed_to_numpy(pw)
    want = Q.quantize("int8", w.numpy())
    assert np.array_equal(parts["data"], want["data"])
    assert np.array_equal(parts["row_scale"], want["row_scale"], equal_nan=True)


# ----------------------------------------------------------------------------- the product


def _operands(m, n, k, seed):
    g = _gen(seed)
    q = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8)
    wq = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
    s = torch.exp(torch.randn(m, generator=g)) / 1024
    ws = torch.exp(torch.randn(n, generator=g)) / 1024
    return q, s, wq, ws


def _weight(wq, ws):
    from strands_decider_b200.weights import PackedWeight

    return PackedWeight("int8", wq.shape[0], wq.shape[1], wq.cuda(), row_scale=ws.cuda())


def _ref(q, s, wq, ws):
    """fp64 on the GPU (exact sums of whole numbers below 2^53)."""
    return ((q.cuda().double() @ wq.cuda().double().T) * s.cuda().double()[:, None]) * ws.cuda().double()


# one row to several tiles; outputs that are no multiple of anything; depths that end inside a tile
SHAPES = [(1, 1, 16), (1, 130, 64), (2, 2048, 2048), (7, 1000, 144), (8, 96, 8208), (9, 257, 1040), (16, 2304, 512),
          (17, 640, 2048), (31, 33, 48), (33, 129, 6144), (64, 1153, 528), (65, 256, 4112), (96, 8224, 256),
          (127, 384, 1024), (129, 127, 272), (200, 2048, 2032), (255, 600, 2064), (257, 520, 128), (511, 1025, 400),
          (1021, 2048, 2048), (1290, 2040, 1040), (2050, 4200, 336), (2050, 4201, 144),
          (4099, 2600, 1040), (9001, 1290, 144),
          (1, 20000, 2048), (3, 130, 16384), (8, 1000, 65536), (9, 16, 16400), (12, 9000, 3088), (16, 2048, 20480)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_store_and_residual(m, n, k):
    from strands_decider_b200 import int8

    q, s, wq, ws = _operands(m, n, k, m + n + k)
    w = _weight(wq, ws)
    ref = _ref(q, s, wq, ws)
    out = torch.full((m, n), 7.0, device="cuda")
    int8.linear(q.cuda(), s.cuda(), w, out)
    assert ((out.double() - ref).abs() <= 4 * U * ref.abs()).all()
    out = torch.randn(m, n, device="cuda") * ref.abs().mean().float()
    want = out.double() + ref
    int8.linear(q.cuda(), s.cuda(), w, out, epilogue="residual")
    assert ((out.double() - want).abs() <= 4 * U * ref.abs() + 1.01 * U * want.abs()).all()


SWIGLU_SHAPES = [(1, 128, 16), (1, 12288, 256), (5, 256, 144), (13, 1152, 2048), (16, 128, 1040), (24, 640, 528),
                 (96, 1024, 2048), (130, 384, 400), (300, 2432, 1024), (600, 5504, 1040), (500, 5504, 1040), (1030, 1280, 272), (2050, 4224, 160),
                 (3333, 3200, 144), (1, 128, 4096), (3, 384, 16384), (8, 20096, 2048), (9, 256, 2064), (16, 12288, 2048)]


@pytest.mark.parametrize("m,n,k", SWIGLU_SHAPES)
@pytest.mark.parametrize("lo", [None, "bf16", "e4m3"])
def test_linear_swiglu(m, n, k, lo):
    from strands_decider_b200 import int8

    q, s, wq, ws = _operands(m, n, k, m + n)
    # |g|, |u| of a few tens at most: the codes' products have a standard deviation of 74^2 sqrt(k)
    s = torch.full((m,), 4.0 / (74.0 ** 2 * k ** 0.5))
    ws = torch.exp(0.2 * torch.randn(n, generator=_gen(n)))
    y = _ref(q, s, wq, ws).reshape(m, -1, 2, 64)
    g, u = y[:, :, 0], y[:, :, 1]
    ref = (g * torch.sigmoid(g) * u).reshape(m, n // 2)
    out = torch.zeros(m, n // 2, dtype=torch.bfloat16, device="cuda")
    lo_t = None
    if lo is not None:
        lo_t = torch.zeros(m, n // 2, dtype=torch.bfloat16 if lo == "bf16" else torch.float8_e4m3fn, device="cuda")
    int8.linear(q.cuda(), s.cuda(), _weight(wq, ws), out, epilogue="swiglu", lo=lo_t)
    got = out.double()
    assert g.abs().max() < 80   # where the bound on the fast functions holds
    fast = 2.0 ** -17 + g.abs().max().item() * 2.0 ** -22
    tol = (2.0 ** -8 + fast) * ref.abs()
    assert ((got - ref).abs() <= tol).all()
    if lo == "bf16":
        got = got + lo_t.double()
        tol = (2.0 ** -16 + 2 * fast) * ref.abs()
    elif lo == "e4m3":
        got = got + lo_t.double() / 64
        tol = (2.0 ** -12 + 2 * fast) * ref.abs() + 2.0 ** -16
    assert ((got - ref).abs() <= tol).all()


@pytest.mark.parametrize("ep", ["store", "residual", "swiglu"])
@pytest.mark.parametrize("m", [12000, 11969, 19200 + 144, 9001])
def test_ragged_token_tiles_come_out_the_same_each_time(m, ep):
    """Store tiles that lie in shared memory until their copies have read them: a last token tile
    that ends early, its next tiles left out, and other units after it."""
    from strands_decider_b200 import int8

    n, k = 640, 64
    q, s, wq, ws = _operands(m, n, k, 3)
    q, s, w = q.cuda(), s.cuda() * 0.01, _weight(wq, ws)
    cols = n // 2 if ep == "swiglu" else n
    dtype = torch.bfloat16 if ep == "swiglu" else torch.float32
    base = torch.randn(m, cols, device="cuda").to(dtype)
    want = None
    for _ in range(50):
        out = int8.linear(q, s, w, base.clone(), epilogue=ep)
        want = out if want is None else want
        assert torch.equal(out, want)
    if ep == "store":
        ref = _ref(q, s, wq, ws)
        assert ((want.double() - ref).abs() <= 4 * U * ref.abs()).all()


@pytest.mark.parametrize("m,n,k,ep", [(200, 12288, 2048, "swiglu"), (32, 2048, 6144, "residual"), (17, 640, 16, "store"),
                                      (96, 8224, 2048, "store"), (96, 12288, 2048, "swiglu"), (112, 1280, 400, "store"),
                                      (128, 2048, 16384, "residual"), (250, 2048, 8208, "store")])
def test_operand_rings_of_every_depth_come_out_the_same_each_time(m, n, k, ep):
    """Two to twelve stages, odd numbers among them, passed once, in part and many times, by launches
    that follow one another without a pause; a token alone gives the same bits."""
    from strands_decider_b200 import int8

    q, s, wq, ws = _operands(m, n, k, 5)
    q, s, w = q.cuda(), s.cuda() * 0.01, _weight(wq, ws)
    cols = n // 2 if ep == "swiglu" else n
    dtype = torch.bfloat16 if ep == "swiglu" else torch.float32
    base = torch.randn(m, cols, device="cuda").to(dtype)
    outs = [base.clone() for _ in range(20)]
    for out in outs:
        int8.linear(q, s, w, out, epilogue=ep)
    for out in outs[1:]:
        assert torch.equal(out, outs[0])
    for i in (0, m // 2, m - 1):
        one = base[i:i + 1].clone()
        int8.linear(q[i:i + 1].contiguous(), s[i:i + 1].contiguous(), w, one, epilogue=ep)
        assert torch.equal(one[0], outs[0][i])


@pytest.mark.parametrize("m", [1, 12, 40, 300])
def test_linear_extreme_codes_at_the_greatest_depth(m):
    """-128 x -128 over k = 65536 is 2^30; signs and single codes come through exactly."""
    from strands_decider_b200 import int8

    k, n = 65536, 130
    q = torch.full((m, k), -128, dtype=torch.int8)
    wq = torch.full((n, k), -128, dtype=torch.int8)
    wq[1::3] = 127
    wq[2::3] = 0
    wq[2::3, 5] = 1
    q[m // 2] = 127
    out = torch.empty(m, n, device="cuda")
    int8.linear(q.cuda(), torch.ones(m, device="cuda"), _weight(wq, torch.ones(n)), out)
    assert torch.equal(out.double(), _ref(q, torch.ones(m), wq, torch.ones(n)).float().double())


@pytest.mark.parametrize("m,k,n,nv", [(3, 256, 700, 443), (30, 2048, 700, 443), (140, 272, 700, 443),
                                      (700, 128, 700, 443), (3001, 144, 4400, 3999), (3001, 144, 4400, 3998),
                                      (3001, 144, 4400, 3996)])
@pytest.mark.parametrize("col", [5, 8])   # where the outputs start: no 16-byte rows, and such rows
def test_linear_strides_partial_outputs_and_neighbours(m, k, n, nv, col):
    """A strided q, fewer outputs than weight rows, a wider out: nothing else is touched."""
    from strands_decider_b200 import int8

    q, s, wq, ws = _operands(m, n, k, 5)
    big = torch.full((m, k + 48), 77, dtype=torch.int8).cuda()
    big[:, 16:16 + k] = q.cuda()
    w = _weight(wq, ws)
    ref = _ref(q, s, wq, ws)[:, :nv]
    wide = nv + 57 + nv % 2 if col == 5 else (nv + 63) // 8 * 8
    for ep in ("store", "residual"):
        out = torch.full((m + 2, wide), 3.0).cuda()
        int8.linear(big[:, 16:16 + k], s.cuda(), w, out[1:-1, col:col + nv], epilogue=ep, n_valid=nv)
        want = ref if ep == "store" else ref + 3
        assert ((out[1:-1, col:col + nv].double() - want).abs() <= 4 * U * ref.abs() + 1.01 * U * want.abs()).all()
        assert (out[0] == 3).all() and (out[-1] == 3).all()
        assert (out[:, :col] == 3).all() and (out[:, col + nv:] == 3).all()
    nv = nv // 128 * 128
    h = torch.full((m + 2, wide), 2.0, dtype=torch.bfloat16).cuda()
    s8 = torch.full((m,), 4.0 / (74.0 ** 2 * k ** 0.5)).cuda()
    int8.linear(big[:, 16:16 + k], s8, _weight(wq, torch.ones(n)), h[1:-1, col:col + nv // 2], epilogue="swiglu",
                n_valid=nv)
    y = _ref(q, s8, wq, torch.ones(n))[:, :nv].reshape(m, nv // 128, 2, 64)
    ref = (torch.nn.functional.silu(y[:, :, 0]) * y[:, :, 1]).reshape(m, nv // 2)
    end = col + nv // 2
    assert ((h[1:-1, col:end].double() - ref).abs() <= (2.0 ** -8 + 2.0 ** -16) * ref.abs()).all()
    assert (h[0] == 2).all() and (h[-1] == 2).all() and (h[:, :col] == 2).all() and (h[:, end:] == 2).all()


@pytest.mark.parametrize("ep", ["store", "residual", "swiglu"])
@pytest.mark.parametrize("m,n,k", [(1200, 768, 1040), (4800, 2048, 272)])
def test_a_row_does_not_depend_on_its_batch(m, n, k, ep):
    """Bit for bit the same row alone, in small, middle and large batches, and run to run."""
    from strands_decider_b200 import int8

    q, s, wq, ws = _operands(m, n, k, 11)
    s = s * 0.01
    w = _weight(wq, ws)
    q, s = q.cuda(), s.cuda()

    base = torch.randn(m, n, device="cuda")

    def run(a, b):
        if ep == "swiglu":
            out = torch.empty(b - a, n // 2, device="cuda", dtype=torch.bfloat16)
        else:
            out = base[a:b].clone()
        return int8.linear(q[a:b], s[a:b], w, out, epilogue=ep)

    whole = run(0, m)
    assert torch.equal(whole, run(0, m))
    for a, b in ((0, 1), (5, 12), (3, 19), (100, 133), (0, 64), (200, 300), (0, 129), (400, 700)):
        assert torch.equal(run(a, b), whole[a:b]), (a, b)


def test_a_row_that_is_not_finite_stays_alone():
    from strands_decider_b200 import int8

    for m in (5, 50, 500):
        x = torch.randn(m, 256)
        x[3, 7] = float("inf")
        q, s = int8.quantize_act(x.cuda())
        _, _, wq, ws = _operands(1, 320, 256, 2)
        out = torch.empty(m, 320, device="cuda")
        int8.linear(q, s, _weight(wq, ws), out)
        bad = torch.isnan(out)
        assert bad[3].all() and not bad[:3].any() and not bad[4:].any()
        resid = torch.zeros(m, 320, device="cuda")
        int8.linear(q, s, _weight(wq, ws), resid, epilogue="residual")
        assert torch.isnan(resid[3]).all() and not torch.isnan(resid[4:]).any()


@pytest.mark.parametrize("m,n", [(4, 256), (40, 256), (300, 256), (12000, 512)])
def test_offsets_past_32_bits(m, n):
    """Codes and outputs whose last rows start past 2^31 elements, on every kernel."""
    from strands_decider_b200 import int8

    q, s, wq, ws = _operands(m, n, 64, m)
    w, ref = _weight(wq, ws), _ref(q, s, wq, ws)
    ld = (1 << 31) // (m - 1) // 16 * 16 + 64
    big = torch.empty((m - 1) * ld + 64, dtype=torch.int8, device="cuda").as_strided((m, 64), (ld, 1))
    big.copy_(q)
    ldo = ld + 512
    out = torch.empty((m - 1) * ldo + n, device="cuda").as_strided((m, n), (ldo, 1))
    int8.linear(big, s.cuda(), w, out)
    assert ((out.double() - ref).abs() <= 4 * U * ref.abs()).all()
    out.fill_(1.0)
    int8.linear(big, s.cuda(), w, out, epilogue="residual")
    assert ((out.double() - ref - 1).abs() <= 4 * U * ref.abs() + 1.01 * U * (ref + 1).abs()).all()


@pytest.mark.parametrize("rows", [3, 70])
def test_row_offsets_past_32_bits(rows):
    from strands_decider_b200 import int8

    k = 272
    ld = (1 << 31) // (rows - 1) // 16 * 16 + 288
    x = torch.empty((rows - 1) * ld + k, dtype=torch.bfloat16, device="cuda").as_strided((rows, k), (ld, 1))
    x.copy_(torch.randn(rows, k))
    q = torch.empty((rows - 1) * ld + k, dtype=torch.int8, device="cuda").as_strided((rows, k), (ld, 1))
    _, s = int8.quantize_act(x, out=q)
    _same_codes(q, s, *Q.quantize_int8_rows(x.float().cpu().numpy()))
    del q
    t = torch.empty((rows - 1) * ld + k, device="cuda").as_strided((rows, k), (ld, 1))
    t.copy_(torch.randn(rows, k))
    w = torch.randn(k).cuda()
    want = Q.rmsnorm_int8(t.cpu().numpy(), w.cpu().numpy(), 1e-6, x.float().cpu().numpy())
    q, s = int8.rmsnorm(t, w, 1e-6, delta=x, resid_out=t)
    _same_codes(q, s, *want[:2])
    assert np.array_equal(t.cpu().numpy(), want[2])


# ----------------------------------------------------------------------------- together, as they are used


def _mlp(x, delta, p, bufs):
    """The MLP half of a layer: x += delta, norm, gate / up, SwiGLU, down, back into x."""
    from strands_decider_b200 import int8

    q, s = int8.rmsnorm(x, p["norm"], 1e-6, delta=delta, resid_out=x, out=bufs["q"], scale=bufs["s"])
    int8.linear(q, s, p["gate_up"], bufs["h"], epilogue="swiglu")
    hq, hs = int8.quantize_act(bufs["h"], out=bufs["hq"], scale=bufs["hs"])
    return int8.linear(hq, hs, p["down"], x, epilogue="residual")


def _mlp_setup(m, hidden=512, inter=1088):
    from strands_decider_b200 import weights as W

    g = torch.Generator(device="cuda").manual_seed(m)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    gate, up, down = randn(inter, hidden) * 0.05, randn(inter, hidden) * 0.05, randn(hidden, inter) * 0.05
    p = {"norm": randn(hidden) * 0.1, "w": (gate, up, down),
         "gate_up": W.interleave_gate_up(W.quantize("int8", gate), W.quantize("int8", up)),
         "down": W.concat_rows([W.quantize("int8", down)])}
    n = 2 * inter
    bufs = {"q": torch.empty(m, hidden, dtype=torch.int8, device="cuda"), "s": torch.empty(m, device="cuda"),
            "h": torch.empty(m, inter, dtype=torch.bfloat16, device="cuda"),
            "hq": torch.empty(m, inter, dtype=torch.int8, device="cuda"), "hs": torch.empty(m, device="cuda")}
    assert p["gate_up"].n >= n
    p["gate_up"] = W.PackedWeight("int8", n, hidden, p["gate_up"].data[:n].contiguous(),
                                  row_scale=p["gate_up"].row_scale[:n].contiguous())
    return p, bufs, randn(m, hidden), randn(m, hidden)


@pytest.mark.parametrize("m", [1, 16, 77, 1000])
def test_mlp_of_the_operators(m):
    """Against the same chain in 64 bits on the device's own codes, step by step exact; and near
    the unquantised MLP: rounding to codes is off by amax / 127 / sqrt(12) in the mean square, and
    a row's amax is at most about 10 of its standard deviations (4 for a Gaussian row, more for
    the SwiGLU's products)."""
    from strands_decider_b200 import weights as W

    p, bufs, x, delta = _mlp_setup(m)
    t = x + delta
    got = _mlp(x.clone(), delta, p, bufs)
    q, s, _ = Q.rmsnorm_int8(x.cpu().numpy(), p["norm"].cpu().numpy(), 1e-6, delta.cpu().numpy())
    _same_codes(bufs["q"], bufs["s"], q, s)
    parts = W.packed_to_numpy(p["gate_up"])
    y = torch.from_numpy(Q.int8_product(q, s, parts["data"], parts["row_scale"])).reshape(m, -1, 2, 64)
    h = (torch.nn.functional.silu(y[:, :, 0]) * y[:, :, 1]).reshape(m, -1)
    assert ((bufs["h"].double().cpu() - h).abs() <= (2.0 ** -8 + 2.0 ** -16) * h.abs()).all()
    hq, hs = Q.quantize_int8_rows(bufs["h"].float().cpu().numpy())
    _same_codes(bufs["hq"], bufs["hs"], hq, hs)
    parts = W.packed_to_numpy(p["down"])
    ref = torch.from_numpy(Q.int8_product(hq, hs, parts["data"], parts["row_scale"]))
    want = t.double().cpu() + ref
    assert ((got.double().cpu() - want).abs() <= 4 * U * ref.abs() + 1.01 * U * want.abs()).all()
    gate, up, down = (w.double() for w in p["w"])
    v = t.double() * torch.rsqrt(t.double().square().mean(-1, keepdim=True) + 1e-6) * (1 + p["norm"].double())
    full = (torch.nn.functional.silu(v @ gate.T) * (v @ up.T)) @ down.T
    off = (got.double() - t.double() - full).norm() / full.norm()
    # six quantised operands, independent; the SiLU's slope is at most 1.1
    assert off < 6 ** 0.5 * 1.1 * 10 / 127 / 12 ** 0.5


def test_mlp_captured_replayed_and_on_two_streams():
    """A captured chain replays on new inputs; two chains on two streams do not meet."""
    sets = [_mlp_setup(m) for m in (9, 150)]
    want = [_mlp(x.clone(), d, p, b).clone() for p, b, x, d in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    xs = [x.clone() for _, _, x, _ in sets]
    for _ in range(5):
        for i, (p, b, x, d) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                xs[i].copy_(x)
                _mlp(xs[i], d, p, b)
    torch.cuda.synchronize()
    assert torch.equal(xs[0], want[0]) and torch.equal(xs[1], want[1])
    for i, (p, b, x, d) in enumerate(sets):
        buf, dd = x.clone(), d.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            _mlp(buf, dd, p, b)
        torch.cuda.synchronize()
        assert torch.equal(buf, x)       # capturing runs nothing
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(buf, want[i])
        x2, d2 = torch.randn_like(x), torch.randn_like(d)
        buf.copy_(x2)
        dd.copy_(d2)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(buf, _mlp(x2.clone(), d2, p, b))


def test_mlps_of_four_threads_on_streams_of_their_own():
    """Calls from several host threads at once, launches of every kind beside one another on the SMs."""
    import threading

    sets = [_mlp_setup(m, hidden=1024, inter=2048) for m in (7, 30, 130, 1400)]
    want = [_mlp(x.clone(), d, p, b).clone() for p, b, x, d in sets]
    torch.cuda.synchronize()
    wrong = []

    def run(i):
        try:
            p, b, x, d = sets[i]
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(40):
                    got = _mlp(x.clone(), d, p, b)
                    if not torch.equal(got, want[i]):
                        wrong.append(i)
        except Exception as e:  # noqa: BLE001 - reported below
            wrong.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong


def test_python_operators_refuse_before_launching():
    from strands_decider_b200 import _lib, int8
    from strands_decider_b200 import weights as W

    x = torch.zeros(4, 64, device="cuda")
    w = W.quantize("int8", torch.randn(128, 64, device="cuda"))
    q, s = int8.quantize_act(x)
    out = torch.zeros(4, 128, device="cuda")
    for bad in (lambda: int8.quantize_act(x.half()), lambda: int8.quantize_act(x[0]),
                lambda: int8.quantize_act(x, lo=x), lambda: int8.quantize_act(x.t()),
                lambda: int8.quantize_act(x, out=torch.empty(4, 64, device="cuda")),
                lambda: int8.quantize_act(x, scale=torch.empty(5, device="cuda")),
                lambda: int8.quantize_act(x, scale=torch.empty(4)),
                lambda: int8.rmsnorm(x, torch.zeros(32, device="cuda"), 1e-6),
                lambda: int8.rmsnorm(x, torch.zeros(64, device="cuda"), 1e-6, resid_out=x),
                lambda: int8.rmsnorm(x, torch.zeros(64, device="cuda"), 1e-6, delta=x.double()),
                lambda: int8.linear(q, s, W.quantize("int4", torch.zeros(256, 128, device="cuda")), out),
                lambda: int8.linear(q, s, w, out, epilogue="gelu"),
                lambda: int8.linear(q, s, w, out, lo=out),
                lambda: int8.linear(q, s, w, out.to(torch.bfloat16)),
                lambda: int8.linear(q, s, w, out[:, :100]),
                lambda: int8.linear(q, s[:3], w, out),
                lambda: int8.linear(x, s, w, out),
                lambda: int8.linear(q, s, w, out, epilogue="swiglu")):
        with pytest.raises(ValueError):
            bad()
    # what only a later argument shows: another device, type, stride or number of outputs
    pw = W.PackedWeight
    wide = torch.zeros(256, 64, dtype=torch.int8, device="cuda")
    act = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    buf = torch.zeros(4, 64, dtype=torch.uint8, device="cuda")
    for bad in (lambda: int8.quantize_act(act, lo=torch.zeros(4, 128, dtype=torch.bfloat16, device="cuda")[:, ::2]),
                lambda: int8.quantize_act(act, lo=torch.zeros(4, 128, dtype=torch.bfloat16, device="cuda")[:, :64]),
                lambda: int8.quantize_act(act.to_sparse()), lambda: int8.quantize_act(act, lo=act.cpu()),
                lambda: int8.rmsnorm(x, torch.zeros(128, device="cuda")[::2], 1e-6),
                lambda: int8.rmsnorm(x, torch.zeros(64), 1e-6),
                lambda: int8.rmsnorm(x, torch.zeros(64, device="cuda"), 1e-6, delta=x[:3]),
                lambda: int8.rmsnorm(x, torch.zeros(64, device="cuda"), 1e-6, delta=x, resid_out=x.to(torch.bfloat16)),
                lambda: int8.linear(q, s, pw("int8", 128, 64, wide[::2], row_scale=w.row_scale), out),
                lambda: int8.linear(q, s, pw("int8", 128, 64, w.data.cpu(), row_scale=w.row_scale), out),
                lambda: int8.linear(q, s, pw("int8", 128, 64, w.data.float(), row_scale=w.row_scale), out),
                lambda: int8.linear(q, s, pw("int8", 128, 64, w.data, row_scale=w.row_scale[:64]), out),
                lambda: int8.linear(q, s, pw("int8", 128, 64, w.data), out),
                lambda: int8.linear(q, s, w, out, n_valid=1 << 40), lambda: int8.linear(q, s, w, out, n_valid=64),
                lambda: int8.linear(q, s, w, act, epilogue="swiglu", lo=act),
                lambda: int8.linear(q, s, w, act, epilogue="swiglu", lo=act.float()),
                lambda: int8.linear(q, s, w, act, epilogue="swiglu", lo=buf.cpu())):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: int8.linear(q, s, w, out, n_valid=1.5), lambda: int8.rmsnorm(x, x[0], None),
                lambda: int8.linear(q, s, w, None)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: int8.quantize_act(x[:, :40]), lambda: int8.quantize_act(x[:0]),
                lambda: int8.rmsnorm(x, torch.zeros(64, device="cuda"), -1.0),
                lambda: int8.linear(q[:, :48], s, w, out)):
        with pytest.raises(_lib.B200Error):
            bad()
    assert (out == 0).all()
