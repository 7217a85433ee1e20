"""The int8 product where its kernels' loops come round: operand rings of every depth passed several
times, weights in several groups of output tiles. The products and their tolerances are those of
test_gpu_int8.py; each case first asserts that it runs what it is meant to."""

from __future__ import annotations

import pytest
import torch

from tests import launch_plans as P
from tests.test_gpu_int8 import U, _gen, _operands, _ref, _weight

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.fail("the -m gpu tests need a CUDA device")
    from strands_decider_b200 import _lib

    _lib.load()
    yield
    torch.cuda.synchronize()
    assert _lib.read_fault() == 0


def _case(m, n, k, ep):
    """Operands on the device, the outputs before the call, and the 64-bit product."""
    q, s, wq, ws = _operands(m, n, k, m + n + k)
    if ep == "swiglu":   # |g| and |u| of a few tens at most
        s = torch.full((m,), 4.0 / (74.0 ** 2 * k ** 0.5))
        ws = torch.exp(0.2 * torch.randn(n, generator=_gen(n)))
    ref = _ref(q, s, wq, ws)
    base = torch.randn(m, n, device="cuda") * ref.abs().mean().float()
    if ep == "swiglu":
        base = torch.zeros(m, n // 2, dtype=torch.bfloat16, device="cuda")
    return q.cuda(), s.cuda(), _weight(wq, ws), base, ref


def _check(out, base, ref, ep):
    if ep == "store":
        assert ((out.double() - ref).abs() <= 4 * U * ref.abs()).all()
    elif ep == "residual":
        want = base.double() + ref
        assert ((out.double() - want).abs() <= 4 * U * ref.abs() + 1.01 * U * want.abs()).all()
    else:
        y = ref.reshape(ref.shape[0], -1, 2, 64)
        g = y[:, :, 0]
        assert g.abs().max() < 80
        h = (g * torch.sigmoid(g) * y[:, :, 1]).reshape(out.shape)
        tol = (2.0 ** -8 + 2.0 ** -17 + g.abs().max().item() * 2.0 ** -22) * h.abs()
        assert ((out.double() - h).abs() <= tol).all()


@pytest.mark.parametrize("m,n,k,ep,cluster,stages", P.RINGS)
def test_operand_rings_passed_several_times(m, n, k, ep, cluster, stages):
    """Launches that follow one another without a pause give the same bits and the right product."""
    from strands_decider_b200 import _lib, int8

    p = P.int8_plan(m, n, k, ep, sms=0)
    assert (p.kernel, p.cluster, p.stages) == (_lib.KERNEL_INT8_SPLIT, cluster, stages) and p.k_blocks > stages
    q, s, w, base, ref = _case(m, n, k, ep)
    outs = [base.clone() for _ in range(12)]
    for out in outs:
        int8.linear(q, s, w, out, epilogue=ep)
    _check(outs[0], base, ref, ep)
    for out in outs[1:]:
        assert torch.equal(out, outs[0])


@pytest.mark.parametrize("m,n,k,tokens", P.GROUPS)
@pytest.mark.parametrize("ep,form", [("store", ""), ("residual", ""), ("residual", "unaligned"), ("swiglu", ""),
                                     ("swiglu", "unaligned"), ("swiglu", "low plane")])
def test_weights_in_several_groups(m, n, k, tokens, ep, form):
    """Each output tile once, in groups that are not all of one size, in every way of writing it."""
    from strands_decider_b200 import _lib, int8

    q, s, w, base, ref = _case(m, n, k, ep)
    cols = base.shape[1]
    wide = torch.full((m, cols + 9), 5.0, dtype=base.dtype, device="cuda")
    out = wide[:, 1:1 + cols].copy_(base) if form == "unaligned" else base.clone()
    lo = torch.zeros_like(base) if form == "low plane" else None
    p = P.int8_plan(m, n, k, ep, lo=64 if lo is not None else 0, sms=0, ldo=out.stride(0), out=out.data_ptr())
    tiles = -(-n // 256)
    assert p.kernel == _lib.KERNEL_INT8_PAIR and p.tile_m == tokens
    assert p.group_tiles < tiles and tiles % p.group_tiles and 2 * p.tiles > p.ctas
    int8.linear(q, s, w, out, epilogue=ep, lo=lo)
    _check(out, base, ref, ep)
    if lo is not None:
        y = ref.reshape(m, -1, 2, 64)
        h = (y[:, :, 0] * torch.sigmoid(y[:, :, 0]) * y[:, :, 1]).reshape(out.shape)
        fast = 2.0 ** -17 + y[:, :, 0].abs().max().item() * 2.0 ** -22
        assert ((out.double() + lo.double() - h).abs() <= (2.0 ** -16 + 2 * fast) * h.abs()).all()
    if form == "unaligned":
        assert (wide[:, :1] == 5).all() and (wide[:, 1 + cols:] == 5).all()
