"""Int8 linears beside linears of another format on another stream."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from tests import launch_plans as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("the -m gpu tests need a CUDA device")
    from strands_decider_b200 import _lib

    _lib.load()
    yield
    torch.cuda.synchronize()
    assert _lib.read_fault() == 0


def test_int8_clusters_beside_pairs_of_one_bf16_plane():
    """Clusters of the int8 split kernel and CTA pairs of b200_linear without a low plane, which take
    all tensor memory columns of an SM: each gives what it gives alone."""
    from strands_decider_b200 import _lib, int8
    from strands_decider_b200 import weights as W

    g = torch.Generator(device="cuda").manual_seed(0)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    calls = []
    for m, n, k, cluster in ((32, 2048, 1024, 2), (64, 2048, 4096, 4), (20, 2048, 4096, 8)):
        assert P.int8_plan(m, n, k, sms=0).cluster == cluster
        q, s = int8.quantize_act(randn(m, k))
        w = W.quantize("int8", randn(n, k))
        out = torch.empty(m, n, device="cuda")
        calls.append((out, lambda q=q, s=s, w=w, out=out: int8.linear(q, s, w, out)))
    m, n, k = 2560, 2048, 512
    assert P.bf16_plan(m, n, k, planes=1).kernel == _lib.KERNEL_BF16_PAIR
    x = randn(m, k).to(torch.bfloat16)
    pw = W.quantize("bf16", randn(n, k))
    qw, big = pw.qweight(), torch.empty(m, n, device="cuda")

    def pair():
        o = _lib.LinearOut(_lib.EP_STORE, n, _lib.ptr(big), n, 0, 0)
        _lib.call("b200_linear", _lib.ptr(x), None, m, k, k, C.byref(qw), C.byref(o), _lib.stream_ptr())

    pair()
    want = [big.clone()]
    for out, call in calls:
        call()
        want.append(out.clone())
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(50):
        with torch.cuda.stream(one):
            for _ in range(4):
                for _, call in calls:
                    call()
        with torch.cuda.stream(two):
            for _ in range(4):
                pair()
    torch.cuda.synchronize()
    for got, w in zip([big] + [out for out, _ in calls], want):
        assert torch.equal(got, w)
