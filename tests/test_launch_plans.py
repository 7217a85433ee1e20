"""Launch plans: which kernel a product takes and what its CTAs ask for (no GPU needed)."""

from __future__ import annotations

import itertools

import pytest

from strands_decider_b200 import _lib
from tests import launch_plans as P


@pytest.fixture(scope="module", autouse=True)
def lib():
    from strands_decider_b200 import build

    build.build()
    return _lib.load()


TOKENS = [*range(1, 130), 130, 160, 200, 255, 256, 257, 300, 400, 511, 600, 1021, 2000, 4099, 8192, 65536]
OUTPUTS = [1, 64, 128, 256, 640, 1024, 1536, 2048, 4096, 8224, 12288, 16384, 32768, 98304]
DEPTHS = [16, 128, 256, 384, 512, 1024, 1152, 2048, 2064, 4096, 6144, 8192, 16384, 65536]


def _cluster_ctas():
    """(shared memory, tensor memory columns, threads) of every kind of CTA that belongs to a cluster
    and takes tensor memory."""
    kinds = {}
    for m, n, k in itertools.product(TOKENS, OUTPUTS, DEPTHS):
        for ep, lo in (("store", 0), ("residual", 0), ("swiglu", 0), ("swiglu", 64)):
            if ep == "swiglu" and n % 128:
                continue
            p = P.int8_plan(m, n, k, ep, lo)
            if p.cluster > 1 and p.tmem_cols:
                kinds[(p.smem_bytes, p.tmem_cols, p.threads)] = (p.kernel, m, n, k, ep)
    for m, n, k, ep, planes in itertools.product((600, 4096, 65536), (2048, 12288), (2048, 6144),
                                                 ("store", "residual", "swiglu"), (1, 2)):
        p = P.bf16_plan(m, n, k, ep, planes)
        if p.cluster > 1:
            kinds[(p.smem_bytes, p.tmem_cols, p.threads)] = (p.kernel, m, n, k, ep, planes)
    return kinds


def test_cluster_ctas_that_fit_one_sm_find_tensor_memory_there():
    """A CTA waits for its columns while others hold them, and ends only after its cluster's others
    have theirs: two clusters that meet on two SMs without columns for both wait for ever. Whatever CTAs
    of cluster kernels an SM has room for (shared memory, 1 KB more for each; threads), the 512 columns
    serve them all."""
    kinds = _cluster_ctas()
    assert {v[0] for v in kinds.values()} == {_lib.KERNEL_BF16_PAIR, _lib.KERNEL_INT8_SPLIT, _lib.KERNEL_INT8_PAIR}
    sm_kb, sm_threads = 228, 2048
    # most columns of any set of CTAs within so many KB (rounded down: more sets fit than do) and threads
    best = {}
    for (smem, cols, threads), _ in kinds.items():
        key = ((smem + 1024) // 1024, threads)
        best[key] = max(best.get(key, 0), cols)
    most = [[0] * (sm_threads // 32 + 1) for _ in range(sm_kb + 1)]
    for kb in range(sm_kb + 1):
        for warps in range(sm_threads // 32 + 1):
            for (c_kb, threads), cols in best.items():
                if c_kb <= kb and threads // 32 <= warps:
                    most[kb][warps] = max(most[kb][warps], most[kb - c_kb][warps - threads // 32] + cols)
    assert most[sm_kb][-1] <= 512


def test_plans_refuse_what_the_linears_refuse():
    for kw in (dict(m=0), dict(k=24), dict(sms=-1), dict(n=4, n_valid=5), dict(ep="swiglu", n=192), dict(out=P.ADDRESS + 2)):
        with pytest.raises(_lib.B200Error):
            P.int8_plan(**{"m": 4, "n": 128, "k": 64, **kw})
    for kw in (dict(m=0), dict(k=64), dict(n=300), dict(sms=0)):
        with pytest.raises(_lib.B200Error):
            P.bf16_plan(**{"m": 4, "n": 256, "k": 128, **kw})
    assert P.bf16_plan(64, 256, 128).kernel == _lib.KERNEL_OTHER
    assert P.int8_plan(1, 2048, 2048).kernel == _lib.KERNEL_INT8_REG
    assert P.int8_plan(8192, 2048, 2048, sms=1).ctas == 2


def _turns(p):
    """How often the k-blocks pass the ring."""
    return p.k_blocks / p.stages


def test_the_ring_cases_pass_rings_of_every_depth():
    for m, n, k, ep, cluster, stages in P.RINGS:
        p = P.int8_plan(m, n, k, ep)
        assert (p.kernel, p.cluster, p.stages) == (_lib.KERNEL_INT8_SPLIT, cluster, stages), (m, n, k)
        assert _turns(p) > 1, (m, n, k)
    assert {c[5] for c in P.RINGS} == set(range(3, 13))
    # a barrier serves every second turn: at every depth some are used again
    assert {c[5] for c in P.RINGS if _turns(P.int8_plan(*c[:4])) > 2} == set(range(3, 13))
    p = P.int8_plan(*P.RINGS[0][:4])
    assert p.ctas > 148 and p.k_blocks == 16 and p.smem_bytes + 1024 <= 114 * 1024
    for m, n, k in itertools.product(TOKENS, OUTPUTS, DEPTHS):   # what the list leaves out is not reached
        p = P.int8_plan(m, n, k)
        if p.kernel == _lib.KERNEL_INT8_SPLIT:
            assert p.stages >= 3 or p.k_blocks <= p.stages


def test_the_group_cases_have_several_uneven_groups():
    for m, n, k, tokens in P.GROUPS:
        for ep in ("store", "residual", "swiglu"):
            p = P.int8_plan(m, n, k, ep)
            tiles_n = -(-n // 256)
            assert p.kernel == _lib.KERNEL_INT8_PAIR and p.tile_m == tokens
            assert p.group_tiles < tiles_n and tiles_n % p.group_tiles and p.tiles > 74
