"""What a model of int8 weights refuses when it is made (no GPU needed)."""

from __future__ import annotations

import ctypes as C

import pytest

from strands_decider_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    from strands_decider_b200 import build

    build.build()
    return _lib.load()


def _create(lib, **kw):
    cfg = _lib.ModelConfig()
    sizes = dict(vocab=512, hidden=256, inter=512, n_layers=2, gdn_heads=2, gdn_dk=128, gdn_dv=128, conv_width=4,
                 attn_heads=4, attn_kv_heads=2, head_dim=64, rope_dim=16, max_pos=1024, eps=1e-6,
                 weight_format=_lib.FMT["int8"])
    for name, v in {**sizes, **kw}.items():
        setattr(cfg, name, v)
    cfg.layer_kind[0], cfg.layer_kind[1] = _lib.LAYER_GDN, _lib.LAYER_ATTN
    h = C.c_void_p()
    status = lib.b200_model_create(C.byref(cfg), C.byref(h))
    if status == 0:
        assert lib.b200_model_destroy(h) == 0
    return status


def test_depths_past_the_int8_linears_are_refused_before_a_forward_starts(lib):
    """A linear's depth ends at 65536: a forward of such a model would stop after its first launches."""
    assert _create(lib) == 0
    assert _create(lib, inter=65536) == 0
    for kw in (dict(inter=65536 + 128), dict(hidden=65536 + 128), dict(gdn_heads=513), dict(attn_heads=1026, attn_kv_heads=2)):
        assert _create(lib, **kw) == 2, kw
        assert lib.b200_last_error().decode().startswith("b200_model_create: ")
        assert _create(lib, weight_format=_lib.FMT["nvfp4"], **kw) == 0   # the other formats have no such limit
