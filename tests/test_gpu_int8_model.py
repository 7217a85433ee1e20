"""Models of int8 weights: the forward runs W8A8.

* The forward equals its operators called one after the other, bit for bit (no sum in it depends
  on an order that changes).
* It follows the CPU emulation (the oracle's torso on int8 codes of every linear's input): rounding
  differences between the two move some codes by one, so the distance of the hidden states is held
  to the distance that the codes themselves make (emulation against unquantised activations).
* Graph replays, prefix slots and appended states work as for the other formats.
"""

from __future__ import annotations

import ctypes as C
import os

import numpy as np
import pytest
import torch

from oracle import quant as Q
from oracle import synth as osynth
from oracle import torso as OT
from strands_decider_b200 import config

from tests.conftest import GOLDEN

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


def _model(spec, seed, graphs=True, slots=8, max_tokens=4096):
    from strands_decider_b200.runtime import DecisionModel
    from strands_decider_b200.weights import DeviceWeights

    w = DeviceWeights.synthetic(spec.with_format("int8"), seed=seed, latent_device="cpu", keep_logical=True)
    return DecisionModel(w, max_tokens=max_tokens, pool_slots=slots, pool_kv_tokens=max_tokens, graphs=graphs)


def _composed(m, ids, cu, max_len):
    """The residual stream of one forward from the public entry points, layer by layer."""
    from strands_decider_b200 import _lib, int8

    s, w = m.spec, m.w
    T = ids.numel()
    st = _lib.stream_ptr()
    x = torch.empty(T, s.hidden, device="cuda")
    _lib.call("b200_embed", _lib.ptr(ids), T, _lib.ptr(w.embed), s.hidden, _lib.ptr(x), st)
    seqs = _lib.Seqs(cu.numel() - 1, T, max_len, _lib.ptr(cu), None, None)
    for li, lt in enumerate(s.layer_types):
        L = w.layers[li]
        lw = w.layer_struct(li)
        q, sc = int8.rmsnorm(x, L["input_norm"], s.eps)
        if lt == config.GDN:
            n = (s.gdn_in_rows + 31) // 32 * 32
            mix = torch.empty(T, n, device="cuda")
            int8.linear(q, sc, L["mix_in"], mix, n_valid=n)
            act = torch.empty(2, T, s.value_dim, dtype=torch.bfloat16, device="cuda")
            scratch = torch.empty(_lib.load().b200_gdn_scratch_floats(s.gdn_heads, T), device="cuda")
            _lib.call("b200_gdn_mixer", C.byref(lw.gdn), C.byref(seqs), _lib.ptr(mix), n, _lib.ptr(act),
                      T * s.value_dim, None, 0, _lib.ptr(scratch), st)
        else:
            n = s.attn_qkv_rows
            mix = torch.empty(T, n, device="cuda")
            int8.linear(q, sc, L["mix_in"], mix, n_valid=n)
            act = torch.empty(2, T, s.attn_o_in, dtype=torch.bfloat16, device="cuda")
            bufs = [torch.empty(T, h, s.head_dim, dtype=torch.bfloat16, device="cuda")
                    for h in (s.attn_heads, s.attn_kv_heads, s.attn_kv_heads)]
            ap = _lib.AttnParams(s.attn_heads, s.attn_kv_heads, s.head_dim, s.rope_dim, s.max_positions, s.eps,
                                 _lib.ptr(L["q_norm"]), _lib.ptr(L["k_norm"]), _lib.ptr(m.rope_cos),
                                 _lib.ptr(m.rope_sin))
            _lib.call("b200_attention", C.byref(ap), C.byref(seqs), _lib.ptr(mix), n, *(_lib.ptr(b) for b in bufs),
                      _lib.ptr(act), T * s.attn_o_in, None, 0, st)
        q, sc = int8.quantize_act(act[0], lo=act[1])
        int8.linear(q, sc, L["mix_out"], x, epilogue="residual", n_valid=s.hidden)
        q, sc = int8.rmsnorm(x, L["post_norm"], s.eps)
        h = torch.empty(T, s.inter, dtype=torch.bfloat16, device="cuda")
        int8.linear(q, sc, L["gate_up"], h, epilogue="swiglu", n_valid=2 * s.inter)
        q, sc = int8.quantize_act(h)
        int8.linear(q, sc, L["down"], x, epilogue="residual", n_valid=s.hidden)
    return x


@pytest.mark.parametrize("spec,lens", [(config.TINY, [1]), (config.TINY, [5, 40, 1, 17]), (config.TINY, [300, 200, 7]),
                                       (config.REDUCED_1024, [96]), (config.REDUCED_1024, [512, 700])],
                         ids=["tiny-1", "tiny-63", "tiny-507", "reduced-96", "reduced-1212"])
def test_forward_is_its_operators(spec, lens):
    m = _model(spec, seed=2)
    ids = torch.randint(0, spec.vocab, (sum(lens),), generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
    cu = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32).cuda()
    m.forward(ids, cu, max_len=max(lens))
    got = m.residual(ids.numel()).clone()
    want = _composed(m, ids, cu, max(lens))
    assert torch.isfinite(got).all() and torch.equal(got, want)


class _Int8:
    """A weight whose `.T` quantises the left operand of `x @ W.T` to int8 rows."""

    def __init__(self, w):
        self.w = w

    @property
    def T(self):
        return self

    def __rmatmul__(self, x):
        q, s = Q.quantize_int8_rows(x.reshape(-1, x.shape[-1]).numpy())
        return torch.from_numpy(q.astype(np.float32) * s[:, None]).reshape(x.shape) @ self.w.T


def test_forward_follows_its_emulation():
    g = np.load(os.path.join(GOLDEN, "reduced_1024_int4.npz"))
    rows = g["ids"].astype(np.int64).tolist()
    spec = config.REDUCED_1024.with_format("int8")
    m = _model(spec, seed=0)
    flat = torch.tensor(sum(rows, []), dtype=torch.int32).cuda()
    cu = torch.tensor([0] + list(np.cumsum([len(r) for r in rows])), dtype=torch.int32).cuda()
    m.forward(flat, cu, max_len=max(map(len, rows)))
    x = m.residual(flat.numel()).cpu()
    W = osynth.device_logical_weights(m.w, seed=0)
    cfg = osynth.torso_config(spec)
    with torch.inference_mode():
        plain = [OT.forward_sequence(cfg, W, torch.tensor(r))[0][-1] for r in rows]
        for L in W["layers"]:
            for part in ("gdn", "attn", "mlp"):
                for key in ("qkv", "z", "b", "a", "out", "q", "k", "v", "o", "gate", "up", "down"):
                    if part in L and key in L[part]:
                        L[part][key] = _Int8(L[part][key])
        emul = [OT.forward_sequence(cfg, W, torch.tensor(r))[0][-1] for r in rows]
        for i in range(len(rows)):
            got = OT.rms_norm_1p(x[int(cu[i + 1]) - 1], m.w.final_norm.cpu(), 1e-6)
            noise = (emul[i] - plain[i]).norm()
            assert 0 < (got - emul[i]).norm() < noise, (i, (got - emul[i]).norm(), noise)
            assert noise < 0.3 * plain[i].norm()


def test_device_weights_are_the_cpu_quantisers():
    from strands_decider_b200.weights import packed_to_numpy

    m = _model(config.TINY, seed=3)
    got = osynth.packed_digest({k: packed_to_numpy(v) for k, v in m.w.logical.items()})
    assert got == osynth.packed_digest(dict(osynth.quantized_linears(config.TINY, 3, "int8")))


def test_graph_replay_equals_eager_launches():
    rows = [torch.randint(0, config.TINY.vocab, (n,), generator=torch.Generator().manual_seed(n)).tolist()
            for n in (16, 32, 48, 32)]
    opt = [[11, 12, 13]] * 4
    outs = []
    for graphs in (True, False):
        m = _model(config.TINY, seed=1, graphs=graphs)
        for _ in range(3):
            out = m.score_prompts(rows, opt, [3] * 4, [1] * 4, [1.0] * 4).cpu()
        outs.append(out)
    assert torch.equal(outs[0].argmax, outs[1].argmax)
    assert torch.equal(outs[0].probs, outs[1].probs)


def test_prefix_and_appended_states():
    """Cached states and full prompts differ by the codes that their rounding differences move:
    both stay as near to each other as W8A8 is to unquantised activations (0.05 of a probability
    on the reduced decider), and one state read by many questions gives each the same answer."""
    m = _model(config.TINY, seed=1)
    g = torch.Generator().manual_seed(4)
    r = lambda n: torch.randint(0, config.TINY.vocab, (n,), generator=g).tolist()  # noqa: E731
    states, chunk, qs = [r(50), r(3)], [r(20), r(33)], [r(9), r(30)]
    opt = [[11, 12, 13]] * 2
    m.prefill_states(states, [0, 1], reserve=64)
    m.append_states(chunk, [0, 1])
    m.append_states([r(1), r(1)], [0, 1])
    tail = m.score_suffixes(qs, [0, 1], opt, [3] * 2, [1] * 2, [1.0] * 2).cpu()
    assert torch.isfinite(tail.probs).all()
    m.prefill_states([states[0] + chunk[0], states[1] + chunk[1]], [0, 1])
    cached = m.score_suffixes(qs, [0, 1], opt, [3] * 2, [1] * 2, [1.0] * 2).cpu()
    full = m.score_prompts([states[i] + chunk[i] + qs[i] for i in range(2)], opt, [3] * 2, [1] * 2, [1.0] * 2).cpu()
    assert (cached.probs - full.probs).abs().max() < 0.05
    many = m.score_suffixes([qs[0]] * 4, [0] * 4, opt * 2, [3] * 4, [1] * 4, [1.0] * 4).cpu()
    assert (many.probs - many.probs[0]).abs().max() == 0


def test_layers_of_another_format_are_refused():
    from strands_decider_b200 import _lib
    from strands_decider_b200.runtime import DecisionModel
    from strands_decider_b200.weights import DeviceWeights

    a = _model(config.TINY, seed=1)
    other = DeviceWeights.synthetic(config.TINY.with_format("int4"), seed=1, latent_device="cpu")
    lw = other.layer_struct(0)
    assert _lib.load().b200_model_set_layer(a._h, 0, C.byref(lw)) == 3
    b = DecisionModel(other, max_tokens=64, pool_slots=2)
    lw = a.w.layer_struct(0)
    assert _lib.load().b200_model_set_layer(b._h, 0, C.byref(lw)) == 3
