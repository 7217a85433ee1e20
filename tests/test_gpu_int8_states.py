"""Cached states of models of int8 weights: filled, grown by a chunk and by single tokens, read by
questions.

* Every such forward is its operators on the same pool, bit for bit, in its residual stream and in
  what it leaves in the pool.
* The states hold what the full prompt would: the question's hidden states follow the CPU emulation of
  the full prompt (the oracle's torso on int8 codes of every linear's input) within the distance that
  the codes themselves make, the emulation's from unquantised activations. Without the state, or
  without any one piece of it, they are at least four times as far off, which each test asserts.
"""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from oracle import synth as osynth
from oracle import torso as OT
from strands_decider_b200 import config
from tests.test_gpu_int8_model import _Int8, _model

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


class _Pool:
    """A copy of a model's cached states."""

    def __init__(self, m):
        from strands_decider_b200 import _lib

        self.t = {n: getattr(m, n).clone() for n in ("slot_len", "slot_kv", "gdn_state", "conv_hist", "k_cache", "v_cache")}
        self.struct = _lib.PrefixPool(m.pool_slots, m.kv_capacity, *(_lib.ptr(t) for t in self.t.values()))


def _composed(m, ids, cu, max_len, pool, prefix, save):
    """The residual stream of one forward from the public entry points, on `pool`."""
    from strands_decider_b200 import _lib, int8

    s, w, T = m.spec, m.w, ids.numel()
    st = _lib.stream_ptr()
    x = torch.empty(T, s.hidden, device="cuda")
    _lib.call("b200_embed", _lib.ptr(ids), T, _lib.ptr(w.embed), s.hidden, _lib.ptr(x), st)
    seqs = _lib.Seqs(cu.numel() - 1, T, max_len, _lib.ptr(cu), _lib.ptr(prefix), _lib.ptr(save))
    seen = {config.GDN: 0, config.ATTN: 0}
    for li, lt in enumerate(s.layer_types):
        L, lw, nth = w.layers[li], w.layer_struct(li), seen[lt]
        seen[lt] += 1
        q, sc = int8.rmsnorm(x, L["input_norm"], s.eps)
        n = (s.gdn_in_rows + 31) // 32 * 32 if lt == config.GDN else s.attn_qkv_rows
        mix = torch.empty(T, n, device="cuda")
        int8.linear(q, sc, L["mix_in"], mix, n_valid=n)
        k = s.value_dim if lt == config.GDN else s.attn_o_in
        act = torch.empty(2, T, k, dtype=torch.bfloat16, device="cuda")
        if lt == config.GDN:
            scratch = torch.empty(_lib.load().b200_gdn_scratch_floats(s.gdn_heads, T), device="cuda")
            _lib.call("b200_gdn_mixer", C.byref(lw.gdn), C.byref(seqs), _lib.ptr(mix), n, _lib.ptr(act), T * k,
                      C.byref(pool.struct), nth, _lib.ptr(scratch), st)
        else:
            bufs = [torch.empty(T, h, s.head_dim, dtype=torch.bfloat16, device="cuda")
                    for h in (s.attn_heads, s.attn_kv_heads, s.attn_kv_heads)]
            ap = _lib.AttnParams(s.attn_heads, s.attn_kv_heads, s.head_dim, s.rope_dim, s.max_positions, s.eps,
                                 _lib.ptr(L["q_norm"]), _lib.ptr(L["k_norm"]), _lib.ptr(m.rope_cos), _lib.ptr(m.rope_sin))
            _lib.call("b200_attention", C.byref(ap), C.byref(seqs), _lib.ptr(mix), n, *(_lib.ptr(b) for b in bufs),
                      _lib.ptr(act), T * k, C.byref(pool.struct), nth, st)
        q, sc = int8.quantize_act(act[0], lo=act[1])
        int8.linear(q, sc, L["mix_out"], x, epilogue="residual", n_valid=s.hidden)
        q, sc = int8.rmsnorm(x, L["post_norm"], s.eps)
        h = torch.empty(T, s.inter, dtype=torch.bfloat16, device="cuda")
        int8.linear(q, sc, L["gate_up"], h, epilogue="swiglu", n_valid=2 * s.inter)
        q, sc = int8.quantize_act(h)
        int8.linear(q, sc, L["down"], x, epilogue="residual", n_valid=s.hidden)
    return x


def _ids(spec, lens, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, spec.vocab, (n,), generator=g).tolist() for n in lens]


def _dev(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


@pytest.mark.parametrize("spec,states,chunks,questions", [(config.TINY, (50, 3), (20, 33), (9, 30)),
                                                          (config.TINY, (300, 64), (1, 130), (3, 200)),
                                                          (config.REDUCED_1024, (96, 160), (32, 5), (32, 40))],
                         ids=["tiny", "tiny-long", "reduced"])
def test_forwards_on_cached_states_are_their_operators(spec, states, chunks, questions):
    m = _model(spec, seed=2, graphs=False)
    m.slot_kv.copy_(_dev([0, 1000] + [0] * 6))
    steps = [(states, [-1, -1], [0, 1]), (chunks, [0, 1], [0, 1]), ((1, 1), [0, 1], [0, 1]), ((1, 1), [0, 1], [0, 1]),
             (questions + questions[:1], [0, 1, 0], [-1, -1, -1])]
    for i, (lens, prefix, save) in enumerate(steps):
        rows = _ids(spec, lens, seed=i)
        ids, cu = _dev(sum(rows, [])), _dev([sum(lens[:j]) for j in range(len(lens) + 1)])
        pool, blank = _Pool(m), _Pool(m)
        prefix, save = _dev(prefix), _dev(save)
        want = _composed(m, ids, cu, max(lens), pool, prefix, save)
        m.forward(ids, cu, prefix, save, max_len=max(lens))
        got = m.residual(ids.numel()).clone()
        assert torch.isfinite(got).all() and torch.equal(got, want), i
        for name in ("gdn_state", "conv_hist", "k_cache", "v_cache"):
            assert torch.equal(getattr(m, name), pool.t[name]), (i, name)
        if i:   # what the state holds is in the result
            alone = _composed(m, ids, cu, max(lens), blank, _dev([-1] * len(lens)), _dev([-1] * len(lens)))
            assert (alone - got).norm() > 0.1 * got.norm()
    assert m.slot_len[:2].tolist() == [a + b + 2 for a, b in zip(states, chunks)]


@pytest.fixture(scope="module")
def tiny():
    """A model, and its oracle's final hidden states with and without quantised activations."""
    m = _model(config.TINY, seed=1)
    spec = config.TINY.with_format("int8")
    cfg = osynth.torso_config(spec)
    plain, codes = osynth.device_logical_weights(m.w, seed=1), osynth.device_logical_weights(m.w, seed=1)
    for L in codes["layers"]:
        for part in ("gdn", "attn", "mlp"):
            for key in ("qkv", "z", "b", "a", "out", "q", "k", "v", "o", "gate", "up", "down"):
                if part in L and key in L[part]:
                    L[part][key] = _Int8(L[part][key])

    def hidden(W, ids, n):
        with torch.inference_mode():
            return OT.forward_sequence(cfg, W, torch.tensor(ids))[0][-n:]

    return m, lambda ids, n: hidden(codes, ids, n), lambda ids, n: hidden(plain, ids, n)


@pytest.mark.parametrize("lens", [(50, 20, 9), (3, 5, 4), (64, 1, 4), (100, 33, 9)], ids=str)
@pytest.mark.parametrize("graphs", [False, True])
def test_grown_states_hold_the_full_prompt(tiny, lens, graphs):
    m, emulated, unquantised = tiny
    m.use_graphs = graphs   # filling and growing the states
    state, chunk, question = _ids(config.TINY, lens, seed=sum(lens))
    one, two, other = _ids(config.TINY, (1, 1, 40), seed=7)
    n = len(question)
    full = state + chunk + one + two + question
    want = emulated(full, n)
    noise = (want - unquantised(full, n)).norm()
    without = [question, chunk + one + two + question, state + one + two + question, state + chunk + two + question,
               state + chunk + one + question, state + chunk + question]
    for ids in without:
        assert (emulated(ids, n) - want).norm() > 4 * noise

    def score(rows, slots=None):
        """The final-normed hidden states of the last row (launched eagerly: a graph's batch is padded)."""
        args = ([[11, 12, 13]] * len(rows), [3] * len(rows), [1] * len(rows), [1.0] * len(rows))
        m.use_graphs = False
        if slots:
            m.score_suffixes(rows, slots, *args)
        else:
            m.score_prompts(rows, *args)
        m.use_graphs = graphs
        x = m.residual(sum(map(len, rows)))[-n:].cpu()
        return OT.rms_norm_1p(x, m.w.final_norm.cpu(), m.spec.eps)

    whole = score([full])
    m.prefill_states([other, state + chunk + one + two], [2, 5])
    cached = score([other, question], [2, 5])
    m.prefill_states([other, state], [2, 5], reserve=64)
    m.append_states([chunk], [5])
    m.append_states([two, one], [2, 5])
    m.append_states([two], [5])
    grown = score([other, question], [2, 5])
    for h in (whole, cached, grown):
        assert (h - want).norm() < noise
