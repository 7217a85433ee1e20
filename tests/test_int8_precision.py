"""What W8A8 costs in probability (CPU, on the oracle): far less than W4A4, far more than the bar.

On the reduced decider (random weights, 4 x 256 ids) int8 codes of every linear's input, one scale
per token, move an option probability by about 0.045 against the same int8 weights with unquantised
activations, every argmax unchanged; the weight-only formats' bar is 2e-3. So W8A8 is a format of
its own that a deployment asks for, not a faster path of another format."""

from __future__ import annotations

import os

import numpy as np
import torch

from oracle import head as OH
from oracle import quant as Q
from oracle import synth as osynth
from oracle import torso as OT
from strands_decider_b200 import config

from tests.conftest import GOLDEN


class _Int8:
    def __init__(self, w):
        self.w = w

    @property
    def T(self):
        return self

    def __rmatmul__(self, x):
        q, s = Q.quantize_int8_rows(x.reshape(-1, x.shape[-1]).numpy())
        return torch.from_numpy(q.astype(np.float32) * s[:, None]).reshape(x.shape) @ self.w.T


def test_int8_activations_on_the_reduced_decider():
    g = np.load(os.path.join(GOLDEN, "reduced_1024_int4.npz"))
    spec = config.REDUCED_1024.with_format("int8")
    W = osynth.logical_weights(spec, seed=0)
    cfg = osynth.torso_config(spec)

    def probs():
        with torch.inference_mode():
            pooled = torch.stack([OT.forward_sequence(cfg, W, torch.tensor(r))[0][-1]
                                  for r in g["ids"].astype(np.int64).tolist()])
            return OH.decide(pooled, W["embed"], torch.tensor(g["opt_ids"].tolist()), torch.tensor([3] * 4),
                             torch.tensor([1.0] * 4))

    plain = probs()
    for L in W["layers"]:
        for part in ("gdn", "attn", "mlp"):
            for key in ("qkv", "z", "b", "a", "out", "q", "k", "v", "o", "gate", "up", "down"):
                if part in L and key in L[part]:
                    L[part][key] = _Int8(L[part][key])
    got = probs()
    assert 2e-3 < (got - plain).abs().max() < 0.1
    assert torch.equal(got.argmax(1), plain.argmax(1))


def test_int8_rows_round_trip_within_half_a_code():
    x = torch.randn(50, 272, generator=torch.Generator().manual_seed(0)).numpy() * 3
    q, s = Q.quantize_int8_rows(x)
    assert np.abs(q).max(axis=1).tolist() == [127] * 50
    # half a code, and the roundings of scale, quotient and product (each 2^-24 of at most 127 codes)
    assert (np.abs(x.astype(np.float64) - q.astype(np.float64) * s[:, None].astype(np.float64))
            <= (0.5 + 127 * 4 * 2.0 ** -24) * s[:, None]).all()
    parts = Q.quantize("int8", x)
    assert np.array_equal(Q.dequantize("int8", parts), q.astype(np.float32) * s[:, None])
