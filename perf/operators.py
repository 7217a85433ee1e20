"""The 8-bit integer (W8A8) operators as they are measured: cases, inputs, plain forms, work.

Three operators, each named by a case's "op":

  norm    t = x + delta; RMSNorm(t) * (1 + w) as int8 codes with one fp32 scale per token
  quant   int8 codes with one fp32 scale per token of an fp32, bf16 or two-plane bf16 activation
  linear  (int8 codes x int8 weight codes) * token scale * channel scale, stored, added to a
          residual stream, or taken through the SwiGLU (weight rows in blocks of 64 gate, 64 up)

A row's codes: a = max |v|, scale = a / 127, code = rint(v * (127 / a)); a row whose scale is not
a normal number has scale 0 and codes 0, one with a value that is not finite scale NaN and codes 0.
"""

import torch

own = False

NORMAL = 2.0 ** -126   # the smallest normal fp32 number


def listed():
    return [
        # one token appended to a cached state (the latency end of the norm)
        {"name": "norm one token", "op": "norm", "rows": 1, "k": 2048, "delta": "none"},
        # one 96-token prompt, the mixer's output added in bf16
        {"name": "norm 96 tokens bf16 delta", "op": "norm", "rows": 96, "k": 2048, "delta": "bf16"},
        # a ragged batch of short prompts at a width that is no power of two, the delta in fp32
        {"name": "norm 4099 tokens fp32 delta", "op": "norm", "rows": 4099, "k": 1152, "delta": "fp32"},
        # 128 states of 512 tokens in one forward (the residual is added by the linear before it)
        {"name": "norm 65536 tokens", "op": "norm", "rows": 65536, "k": 2048, "delta": "none"},
        # the attention output of 128 requests x 3 questions of 32 tokens, as hi / lo planes
        {"name": "quant 12288 tokens planes", "op": "quant", "rows": 12288, "k": 2048, "type": "planes"},
        # one token's SwiGLU output before the down-projection
        {"name": "quant one token bf16", "op": "quant", "rows": 1, "k": 6144, "type": "bf16"},
        # the SwiGLU outputs of a whole 128-state forward
        {"name": "quant 65536 tokens bf16", "op": "quant", "rows": 65536, "k": 6144, "type": "bf16"},
        # one appended token: the gate / up projection reads 25 MB of weights for one row
        {"name": "linear one token swiglu", "op": "linear", "rows": 1, "n": 12288, "k": 2048, "ep": "swiglu"},
        # 13 appended tokens (one per live state): the down-projection into the residual stream
        {"name": "linear 13 tokens residual", "op": "linear", "rows": 13, "n": 2048, "k": 6144, "ep": "residual"},
        # one 96-token prompt through the GDN in-projection (q, k, v, z and the two gate columns per head)
        {"name": "linear 96 tokens store", "op": "linear", "rows": 96, "n": 8224, "k": 2048, "ep": "store"},
        # a ragged batch of questions through the attention output projection
        {"name": "linear 1021 tokens residual", "op": "linear", "rows": 1021, "n": 2048, "k": 2048, "ep": "residual"},
        # the gate / up projection of 128 states of 512 tokens: the largest product of a step
        {"name": "linear 65536 tokens swiglu", "op": "linear", "rows": 65536, "n": 12288, "k": 2048, "ep": "swiglu"},
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    """Another case of the listed ranges: rows 1 .. 65536, depths 128 .. 8192 in steps of 16 (the
    alignment of an int8 row), outputs 64 .. 16384 (any number; in steps of 128 for the SwiGLU)."""
    op = rng.choice(["norm", "quant", "linear", "linear"])
    rows = _log_int(rng, 1, 65536)
    k = 16 * _log_int(rng, 8, 512)
    if op == "norm":
        rows = max(1, min(rows, 65536 * 2048 // k))
        return {"op": op, "rows": rows, "k": k, "delta": rng.choice(["none", "bf16", "fp32"])}
    if op == "quant":
        kind = rng.choice(["fp32", "bf16", "planes"])
        rows = max(1, min(rows, 65536 * 6144 // (k * (1 if kind == "bf16" else 2))))
        return {"op": op, "rows": rows, "k": k, "type": kind}
    ep = rng.choice(["store", "residual", "swiglu"])
    n = 128 * _log_int(rng, 1, 128) if ep == "swiglu" else _log_int(rng, 64, 16384)
    # no more products, and no more output bytes, than the largest listed case
    width = {"store": 4, "residual": 8, "swiglu": 1}[ep]
    rows = max(1, min(rows, 65536 * 12288 * 2048 // (n * k), 65536 * 12288 // (n * width)))
    return {"op": op, "rows": rows, "n": n, "k": k, "ep": ep}


def _codes(x):
    """Int8 codes and scales of a rows x k fp32 tensor of ordinary values (for making inputs)."""
    a = x.abs().amax(-1, keepdim=True).clamp_min(1e-20)
    return torch.round(x * (127.0 / a)).to(torch.int8), (a[:, 0] / 127.0).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    rows, k = case["rows"], case["k"]
    s = {"op": case["op"], "rows": rows, "k": k}
    if case["op"] == "norm":
        # a residual stream: unit-scale features with a few large channels, rows of varied size
        s["x"] = randn(rows, k).mul_(1.0 + 6.0 * (torch.rand(k, device="cuda", generator=g) > 0.98))
        s["x"].mul_(torch.exp(randn(rows, 1)))
        s["delta"] = None
        if case["delta"] != "none":
            s["delta"] = randn(rows, k).to(torch.bfloat16 if case["delta"] == "bf16" else torch.float32)
        s["w"] = randn(k).mul_(0.1)
        s["eps"] = 2.0 ** -20   # a single-precision number, so that every form adds the same one
        s["q"] = torch.empty(rows, k, dtype=torch.int8, device="cuda")
        s["scale"] = torch.empty(rows, device="cuda")
        s["sum"] = torch.empty(rows, k, device="cuda") if s["delta"] is not None else None
        return s
    if case["op"] == "quant":
        x = randn(rows, k).mul_(torch.exp(randn(rows, 1)))
        x.mul_(torch.sigmoid(randn(1, k).mul_(2.0)))
        s["lo"] = None
        if case["type"] == "planes":
            planes = torch.empty(2, rows, k, dtype=torch.bfloat16, device="cuda")
            planes[0].copy_(x)
            planes[1].copy_(x - planes[0].float())
            s["x"], s["lo"] = planes[0], planes[1]
        else:
            s["x"] = x.to(torch.bfloat16) if case["type"] == "bf16" else x
        s["q"] = torch.empty(rows, k, dtype=torch.int8, device="cuda")
        s["scale"] = torch.empty(rows, device="cuda")
        return s
    n = case["n"]
    s["n"], s["ep"] = n, case["ep"]
    s["q"], s["scale"] = _codes(randn(rows, k))
    s["wq"], s["w_scale"] = _codes(randn(n, k).mul_(0.02))
    if case["ep"] == "swiglu":
        s["out"] = torch.empty(rows, n // 2, dtype=torch.bfloat16, device="cuda")
    else:
        s["out"] = randn(rows, n)
    return s


def _row_codes(v):
    """The codes of fp32 rows in single fp32 roundings: tensors divide tensors, since torch turns a
    division by or of a Python number into a product with a reciprocal."""
    a = v.abs().amax(-1)
    finite = torch.isfinite(v).all(-1)
    c127 = torch.full_like(a, 127.0)
    scale = a / c127
    live = finite & (scale >= NORMAL)
    inv = torch.where(live, c127 / a, torch.zeros_like(a))
    v = torch.where(live[:, None], v, torch.zeros_like(v))
    q = torch.round(v * inv[:, None]).to(torch.int8)
    scale = torch.where(live, scale, torch.zeros_like(scale))
    return q, torch.where(finite, scale, torch.full_like(scale, float("nan")))


def _plain_norm(s):
    t = s["x"] if s["delta"] is None else s["x"] + s["delta"].float()
    # a code may sit next to a rounding border: the sum of squares is taken in 64 bits
    r = torch.rsqrt(t.double().square().sum(-1) / s["k"] + s["eps"]).float()
    q, scale = _row_codes((t * r[:, None]) * (1.0 + s["w"]))
    out = {"q": q, "scale": scale}
    if s["delta"] is not None:
        out["sum"] = t
    return out


def _plain_quant(s):
    v = s["x"].float()
    if s["lo"] is not None:
        v = v + s["lo"].float()
    q, scale = _row_codes(v)
    return {"q": q, "scale": scale}


def _plain_linear(s):
    y = (s["q"].float() @ s["wq"].float().t()) * s["scale"][:, None] * s["w_scale"]
    if s["ep"] == "store":
        return {"out": y}
    if s["ep"] == "residual":
        return {"out": s["out"].add_(y)}
    y = y.view(s["rows"], s["n"] // 128, 2, 64)
    gate, up = y[:, :, 0], y[:, :, 1]
    h = gate / (1.0 + torch.exp(-gate)) * up
    return {"out": h.reshape(s["rows"], s["n"] // 2).to(torch.bfloat16)}


def _own(s):
    from strands_decider_b200 import int8

    if s["op"] == "norm":
        int8.rmsnorm(s["x"], s["w"], s["eps"], delta=s["delta"], resid_out=s["sum"], out=s["q"], scale=s["scale"])
        return {"q": s["q"], "scale": s["scale"]} if s["sum"] is None else \
            {"q": s["q"], "scale": s["scale"], "sum": s["sum"]}
    if s["op"] == "quant":
        int8.quantize_act(s["x"], lo=s["lo"], out=s["q"], scale=s["scale"])
        return {"q": s["q"], "scale": s["scale"]}
    if "weight" not in s:   # the packed weight that a program keeps: these tensors, no other layout
        from strands_decider_b200.weights import PackedWeight

        s["weight"] = PackedWeight("int8", s["n"], s["k"], s["wq"], row_scale=s["w_scale"])
    int8.linear(s["q"], s["scale"], s["weight"], s["out"], epilogue=s["ep"])
    return {"out": s["out"]}


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "quant": _plain_quant, "linear": _plain_linear}[state["op"]](state)


def work(case):
    rows, k = case["rows"], case["k"]
    if case["op"] == "norm":
        d = {"none": 0, "bf16": 2, "fp32": 4}[case["delta"]]
        moved = rows * k * (4 + d + 1 + (4 if d else 0)) + 4 * k + 4 * rows
        return {"bytes": moved, "flops": 8 * rows * k}
    if case["op"] == "quant":
        width = 2 if case["type"] == "bf16" else 4
        return {"bytes": rows * k * (width + 1) + 4 * rows, "flops": 3 * rows * k}
    n = case["n"]
    out = {"store": 4, "residual": 8, "swiglu": 1}[case["ep"]]
    return {"bytes": rows * k + n * k + 4 * rows + 4 * n + rows * n * out, "flops": 2 * rows * n * k}


def exact(case, seed):
    """The definitions in 64 bits. A code is a whole number and a border case may fall either way in
    64 bits, so codes have no such value; scales, sums and products have."""
    s = prepare(case, seed)
    if case["op"] == "linear":
        m, n = s["rows"], s["n"]
        acc = torch.empty(m, n, dtype=torch.float64, device="cuda")
        for i in range(0, m, 8192):
            acc[i:i + 8192] = s["q"][i:i + 8192].double() @ s["wq"].double().T
        acc *= s["w_scale"].double()
        acc *= s["scale"].double()[:, None]
        if case["ep"] == "store":
            return {"out": acc}
        if case["ep"] == "residual":
            return {"out": acc + s["out"].double()}
        blocks = acc.reshape(m, -1, 128)
        h = torch.empty(m, n // 128, 64, dtype=torch.float64, device="cuda")
        for i in range(0, m, 8192):
            a = blocks[i:i + 8192, :, :64]
            h[i:i + 8192] = a * torch.sigmoid(a) * blocks[i:i + 8192, :, 64:]
        return {"out": h.reshape(m, n // 2)}
    if case["op"] == "quant":
        v = s["x"].double() if s["lo"] is None else s["x"].double() + s["lo"].double()
        return {"q": None, "scale": v.abs().max(dim=1).values / 127}
    t = s["x"].double()
    if s["delta"] is not None:
        t = t + s["delta"].double()
    v = t / torch.sqrt((t * t).mean(dim=1, keepdim=True) + s["eps"]) * (1 + s["w"].double())
    out = {"q": None, "scale": v.abs().max(dim=1).values / 127}
    if s["delta"] is not None:
        out["sum"] = t
    return out
