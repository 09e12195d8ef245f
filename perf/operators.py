"""The FFN half of a layer and its 4-bit weights, as measurable cases.

``op`` says which operator a case is a pass through:

``quantize``  a weight tensor [experts, n, k] to microscaled 4-bit floating point
              (blocks of 32 along k share a power-of-two scale) and read back
``linear``    ``rows`` activation rows times a 4-bit weight matrix [n, k]
``route``     the experts of ``rows`` tokens: logits, top-k, softmax weights
``moe``       a whole mixture-of-experts layer for ``rows`` tokens: the routing,
              the chosen experts' gated FFN, ``shared`` experts that every token
              takes behind a sigmoid gate, the weighted sum

Sizes are those of the default configuration (hidden 2048; 12352 and 9856 rows
are the input projections of a DeltaNet and of a QSA layer, 2048 x 4096 the
output projection) with generic expert counts and widths.

Routing is a choice between values that may lie close together, so its logits
are formed in 64 bits on both sides.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
ES = {"bf16": 2, "f32": 4}
BLOCK = 32
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)      # the magnitudes of E2M1, by code


# ---------------------------------------------------------------------------
# the cases


def listed():
    return [
        # an output projection converted while a model is loaded
        {"name": "quantize_output", "op": "quantize", "experts": 1, "n": 2048, "k": 4096, "dtype": "bf16"},
        # one matrix of every expert of a layer, from a float checkpoint
        {"name": "quantize_experts", "op": "quantize", "experts": 100, "n": 512, "k": 2048, "dtype": "f32"},
        # a single user's token through a DeltaNet layer's input projections
        {"name": "linear_token", "op": "linear", "rows": 1, "n": 12352, "k": 2048, "dtype": "bf16"},
        # a server's batch through an output projection, float activations
        {"name": "linear_batch", "op": "linear", "rows": 14, "n": 2048, "k": 4096, "dtype": "f32"},
        # the benchmark's prefill chunk through a DeltaNet layer's input projections
        {"name": "linear_chunk", "op": "linear", "rows": 128, "n": 12352, "k": 2048, "dtype": "bf16"},
        # a long message through a QSA layer's input projections
        {"name": "linear_prompt", "op": "linear", "rows": 2000, "n": 9856, "k": 2048, "dtype": "bf16"},
        # a single user's token: the smallest call
        {"name": "route_token", "op": "route", "rows": 1, "experts": 128, "top_k": 8, "hidden": 2048, "dtype": "bf16"},
        # a long prompt over many small experts
        {"name": "route_prompt", "op": "route", "rows": 4001, "experts": 256, "top_k": 10, "hidden": 2048,
         "dtype": "bf16"},
        # a single user's token through a layer of 128 experts
        {"name": "moe_token", "op": "moe", "rows": 1, "experts": 128, "top_k": 8, "hidden": 2048, "inter": 512,
         "shared": 1, "format": "plain", "dtype": "bf16"},
        # a server's batch of conversations, 4-bit experts
        {"name": "moe_batch", "op": "moe", "rows": 9, "experts": 128, "top_k": 8, "hidden": 2048, "inter": 512,
         "shared": 1, "format": "mx4", "dtype": "bf16"},
        # the benchmark's prefill chunk, 4-bit experts
        {"name": "moe_chunk", "op": "moe", "rows": 128, "experts": 128, "top_k": 8, "hidden": 2048, "inter": 512,
         "shared": 1, "format": "mx4", "dtype": "bf16"},
        # a long message over 64 wider experts
        {"name": "moe_prompt", "op": "moe", "rows": 2000, "experts": 64, "top_k": 8, "hidden": 2048, "inter": 768,
         "shared": 1, "format": "plain", "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "route", "moe", "moe", "moe"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "quantize":
        k = BLOCK * rng.randint(2, 128)
        n = _log(rng, 32, 12352)
        return {"op": op, "experts": _log(rng, 1, max(1, min(64, 80000000 // (n * k)))), "n": n, "k": k, "dtype": dtype}
    if op == "linear":
        k = BLOCK * rng.randint(2, 128)
        n = _log(rng, 32, min(12352, 20000000 // k))
        return {"op": op, "rows": _log(rng, 1, 2000 if dtype == "bf16" else 500), "n": n, "k": k, "dtype": dtype}
    if op == "route":
        experts = _log(rng, 8, 512)
        return {"op": op, "rows": _log(rng, 1, 2000 if experts > 256 else 4001), "experts": experts,
                "top_k": rng.randint(1, min(16, experts)), "hidden": BLOCK * rng.randint(8, 80), "dtype": dtype}
    experts = _log(rng, 8, 128)
    return {"op": op, "rows": _log(rng, 1, 1500 if dtype == "bf16" else 200), "experts": experts,
            "top_k": rng.randint(1, 8), "hidden": BLOCK * rng.randint(16, 80), "inter": BLOCK * rng.randint(4, 24),
            "shared": rng.randint(0, 2), "format": rng.choice(["plain", "mx4"]), "dtype": dtype}


def work(case):
    es = ES[case["dtype"]]
    if case["op"] == "quantize":
        n = case["experts"] * case["n"] * case["k"]
        # in, codes and scales out, the values they stand for out
        return {"bytes": n * es + n * 17 // 32 + n * es, "flops": 0}
    if case["op"] == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": n * k * 17 // 32 + (m * k + m * n) * es, "flops": 2 * m * n * k}
    t, e, kk, h = case["rows"], case["experts"], case["top_k"], case["hidden"]
    if case["op"] == "route":
        return {"bytes": (t + e) * h * es + t * kk * 8, "flops": 2 * t * e * h}
    i, s = case["inter"], case["shared"]
    # the distinct experts that uniform routing is expected to reach
    reached = e * (1.0 - (1.0 - min(kk, e) / e) ** t) + s
    per_weight = 17 / 32 if case["format"] == "mx4" else es
    return {"bytes": int(reached * 3 * h * i * per_weight + (e + 1) * h * es + 2 * t * h * es),
            "flops": 2 * t * (kk + s) * 3 * h * i + 2 * t * e * h}


# ---------------------------------------------------------------------------
# 4-bit blocks in elementary operations


def _power_of_two(e):
    """2^e for whole e of -126 to 127, exactly (exp2 is off by a rounding on some devices)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantize_plain(w):
    """(codes uint8 [..., k / 2], low nibble first; scale bytes [..., k / 32]) of w."""
    x = w.float().unflatten(-1, (-1, BLOCK))
    amax = x.abs().amax(-1)
    bits = amax.view(torch.int32)
    exponent = torch.where(bits >= 0x00800000, (bits >> 23) - 127, torch.full_like(bits, -127))
    exponent = (exponent - 2).clamp(min=-127)
    # two multiplications by powers of two: the scale's inverse may exceed a float
    half = -(exponent // 2)
    y = x * _power_of_two(half)[..., None] * _power_of_two(-exponent - half)[..., None]
    m = y.abs()
    # to nearest, ties to the even code: the border below an odd code excludes its own value
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75).to(torch.uint8) + (m > 1.25).to(torch.uint8)
            + (m >= 1.75).to(torch.uint8) + (m > 2.5).to(torch.uint8) + (m >= 3.5).to(torch.uint8)
            + (m > 5.0).to(torch.uint8))
    code = code + 8 * torch.signbit(x).to(torch.uint8)
    code = code.flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (exponent + 127).to(torch.uint8)


def _dequantize_plain(codes, scales):
    grid = torch.tensor(GRID + tuple(-v for v in GRID), device=codes.device)
    nibbles = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    values = grid[nibbles.long()].unflatten(-1, (-1, BLOCK))
    half = (scales.int() - 127) // 2
    return (values * _power_of_two(half)[..., None] * _power_of_two(scales.int() - 127 - half)[..., None]).flatten(-2)


# ---------------------------------------------------------------------------
# inputs, made from the seed alone


def _package():
    import __graft_entry__
    return __graft_entry__.load_package()


def _weights(g, shape, dtype):
    """Normal weights of a layer: rows of unit gain."""
    return (torch.randn(*shape, generator=g, device=DEV) * shape[-1] ** -0.5).to(dtype)


def _mx4_weights(g, shape):
    """Codes and scales of normal weights, an expert at a time."""
    parts = [_quantize_plain(_weights(g, shape[-2:], torch.float32)) for _ in range(math.prod(shape[:-2]))]
    codes, scales = (torch.stack(p) for p in zip(*parts))
    return codes.reshape(*shape[:-1], -1), scales.reshape(*shape[:-1], -1)


def _raw(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DT[case["dtype"]]
    if case["op"] == "quantize":
        w = _weights(g, (case["experts"], case["n"], case["k"]), torch.float32)
        # channels of different size, as trained weights have them
        w *= torch.exp(torch.randn(case["experts"], case["n"], 1, generator=g, device=DEV))
        return {"w": w.to(dt)}
    if case["op"] == "linear":
        codes, scales = _mx4_weights(g, (case["n"], case["k"]))
        return {"x": torch.randn(case["rows"], case["k"], generator=g, device=DEV).to(dt), "codes": codes,
                "scales": scales}
    h, e = case["hidden"], case["experts"]
    raw = {"x": torch.randn(case["rows"], h, generator=g, device=DEV).to(dt), "router": _weights(g, (e, h), dt)}
    if case["op"] == "route":
        return raw
    i, s = case["inter"], case["shared"]
    make = (lambda *shape: _mx4_weights(g, shape)) if case["format"] == "mx4" else (lambda *shape: _weights(g, shape, dt))
    raw["gate"], raw["up"], raw["down"] = make(e, i, h), make(e, i, h), make(e, h, i)
    if s:
        raw["shared"] = (make(s, i, h), make(s, i, h), make(s, h, i))
        raw["shared_router"] = _weights(g, (h,), dt)
    return raw


def prepare(case, seed):
    state = {"case": case, **_raw(case, seed)}
    if not own:
        return state
    # the weights as a serving program keeps them: laid out once
    qm = _package()
    lay = (lambda p: qm.Mx4Weight.from_codes(*p)) if case.get("format", "mx4") == "mx4" else (lambda p: p)
    if case["op"] == "linear":
        state["weight"] = lay((state.pop("codes"), state.pop("scales")))
    elif case["op"] == "moe":
        shared = state.pop("shared", None)
        state["weights"] = qm.MoeWeights(
            state.pop("router"), lay(state.pop("gate")), lay(state.pop("up")), lay(state.pop("down")),
            top_k=min(case["top_k"], case["experts"]),
            shared=None if shared is None else tuple(lay(p) for p in shared),
            shared_router=state.pop("shared_router", None))
    state["qm"] = qm
    return state


# ---------------------------------------------------------------------------
# one pass


def _run_own(state):
    qm, op = state["qm"], state["case"]["op"]
    if op == "quantize":
        return qm.mx4_quantize(state["w"]).dequantize(state["w"].dtype)
    if op == "linear":
        return qm.mx4_linear(state["x"], state["weight"])
    if op == "route":
        return qm.moe_route(state["x"], state["router"], state["case"]["top_k"])
    return qm.moe(state["x"], state["weights"])


def _route_plain(x, router, top_k):
    logits = x.double() @ router.double().t()
    order = logits.sort(dim=-1, descending=True, stable=True)
    ids, top = order.indices[:, :top_k], order.values[:, :top_k]
    p = torch.exp(top - top[:, :1])
    return ids.int(), (p / p.sum(-1, keepdim=True)).float()


def _ffn_plain(x, gate, up, down):
    a = x @ gate.t()
    return ((a / (1.0 + torch.exp(-a))) * (x @ up.t())) @ down.t()


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    op, dt = case["op"], DT[case["dtype"]]
    if op == "quantize":
        return _dequantize_plain(*_quantize_plain(state["w"])).to(dt)
    x = state["x"].float()
    if op == "linear":
        return (x @ _dequantize_plain(state["codes"], state["scales"]).t()).to(dt)
    top_k = min(case["top_k"], case["experts"])
    ids, weights = _route_plain(state["x"], state["router"], top_k)
    if op == "route":
        return ids, weights
    if case["format"] == "mx4":
        def expert(p, e):
            return _dequantize_plain(p[0][e], p[1][e])
    else:
        def expert(p, e):
            return p[e].float()
    y = torch.zeros_like(x)
    for e in ids.unique().tolist():
        token, slot = (ids == e).nonzero(as_tuple=True)
        out = _ffn_plain(x[token], expert(state["gate"], e), expert(state["up"], e), expert(state["down"], e))
        y[token] += weights[token, slot, None] * out
    if case["shared"]:
        scale = 1.0 / (1.0 + torch.exp(-(x @ state["shared_router"].float())))
        for s in range(case["shared"]):
            y += scale[:, None] * _ffn_plain(x, *(expert(p, s) for p in state["shared"]))
    return y.to(dt)


# ---------------------------------------------------------------------------
# the definition in 64 bits


def _two_to(n):
    return ((n.long() + 1023) << 52).view(torch.float64)


def _values(weight, e, mx4):
    """Expert e's weights as doubles; 4-bit ones from sign, exponent and mantissa bits."""
    if not mx4:
        return weight[e].double()
    codes, scales = weight[0][e], weight[1][e]
    c = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.int64, device=codes.device)
    c[..., 0::2], c[..., 1::2] = (codes % 16).long(), (codes // 16).long()
    exponent, mantissa = (c >> 1) & 3, c & 1
    magnitude = torch.where(exponent == 0, 0.5 * mantissa, (1.0 + 0.5 * mantissa) * _two_to(exponent - 1))
    s = _two_to(scales.int() - 127)
    return torch.where(c >= 8, -magnitude, magnitude).double() * s.repeat_interleave(BLOCK, -1)


def _exact_quantize(w):
    out = torch.empty(w.shape, dtype=torch.float64, device=w.device)
    grid = torch.tensor(GRID, dtype=torch.float64, device=w.device)
    for e in range(w.shape[0]):
        b = w[e].double().reshape(-1, BLOCK)
        _, exp = torch.frexp(b.abs().amax(1, keepdim=True))        # amax in [2^(exp-1), 2^exp)
        scale = _two_to((exp - 3).clamp(min=-127))
        m = b.abs() / scale
        hi = torch.searchsorted(grid, m.contiguous()).clamp(max=7)
        lo = (hi - 1).clamp(min=0)
        below, above = m - grid[lo], grid[hi] - m
        pick = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
        out[e] = (torch.copysign(grid[pick], b) * scale).reshape(w.shape[1:])
    return out


def exact(case, seed):
    raw = _raw(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_quantize(raw["w"])
    x = raw["x"].double()
    if op == "linear":
        return x @ _values((raw["codes"][None], raw["scales"][None]), 0, True).t()
    t, k = x.shape[0], min(case["top_k"], case["experts"])
    logits = x @ raw["router"].double().t()
    prob = torch.softmax(logits, -1)
    # rank of every expert: those above it, and equals of lower index
    ids = torch.empty(t, k, dtype=torch.int32, device=x.device)
    left = logits.clone()
    for j in range(k):
        best = left.amax(-1, keepdim=True)
        first = (left == best).int().argmax(-1)
        ids[:, j] = first.int()
        left.scatter_(1, first[:, None], -math.inf)
    chosen = prob.gather(1, ids.long())
    chosen = chosen / chosen.sum(-1, keepdim=True)
    if op == "route":
        return ids, chosen
    mx4 = case["format"] == "mx4"
    dense = torch.zeros_like(prob).scatter_(1, ids.long(), chosen)
    y = torch.zeros_like(x)
    for e in range(case["experts"]):
        rows = dense[:, e].nonzero()[:, 0]
        if rows.numel():
            xe = x[rows]
            hid = torch.nn.functional.silu(xe @ _values(raw["gate"], e, mx4).t()) * (xe @ _values(raw["up"], e, mx4).t())
            y.index_add_(0, rows, dense[rows, e, None] * (hid @ _values(raw["down"], e, mx4).t()))
    for s in range(case["shared"]):
        gate, up, down = (_values(p, s, mx4) for p in raw["shared"])
        open_ = torch.sigmoid(x @ raw["shared_router"].double())
        y += open_[:, None] * ((torch.nn.functional.silu(x @ gate.t()) * (x @ up.t())) @ down.t())
    return y
