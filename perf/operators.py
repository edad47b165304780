"""Workloads of the operators a mixture-of-experts or dense transformer block needs around the
dynamically quantized Linear: the product with bias, activation and residual in its epilogue, the
router, the products grouped by expert, and the weighted sum of the experts' results.

``listed()`` and ``draw()`` give cases, ``prepare()`` makes a case's inputs on the GPU, ``run()``
is one call of the operator: the framework's (``own`` true) or the same arithmetic in elementary
torch operations.  ``exact()`` gives the operator's definition in 64 bits.

The quantization grid is part of the operators' definition: one scale per row,
``s = max(max|x| / 127.5, 1e-8)``, codes ``clamp(rint(x * (1 / s)), -128, 127)``, every step one
IEEE fp32 operation.  Gate and up projections are interleaved in blocks of eight rows.
"""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


# ---- cases ---------------------------------------------------------------------------------
def listed():
    return [
        # router of one decoding step: 16 sequences, 64 experts, latency counts
        {"name": "route_decode", "op": "route", "tokens": 16, "experts": 64, "top_k": 4, "type": "bf16",
         "renormalize": True, "padding": 0.0},
        # router of a padded prompt batch (a quarter of the rows are masked: all logits -inf)
        {"name": "route_prompt", "op": "route", "tokens": 16384, "experts": 128, "top_k": 8, "type": "fp32",
         "renormalize": False, "padding": 0.25},
        # down projection of the decode MLP 4096 <-> 14336 at batch 1, residual stream added
        {"name": "linear_decode_down", "op": "linear", "rows": 1, "inner": 14336, "cols": 4096, "type": "bf16",
         "activation": None, "bias": False, "residual": True},
        # gate and up projections of the same MLP for 16 sequences
        {"name": "linear_decode_swiglu", "op": "linear", "rows": 16, "inner": 4096, "cols": 28672, "type": "bf16",
         "activation": "swiglu", "bias": False, "residual": False},
        # first feed-forward layer of the small encoder (32 x 256 tokens, 512 -> 2048, GELU), fp32
        {"name": "linear_encoder_gelu", "op": "linear", "rows": 8192, "inner": 512, "cols": 2048, "type": "fp32",
         "activation": "gelu", "bias": True, "residual": False},
        # nothing a multiple of anything
        {"name": "linear_odd", "op": "linear", "rows": 333, "inner": 1003, "cols": 1235, "type": "fp16",
         "activation": "gelu_tanh", "bias": True, "residual": True},
        # prefill-sized product, contraction over the wide side, residual stream added
        {"name": "linear_prefill_down", "op": "linear", "rows": 16384, "inner": 28672, "cols": 8192, "type": "bf16",
         "activation": None, "bias": False, "residual": True},
        # one decoding step of 8 sequences over 32 experts: most experts see no or one row
        {"name": "experts_decode_swiglu", "op": "experts", "tokens": 8, "experts": 32, "top_k": 4, "inner": 4096,
         "cols": 4096, "type": "bf16", "activation": "swiglu", "bias": False, "sorted_rows": False, "skew": 0.3,
         "padding": 0.0},
        # down projection of a middle-sized batch, many small experts, rows already in expert order
        {"name": "experts_batch_down", "op": "experts", "tokens": 1000, "experts": 64, "top_k": 6, "inner": 1408,
         "cols": 2048, "type": "bf16", "activation": None, "bias": True, "sorted_rows": True, "skew": 0.7,
         "padding": 0.1},
        # gate and up projections of a prompt over 16 large experts
        {"name": "experts_prompt_swiglu", "op": "experts", "tokens": 8192, "experts": 16, "top_k": 2, "inner": 4096,
         "cols": 28672, "type": "bf16", "activation": "swiglu", "bias": False, "sorted_rows": False, "skew": 0.7,
         "padding": 0.0},
        # results of a decoding step brought together
        {"name": "combine_decode", "op": "combine", "tokens": 16, "experts": 64, "top_k": 4, "cols": 4096, "type": "bf16",
         "residual": True, "padding": 0.0},
        # results of a prompt brought together
        {"name": "combine_prompt", "op": "combine", "tokens": 16384, "experts": 128, "top_k": 8, "cols": 4096,
         "type": "bf16", "residual": True, "padding": 0.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["route", "linear", "linear", "experts", "experts", "combine"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    padding = rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.6), 3)])
    if kind == "route":
        experts = _log(rng, 2, 256)
        return {"op": "route", "tokens": _log(rng, 1, 16384), "experts": experts,
                "top_k": rng.randint(1, min(8, experts)), "type": dtype, "renormalize": rng.random() < 0.5,
                "padding": padding}
    if kind == "combine":
        experts = _log(rng, 4, 128)
        return {"op": "combine", "tokens": _log(rng, 1, 16384), "experts": experts,
                "top_k": rng.randint(1, min(8, experts)), "cols": _log(rng, 64, 4096), "type": dtype,
                "residual": rng.random() < 0.5, "padding": padding}
    activation = rng.choice([None, "relu", "gelu", "gelu_tanh", "silu", "swiglu"])
    inner, cols = _log(rng, 64, 16384), _log(rng, 64, 16384)
    if activation == "swiglu":
        cols = max(16, cols // 16 * 16)
    if kind == "linear":
        return {"op": "linear", "rows": _log(rng, 1, 8192), "inner": inner, "cols": cols, "type": dtype,
                "activation": activation, "bias": rng.random() < 0.5, "residual": rng.random() < 0.5}
    experts = _log(rng, 2, 128)
    while experts * inner * cols > 16 * 28672 * 4096:  # the largest listed set of weights
        experts = max(2, experts // 2)
        if experts == 2:
            break
    return {"op": "experts", "tokens": _log(rng, 1, 4096), "experts": experts, "top_k": rng.randint(1, min(6, experts)),
            "inner": inner, "cols": cols, "type": dtype, "activation": activation, "bias": rng.random() < 0.5,
            "sorted_rows": rng.random() < 0.5, "skew": round(rng.uniform(0.0, 1.0), 2), "padding": padding}


# ---- inputs --------------------------------------------------------------------------------
def _weights(gen, shape):
    """int8 codes and scales of normally distributed float weights (one scale per output row)."""
    codes = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat = codes.view(-1, shape[-1])
    step = max(1, (1 << 26) // shape[-1])  # in pieces: the float copy of a large set of experts is not kept
    for i in range(0, flat.shape[0], step):
        part = flat[i:i + step]
        part.copy_(torch.randn(part.shape, device="cuda", generator=gen).mul_(30.0).round_().clamp_(-128, 127))
    scale = (0.02 / 30.0) * (0.75 + 0.5 * torch.rand(shape[:-1], device="cuda", generator=gen))
    return codes, scale


def _kept(codes):
    """The codes as a program keeps them: with the framework, once, in rows on 16-byte boundaries."""
    if not own:
        return codes
    from lucid_b200.nn.quantized.dynamic import functional as F

    return F.pack_weight(codes)


def _activations(gen, shape, dtype):
    """Normal values whose rows differ in size, with a few channels far above the rest."""
    x = torch.randn(shape, device="cuda", generator=gen)
    x *= torch.exp(0.5 * torch.randn((shape[0], 1), device="cuda", generator=gen))
    loud = torch.rand((1, shape[1]), device="cuda", generator=gen) < 0.002
    return torch.where(loud, 12.0 * x, x).to(dtype)


def _logits(gen, case):
    tokens, experts = case["tokens"], case["experts"]
    logits = torch.randn((tokens, experts), device="cuda", generator=gen)
    logits += case.get("skew", 0.5) * torch.randn((1, experts), device="cuda", generator=gen)
    logits[tokens - int(tokens * case["padding"]):] = -math.inf  # the padded end of the batch goes to no expert
    return logits


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = _TYPES[case["type"]]
    state = {"case": case}
    if case["op"] == "route":
        state["logits"] = _logits(gen, case).to(dtype)
        return state
    if case["op"] == "linear":
        m, n, k = case["rows"], case["cols"], case["inner"]
        state["x"] = _activations(gen, (m, k), dtype)
        state["weight"], state["scale"] = _weights(gen, (n, k))
        state["weight"] = _kept(state["weight"])
        state["bias"] = 0.1 * torch.randn(n, device="cuda", generator=gen) if case["bias"] else None
        out = n // 2 if case["activation"] == "swiglu" else n
        state["residual"] = torch.randn((m, out), device="cuda", generator=gen).to(dtype) if case["residual"] else None
        return state
    state["route"] = _route(_logits(gen, case), case["top_k"], True)
    if own:  # the operators take a router's results from wherever they come
        from lucid_b200.nn.quantized.dynamic import functional as F

        state["routing"] = F.ExpertRouting(*state["route"])
    rows = case["tokens"] * case["top_k"]
    if case["op"] == "combine":
        state["y"] = torch.randn((rows, case["cols"]), device="cuda", generator=gen).to(dtype)
        state["residual"] = (torch.randn((case["tokens"], case["cols"]), device="cuda", generator=gen).to(dtype)
                             if case["residual"] else None)
        return state
    n, k, e = case["cols"], case["inner"], case["experts"]
    state["x"] = _activations(gen, (rows if case["sorted_rows"] else case["tokens"], k), dtype)
    state["weight"], state["scale"] = _weights(gen, (e, n, k))
    state["weight"] = _kept(state["weight"])
    state["bias"] = 0.1 * torch.randn((e, n), device="cuda", generator=gen) if case["bias"] else None
    return state


# ---- plain forms ---------------------------------------------------------------------------
def _codes(x):
    x = x.float()
    largest = x.abs().amax(-1, keepdim=True)
    s = (largest / torch.full_like(largest, 127.5)).clamp_min(1e-8)  # (a Python divisor would become a multiplication)
    return (x * (1.0 / s)).round_().clamp_(-128, 127), s


def _activate(y, name):
    if name is None:
        return y
    if name == "relu":
        return torch.clamp_min(y, 0.0)
    if name == "gelu":
        return 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    if name == "silu":
        return y / (1.0 + torch.exp(-y))
    g, u = y.unflatten(-1, (-1, 2, 8)).unbind(-2)  # swiglu: eight gate columns, their eight up columns, and so on
    return (g / (1.0 + torch.exp(-g)) * u).flatten(-2)


def _product(q, s, weight, scale, bias, activation):
    y = (q @ weight.float().t()) * s * scale  # sums of integers: exact in 32 bits below 2^24
    if bias is not None:
        y = y + bias
    return _activate(y, activation)


def _route(logits, top_k, renormalize):
    """(weights, experts, offsets, positions); an expert of -1 and a position of -1 for what is not routed."""
    tokens, count = logits.shape
    values, experts = torch.sort(logits.float(), dim=-1, descending=True, stable=True)  # equal logits: lowest index
    p = torch.exp(values - values[:, :1])
    values, experts = values[:, :top_k], experts[:, :top_k]
    total = p[:, :top_k].sum(-1, keepdim=True) if renormalize else p.sum(-1, keepdim=True)
    none = values == -math.inf
    weights = torch.where(none, 0.0, p[:, :top_k] / total)
    experts = torch.where(none, -1, experts).int()
    flat = experts.reshape(-1)
    order = torch.sort(torch.where(flat < 0, count, flat), stable=True).indices
    positions = torch.empty_like(flat)
    positions[order] = torch.arange(flat.numel(), dtype=torch.int32, device=flat.device)
    positions = torch.where(flat < 0, -1, positions).view(tokens, top_k)
    per = (flat[:, None] == torch.arange(count, device=flat.device)).sum(0)
    offsets = torch.cat([per.new_zeros(1), per.cumsum(0)]).int()
    return weights, experts, offsets, positions


def _source_rows(positions, rows):
    """Token of every row in expert order."""
    flat = positions.reshape(-1).long()
    slots = torch.arange(flat.numel(), device=flat.device)[flat >= 0]
    source = torch.zeros(rows, dtype=torch.long, device=flat.device)
    source[flat[flat >= 0]] = slots // positions.shape[1]
    return source


def _experts(state, case):
    _, _, offsets, positions = state["route"]
    q, s = _codes(state["x"])
    rows = case["tokens"] * case["top_k"]
    if not case["sorted_rows"]:
        source = _source_rows(positions, rows)
        q, s = q[source], s[source]
    out = case["cols"] // 2 if case["activation"] == "swiglu" else case["cols"]
    y = torch.zeros((rows, out), dtype=state["x"].dtype, device="cuda")  # rows behind the last expert's are zero
    ends = offsets.tolist()
    for e in range(case["experts"]):
        a, b = ends[e], ends[e + 1]
        if a < b:
            y[a:b] = _product(q[a:b], s[a:b], state["weight"][e], state["scale"][e],
                              None if state["bias"] is None else state["bias"][e], case["activation"])
    return y


def _combine(state):
    weights, _, _, positions = state["route"]
    picked = state["y"][positions.clamp_min(0).long()].float()
    out = torch.where(positions[..., None] < 0, 0.0, picked * weights[..., None]).sum(1)
    if state["residual"] is not None:
        out = out + state["residual"].float()
    return out.to(state["y"].dtype)


def run(state):
    case = state["case"]
    if own:
        from lucid_b200.nn.quantized.dynamic import functional as F

        if case["op"] == "route":
            r = F.route_experts(state["logits"], case["top_k"], renormalize=case["renormalize"])
            return r.weights, r.experts, r.offsets, r.positions
        if case["op"] == "linear":
            return F.linear(state["x"], state["weight"], state["scale"], state["bias"], activation=case["activation"],
                            residual=state["residual"])
        if case["op"] == "experts":
            return F.expert_linear(state["x"], state["weight"], state["scale"], state["routing"], state["bias"],
                                   activation=case["activation"], sorted_rows=case["sorted_rows"])
        return F.combine_experts(state["y"], state["routing"], residual=state["residual"])
    if case["op"] == "route":
        return _route(state["logits"], case["top_k"], case["renormalize"])
    if case["op"] == "linear":
        q, s = _codes(state["x"])
        y = _product(q, s, state["weight"], state["scale"], state["bias"], case["activation"])
        if state["residual"] is not None:
            y = y + state["residual"].float()
        return y.to(state["x"].dtype)
    if case["op"] == "experts":
        return _experts(state, case)
    return _combine(state)


# ---- what a pass cannot do without ---------------------------------------------------------
def work(case):
    size = _SIZE[case["type"]]
    if case["op"] == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        return {"bytes": t * e * size + 12 * t * k + 4 * (e + 1), "flops": 4 * t * e}
    if case["op"] == "combine":
        t, k, n = case["tokens"], case["top_k"], case["cols"]
        routed = t - int(t * case["padding"])
        return {"bytes": routed * k * n * size + 8 * t * k + t * n * size * (2 if case["residual"] else 1),
                "flops": 2 * routed * k * n}
    k, n = case["inner"], case["cols"]
    out = n // 2 if case["activation"] == "swiglu" else n
    if case["op"] == "linear":
        m = case["rows"]
        return {"bytes": m * k * size + n * k + 4 * n * (2 if case["bias"] else 1)
                + m * out * size * (2 if case["residual"] else 1), "flops": 2 * m * n * k}
    t, e, top = case["tokens"], case["experts"], case["top_k"]
    routed = t - int(t * case["padding"])
    hit = e * (1.0 - (1.0 - top / e) ** routed)  # experts that see a row, were the choices even
    return {"bytes": int(routed * (top if case["sorted_rows"] else 1) * k * size
                         + hit * n * (k + (8 if case["bias"] else 4)) + t * top * out * size + 4 * t * top),
            "flops": 2 * routed * top * n * k}


# ---- the definition in 64 bits -------------------------------------------------------------
def _grid64(x):
    """Codes and scale of each row.  The quotients and the product of two fp32 numbers, formed in 64 bits and
    rounded to 32, are the IEEE fp32 results that the grid is defined by."""
    wide = x.double()
    largest = torch.maximum(wide.max(1).values, -wide.min(1).values)
    scale = torch.maximum((largest / 127.5).float(), torch.tensor(1e-8, device=x.device)).double()
    inverse = (1.0 / scale).float().double()
    codes = torch.round((wide * inverse[:, None]).float().double())
    return codes.clamp(-128.0, 127.0), scale


def _finish64(acc, bias, activation):
    y = acc if bias is None else acc + bias.double()
    if activation == "relu":
        return y.clamp(min=0.0)
    if activation == "gelu":
        return y * torch.special.ndtr(y)
    if activation == "gelu_tanh":
        return y * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3))
    if activation == "silu":
        return y * torch.sigmoid(y)
    if activation == "swiglu":
        at = torch.arange(y.shape[1] // 2, device=y.device)
        gate = at // 8 * 16 + at % 8
        return y[:, gate] * torch.sigmoid(y[:, gate]) * y[:, gate + 8]
    return y


def _multiply64(codes, row_scale, weight, weight_scale, bias, activation):
    wide = weight.double()
    pieces = []
    for part, s in zip(codes.split(2048), row_scale.split(2048)):
        acc = part @ wide.t()
        pieces.append(_finish64(acc * s[:, None] * weight_scale.double(), bias, activation))
    return torch.cat(pieces)


def _route64(logits, top_k, renormalize):
    x = logits.double().cpu()
    tokens, count = x.shape
    weights = torch.zeros((tokens, top_k), dtype=torch.float64)
    experts = torch.full((tokens, top_k), -1, dtype=torch.int32)
    left = x.clone()
    for j in range(top_k):
        best = left.max(1).values
        first = (left == best[:, None]).int().argmax(1)  # the lowest index of the largest
        live = best > -math.inf
        experts[live, j] = first[live].int()
        left[torch.arange(tokens)[live], first[live]] = -math.inf
    chosen = torch.gather(x, 1, experts.clamp(min=0).long())
    chosen = torch.where(experts < 0, -math.inf, chosen)
    for t in range(tokens):
        if experts[t, 0] >= 0:
            weights[t] = torch.exp(chosen[t] - torch.logsumexp(chosen[t] if renormalize else x[t], 0))
    of = [[] for _ in range(count)]
    for at, e in enumerate(experts.view(-1).tolist()):
        if e >= 0:
            of[e].append(at)
    positions = torch.full((tokens * top_k,), -1, dtype=torch.int32)
    offsets = [0]
    for list_ in of:
        for i, at in enumerate(list_):
            positions[at] = offsets[-1] + i
        offsets.append(offsets[-1] + len(list_))
    return (weights.to(logits.device), experts.to(logits.device),
            torch.tensor(offsets, dtype=torch.int32, device=logits.device), positions.view(tokens, top_k).to(logits.device))


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "route":
        return _route64(state["logits"], case["top_k"], case["renormalize"])
    if case["op"] == "linear":
        codes, scale = _grid64(state["x"])
        y = _multiply64(codes, scale, state["weight"], state["scale"], state["bias"], case["activation"])
        return y if state["residual"] is None else y + state["residual"].double()
    weights, experts, offsets, positions = state["route"]
    tokens, top_k = positions.shape
    if case["op"] == "combine":
        out = torch.zeros((tokens, case["cols"]), dtype=torch.float64, device="cuda")
        for j in range(top_k):
            live = experts[:, j] >= 0
            out[live] += weights[live, j].double()[:, None] * state["y"][positions[live, j].long()].double()
        return out if state["residual"] is None else out + state["residual"].double()
    codes, scale = _grid64(state["x"])
    width = case["cols"] // 2 if case["activation"] == "swiglu" else case["cols"]
    y = torch.zeros((tokens * top_k, width), dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        token, slot = torch.nonzero(experts == e, as_tuple=True)
        if token.numel():
            to = positions[token, slot].long()
            at = to if case["sorted_rows"] else token
            y[to] = _multiply64(codes[at], scale[at], state["weight"][e], state["scale"][e],
                                None if state["bias"] is None else state["bias"][e], case["activation"])
    return y
