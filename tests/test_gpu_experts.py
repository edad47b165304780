"""GPU parity of the Linear with a fused epilogue, the router, the products grouped by expert and their
combination against plain implementations in 64 bits.

Tolerances (derived, not fitted).  Codes, scales, integer sums and every routing integer are exact.  A result
is act(p + b) + r with p = acc * sx * sw: converting acc and the two products round three times, the bias once,
so the pre-activation is off by at most 4 * 2^-24 (|p| + |b|); no activation has a slope above 1.13.  Evaluating
the activation itself is off by at most 2^-20 |v|: erf and exp of the library are good to 2 ulp, and the hardware
exponential's relative error (2 + 1.173 |x|) 2^-23 enters through sigma (1 - sigma), whose product with it stays
below 0.65 * 2^-23, next to a division of 2 ulp.  SwiGLU multiplies that by the up value, whose own error counts
with |silu(gate)|.  The residual adds one fp32 rounding, and the result is rounded once to its type (half a
step, eps / 2)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def F():
    from lucid_b200.nn.quantized.dynamic import functional

    return functional


@pytest.fixture(scope="module")
def ops():
    from lucid_b200._C import ops

    return ops


def f64(t):
    return t.detach().cpu().double().numpy()


# ---- plain implementations -----------------------------------------------------------------
def plain_codes(x):
    """Codes and scale of each row; every fp32 step of the grid as a 64-bit operation rounded to fp32 (exact for
    products and quotients of two fp32 numbers)."""
    x = x.detach().cpu().float().numpy()
    clean = np.where(np.isnan(x), np.float32(0), x)
    largest = np.abs(clean).max(1, initial=0.0).astype(np.float32)
    s = np.maximum((largest.astype(np.float64) / 127.5).astype(np.float32), np.float32(1e-8))
    inv = (1.0 / s.astype(np.float64)).astype(np.float32)
    with np.errstate(invalid="ignore"):
        v = (x.astype(np.float64) * inv.astype(np.float64)[:, None]).astype(np.float32)
        q = np.clip(np.rint(v), -128, 127)
    return np.where(np.isnan(q), 0.0, q).astype(np.int64), s.astype(np.float64)


_ERF = np.vectorize(math.erf, otypes=[float])


def sigmoid(v):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-v))


def plain_activation(v, name):
    if name == "relu":
        return np.maximum(v, 0.0)
    if name == "gelu":
        return 0.5 * v * (1.0 + _ERF(v * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return v * sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3))
    if name == "silu":
        return v * sigmoid(v)
    return v


def plain_product(q, s, w, sw, bias, activation, residual=None, zero=0):
    """(result, bound on the error before the final rounding)."""
    acc = (q - zero) @ w.astype(np.int64).T
    p = acc.astype(np.float64) * s[:, None] * sw[None, :]
    b = np.zeros(w.shape[0]) if bias is None else bias
    v = p + b
    before = 4 * U * (np.abs(p) + np.abs(b))
    if activation == "swiglu":
        m, half = v.shape[0], v.shape[1] // 2
        g, u = (a.reshape(m, half) for a in np.moveaxis(v.reshape(m, half // 8, 2, 8), 2, 0))
        eg, eu = (a.reshape(m, half) for a in np.moveaxis(before.reshape(m, half // 8, 2, 8), 2, 0))
        a = g * sigmoid(g)
        y = a * u
        err = np.abs(u) * (1.13 * eg + 2.0 ** -20 * np.abs(g)) + np.abs(a) * eu + U * np.abs(y)
    else:
        y = plain_activation(v, activation)
        err = before if activation in (None, "relu") else 1.13 * before + 2.0 ** -20 * np.abs(v)
    if residual is not None:
        y = y + residual
        err = err + U * np.abs(y)
    return y, err


def check(got, want, err, dtype):
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # spacing of the subnormals
    bound = err + half * (np.abs(want) + err) + tiny
    diff = np.abs(f64(got) - want)
    worst = (diff / bound).max(initial=0.0)
    assert got.dtype == dtype and worst <= 1.0, f"error of {worst:.3g} times its bound"


def plain_route(logits, top_k, renormalize):
    x = logits.detach().cpu().double().numpy()
    t, e = x.shape
    weights = np.zeros((t, top_k))
    experts = np.full((t, top_k), -1)
    for i in range(t):
        row = np.where(np.isnan(x[i]), -np.inf, x[i])
        order = [j for j in np.argsort(-row, kind="stable") if row[j] > -np.inf]
        chosen = order[:top_k]
        if not chosen:
            continue
        top = row[chosen[0]]
        with np.errstate(invalid="ignore"):
            mass = np.exp(row - top) if np.isfinite(top) else (row == top).astype(float)
        total = mass[chosen].sum() if renormalize else mass[order].sum()
        experts[i, :len(chosen)] = chosen
        weights[i, :len(chosen)] = mass[chosen] / total
    flat = experts.reshape(-1)
    positions = np.full(t * top_k, -1)
    offsets = [0]
    for j in range(e):
        at = np.flatnonzero(flat == j)
        positions[at] = offsets[-1] + np.arange(at.size)
        offsets.append(offsets[-1] + at.size)
    return weights, experts, np.array(offsets), positions.reshape(t, top_k)


def make_weight(g, *shape):
    w = torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int8)
    return w, 0.002 * (0.5 + torch.rand(shape[:-1], generator=g, device="cuda"))


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


# ---- quantizer -------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 16), (5, 100), (17, 128), (9, 1024), (4, 1003), (3, 4096), (2, 8192),
                                       (2, 16384), (1, 28672), (1, 40000)])
def test_quantize_tokens(ops, dtype, rows, cols):
    g = generator(rows * 7 + cols)
    x = (torch.randn(rows, cols, generator=g, device="cuda") * torch.rand(rows, 1, generator=g, device="cuda") * 9).to(dtype)
    q, s = ops.quantize_tokens(x)
    want_q, want_s = plain_codes(x)
    np.testing.assert_array_equal(q.cpu().numpy().astype(np.int64), want_q)
    np.testing.assert_array_equal(f64(s), want_s)


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_tokens_special_values(ops, dtype):
    x = torch.zeros(6, 64, device="cuda")
    x[1, 3] = float("nan")
    x[1, 5] = -2.0
    x[2, 7] = float("inf")
    x[2, 8] = 3.0
    x[3] = torch.linspace(-1, 1, 64, device="cuda")
    x[4, 0] = 1e-7
    x[5, 0] = -65000.0
    x = x.to(dtype)
    q, s = ops.quantize_tokens(x)
    want_q, want_s = plain_codes(x)
    np.testing.assert_array_equal(q.cpu().numpy().astype(np.int64), want_q)
    np.testing.assert_array_equal(f64(s), want_s)


def test_quantize_tokens_scatters_and_stops(ops):
    g = generator(3)
    x = torch.randn(7, 200, generator=g, device="cuda")
    perm = torch.randperm(21, generator=g, device="cuda").int().view(7, 3).contiguous()
    perm[2, 1] = -1
    perm[5, 0] = 21  # outside: skipped
    q, s = ops.quantize_tokens(x, positions=perm, out_rows=21)
    want_q, want_s = plain_codes(x)
    for t in range(7):
        for j in range(3):
            at = int(perm[t, j])
            if 0 <= at < 21:
                np.testing.assert_array_equal(q[at].cpu().numpy().astype(np.int64), want_q[t])
                assert float(s[at]) == want_s[t]
    valid = torch.tensor([4], dtype=torch.int32, device="cuda")
    store = torch.full((7, 208), 99, dtype=torch.int8, device="cuda")
    scale = torch.full((7,), -1.0, device="cuda")
    from lucid_b200._C._loader import LC_F32, check as ok, lib

    ok(lib.lc_quantize_tokens(x.data_ptr(), LC_F32, 7, 200, 200, None, 1, 7, valid.data_ptr(), store.data_ptr(), 208,
                              scale.data_ptr(), torch.cuda.current_stream().cuda_stream))
    np.testing.assert_array_equal(store[:4, :200].cpu().numpy().astype(np.int64), want_q[:4])
    assert (store[4:] == 99).all() and (scale[4:] == -1).all()  # rows behind the count stay as they were


# ---- dense product with epilogue ---------------------------------------------------------------
SHAPES = [(1, 1, 1), (1, 16, 64), (3, 130, 100), (16, 256, 512), (17, 128, 4096), (64, 300, 640), (65, 4096, 256),
          (130, 256, 128), (257, 520, 1040), (513, 272, 2080), (1, 4096, 14336), (33, 48, 8192)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("variant", [1, 2, 3, 4, 5, 6])
@pytest.mark.parametrize("unsigned", [False, True])
def test_product_is_exact_in_both_forms(ops, m, n, k, variant, unsigned):
    """With unit scales and fp32 results the product is the integer sum rounded once."""
    g = generator(m + 3 * n + 5 * k)
    lo, hi, dt = (0, 256, torch.uint8) if unsigned else (-128, 128, torch.int8)
    q = ops.pad_rows_to_16(torch.randint(lo, hi, (m, k), generator=g, device="cuda").to(dt))
    w = ops.pad_rows_to_16(torch.randint(-128, 128, (n, k), generator=g, device="cuda").to(torch.int8))
    wsum = w.int().sum(1, dtype=torch.int32) if unsigned else None
    zx = torch.tensor(113.0, device="cuda") if unsigned else None
    one = torch.ones(n, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = ops.grouped_qlinear_i8(q, w, torch.ones(1, device="cuda"), one, zx=zx, wsum=wsum, status=status, variant=variant)
    acc = (q.cpu().numpy().astype(np.int64) - (113 if unsigned else 0)) @ w.cpu().numpy().astype(np.int64).T
    np.testing.assert_array_equal(y.cpu().numpy(), acc.astype(np.float32))
    assert int(status) == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", [None, "relu", "gelu", "gelu_tanh", "silu", "swiglu"])
@pytest.mark.parametrize("m,n,k", [(1, 64, 96), (5, 48, 1003), (40, 272, 256), (200, 528, 512), (300, 80, 130)])
def test_linear(F, dtype, activation, m, n, k):
    g = generator(m + n + k)
    x = (2 * torch.randn(m, k, generator=g, device="cuda")).to(dtype)
    w, sw = make_weight(g, n, k)
    width = n // 2 if activation == "swiglu" else n
    for with_bias, with_residual in ((False, False), (True, True)):
        bias = torch.randn(n, generator=g, device="cuda") if with_bias else None
        res = torch.randn(m, width, generator=g, device="cuda").to(dtype) if with_residual else None
        y = F.linear(x, w, sw, bias, activation=activation, residual=res)
        q, s = plain_codes(x)
        want, err = plain_product(q, s, w.cpu().numpy(), f64(sw), None if bias is None else f64(bias), activation,
                                  None if res is None else f64(res))
        check(y, want, err, dtype)


@pytest.mark.parametrize("activation", ["gelu", "gelu_tanh", "silu", "swiglu"])
@pytest.mark.parametrize("dtype", TYPES)
def test_activations_over_their_range(ops, activation, dtype):
    """Pre-activations from -60 to 60, the tails included: acc = q * 1 with a scale per output column."""
    k, n = 16, 4096
    q = torch.zeros(3, k, dtype=torch.int8, device="cuda")
    q[:, 0] = torch.tensor([1, -1, 0], dtype=torch.int8)
    w = torch.zeros(n, k, dtype=torch.int8, device="cuda")
    w[:, 0] = 1
    sw = torch.linspace(1e-3, 60.0, n, device="cuda")
    y = ops.grouped_qlinear_i8(q, w, torch.ones(1, device="cuda"), sw, activation=activation, out_dtype=dtype)
    want, err = plain_product(q.cpu().numpy().astype(np.int64), np.ones(3), w.cpu().numpy(), f64(sw), None, activation)
    check(y, want, err, dtype)


def test_linear_shapes_strides_and_types(F):
    g = generator(11)
    w, sw = make_weight(g, 96, 160)
    wide = torch.randn(4, 6, 320, generator=g, device="cuda")
    x = wide[:, ::2, 7:167]  # neither dense nor aligned
    bias = torch.randn(96, generator=g, device="cuda", dtype=torch.float64).float()
    res = torch.randn(96, 4, 3, generator=g, device="cuda").permute(1, 2, 0)
    y = F.linear(x, w, sw, bias, activation="silu", residual=res)
    assert y.shape == (4, 3, 96)
    q, s = plain_codes(x.reshape(-1, 160))
    want, err = plain_product(q, s, w.cpu().numpy(), f64(sw), f64(bias), "silu", f64(res.reshape(-1, 96)))
    check(y.reshape(-1, 96), want, err, torch.float32)
    y16 = F.linear(x, w, sw, bias, activation="silu", residual=res.half(), out_dtype=torch.float16)
    want, err = plain_product(q, s, w.cpu().numpy(), f64(sw), f64(bias), "silu", f64(res.half().reshape(-1, 96)))
    check(y16.reshape(-1, 96), want, err, torch.float16)
    one = F.linear(x[0, 0], w, sw, bias)  # a vector
    assert one.shape == (96,)
    want, err = plain_product(q[:1], s[:1], w.cpu().numpy(), f64(sw), f64(bias), None)
    check(one[None], want, err, torch.float32)
    # a weight that is a slice of a larger one (rows on 16-byte boundaries): read where it lies
    big, bsw = make_weight(g, 200, 512)
    part = big[8:104, 16:176]
    assert F.pack_weight(part) is part
    y = F.linear(x, part, bsw[8:104])
    want, err = plain_product(q, s, part.cpu().numpy(), f64(bsw[8:104]), None, None)
    check(y.reshape(-1, 96), want, err, torch.float32)
    assert F.linear(x[:0], w, sw).shape == (0, 3, 96)


def test_extreme_codes_and_rows_of_zeros(F):
    k = 8192
    x = torch.zeros(3, k, device="cuda")
    x[0] = -1.0
    x[1] = 1.0  # (absmax / 127.5 = one step: code 127.5 rounds to 128 and is clamped to 127)
    w = torch.full((130, k), -128, dtype=torch.int8, device="cuda")
    sw = torch.ones(130, device="cuda")
    y = F.linear(x, w, sw)
    q, s = plain_codes(x)
    want, err = plain_product(q, s, w.cpu().numpy(), f64(sw), None, None)
    check(y, want, err, torch.float32)
    assert (y[2] == 0).all()


# ---- router ------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,experts,top_k", [(1, 1, 1), (1, 8, 2), (16, 64, 4), (100, 7, 7), (128, 33, 5), (129, 256, 8),
                                                  (1000, 60, 6), (2000, 128, 8), (64, 1024, 32), (300, 1000, 3)])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route(F, dtype, tokens, experts, top_k, renormalize):
    g = generator(tokens + experts)
    logits = (2 * torch.randn(tokens, experts, generator=g, device="cuda")).to(dtype)
    if tokens > 3:
        logits[tokens - tokens // 4:] = -math.inf             # padding
        logits[1, :max(1, experts - top_k // 2)] = -math.inf   # fewer candidates than choices
        logits[2] = 1.0                                        # all equal: the lowest experts
    r = F.route_experts(logits, top_k, renormalize=renormalize)
    weights, chosen, offsets, positions = plain_route(logits, top_k, renormalize)
    np.testing.assert_array_equal(r.experts.cpu().numpy(), chosen)
    np.testing.assert_array_equal(r.offsets.cpu().numpy(), offsets)
    np.testing.assert_array_equal(r.positions.cpu().numpy(), positions)
    # expf 2 ulp on either side of the quotient, log2(experts) + 32 additions of positive terms, one division
    np.testing.assert_allclose(r.weights.cpu().numpy(), weights, rtol=48 * 2.0 ** -23, atol=1e-37)


@pytest.mark.parametrize("experts,top_k", [(20, 20), (50, 32), (64, 8), (100, 16), (129, 8), (200, 32), (256, 9), (500, 12)])
def test_route_equal_logits(F, experts, top_k):
    # three values, so that nearly every choice is among equals; a NaN and a -inf between them
    logits = torch.randint(0, 3, (70, experts), generator=generator(experts), device="cuda").float()
    logits[::3, 7] = math.nan
    logits[::2, 9:12] = -math.inf
    r = F.route_experts(logits, top_k)
    weights, chosen, offsets, positions = plain_route(logits, top_k, True)
    np.testing.assert_array_equal(r.experts.cpu().numpy(), chosen)
    np.testing.assert_array_equal(r.offsets.cpu().numpy(), offsets)
    np.testing.assert_array_equal(r.positions.cpu().numpy(), positions)
    np.testing.assert_allclose(r.weights.cpu().numpy(), weights, rtol=48 * 2.0 ** -23)


@pytest.mark.parametrize("tokens,experts,top_k", [(5000, 600, 4), (6001, 1024, 2), (20000, 255, 8), (3333, 12, 12), (9_800_000, 3, 1)])
def test_route_many_tokens(F, tokens, experts, top_k):
    # the order "by expert, then by token" is the stable sort of the choices, which a sort of integers gives exactly
    logits = torch.randn(tokens, experts, generator=generator(tokens), device="cuda")
    r = F.route_experts(logits, top_k)
    assert torch.equal(r.experts.long(), torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :top_k])
    flat = r.experts.reshape(-1).long()
    order = torch.sort(flat, stable=True)[1]
    positions = torch.empty_like(order)
    positions[order] = torch.arange(order.numel(), device="cuda")
    assert torch.equal(r.positions.reshape(-1).long(), positions)
    counts = torch.bincount(flat, minlength=experts)
    assert torch.equal(r.offsets.long(), torch.cat([counts.new_zeros(1), counts.cumsum(0)]))


def test_route_special_logits(F):
    inf, nan, low = math.inf, math.nan, torch.finfo(torch.float32).min
    logits = torch.tensor([[inf, 1.0, inf, 0.0], [nan, 1.0, 2.0, nan], [nan, nan, nan, nan], [low, low, low, low],
                           [-inf, low, -inf, -inf], [0.0, -0.0, 0.0, -0.0], [inf, -inf, nan, 3.0]], device="cuda")
    for renormalize in (True, False):
        r = F.route_experts(logits, 3, renormalize=renormalize)
        weights, chosen, offsets, positions = plain_route(logits, 3, renormalize)
        np.testing.assert_array_equal(r.experts.cpu().numpy(), chosen)
        np.testing.assert_array_equal(r.offsets.cpu().numpy(), offsets)
        np.testing.assert_array_equal(r.positions.cpu().numpy(), positions)
        np.testing.assert_allclose(r.weights.cpu().numpy(), weights, rtol=48 * 2.0 ** -23)


def test_route_strided_and_empty(F):
    g = generator(5)
    wide = torch.randn(200, 96, generator=g, device="cuda")
    for logits in (wide[::2, 5:45], wide.t()[:40, :]):
        r = F.route_experts(logits, 4)
        weights, chosen, offsets, positions = plain_route(logits, 4, True)
        np.testing.assert_array_equal(r.experts.cpu().numpy(), chosen)
        np.testing.assert_array_equal(r.positions.cpu().numpy(), positions)
    r = F.route_experts(wide[:0], 4)
    assert r.rows == 0 and (r.offsets == 0).all()
    assert F.expert_linear(wide[:0], *make_weight(g, 96, 16, 96), r).shape == (0, 16)


# ---- grouped products ----------------------------------------------------------------------------
def routing_of(F, counts, top_k, g, extra=0):
    """A routing whose expert e owns counts[e] rows, with `extra` choices that go nowhere."""
    total = sum(counts)
    slots = total + extra
    assert slots % top_k == 0
    flat = torch.cat([torch.full((c,), e, dtype=torch.int32) for e, c in enumerate(counts)] +
                     [torch.full((extra,), -1, dtype=torch.int32)])
    perm = torch.randperm(slots, generator=torch.Generator().manual_seed(total + extra))
    flat = flat[perm]
    order = torch.argsort(torch.where(flat < 0, len(counts), flat), stable=True)
    positions = torch.empty(slots, dtype=torch.int32)
    positions[order] = torch.arange(slots, dtype=torch.int32)
    positions[flat < 0] = -1
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32)
    weights = torch.rand(slots, generator=torch.Generator().manual_seed(1))
    return F.ExpertRouting(*(t.cuda() for t in (weights.view(-1, top_k), flat.view(-1, top_k), offsets,
                                                positions.view(-1, top_k))))


COUNTS = {
    "one_each": ([1] * 12, 4, 0),
    "some_empty": ([0, 3, 0, 0, 17, 1, 0, 11], 2, 4),
    "all_in_one": ([0, 0, 130, 0], 2, 0),
    "tile_edges": ([16, 64, 65, 128, 256, 257, 31, 1], 2, 6),
    "nothing": ([0, 0, 0], 2, 8),
    "large": ([700, 3, 512, 0, 255, 900], 6, 18),
}


@pytest.mark.parametrize("case", list(COUNTS))
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation,n,k", [(None, 130, 260), ("swiglu", 288, 512), ("gelu", 256, 100)])
@pytest.mark.parametrize("sorted_rows", [False, True])
def test_expert_linear(F, case, dtype, activation, n, k, sorted_rows):
    counts, top_k, extra = COUNTS[case]
    g = generator(n + k)
    r = routing_of(F, counts, top_k, g, extra)
    x = (2 * torch.randn(r.rows if sorted_rows else r.tokens, k, generator=g, device="cuda")).to(dtype)
    if sorted_rows:
        x[sum(counts):] = math.nan  # what lies behind the last expert's rows is not read
    w, sw = make_weight(g, len(counts), n, k)
    bias = torch.randn(len(counts), n, generator=g, device="cuda")
    y = F.expert_linear(x, w, sw, r, bias, activation=activation, sorted_rows=sorted_rows)
    assert y.shape == (r.rows, n // 2 if activation == "swiglu" else n)
    q, s = plain_codes(x)
    source = np.zeros(r.rows, dtype=np.int64)
    positions = r.positions.cpu().numpy().reshape(-1)
    source[positions[positions >= 0]] = np.flatnonzero(positions >= 0) // top_k
    at = 0
    for e, c in enumerate(counts):
        rows = np.arange(at, at + c) if sorted_rows else source[at:at + c]
        want, err = plain_product(q[rows], s[rows], w[e].cpu().numpy(), f64(sw[e]), f64(bias[e]), activation)
        check(y[at:at + c], want, err, dtype)
        at += c
    assert (y[at:] == 0).all()


@pytest.mark.parametrize("variant", [1, 2, 3, 4, 5, 6])
@pytest.mark.parametrize("case", list(COUNTS))
def test_grouped_product_forms_agree(ops, F, variant, case):
    counts, top_k, extra = COUNTS[case]
    g = generator(1)
    rows, n, k = sum(counts) + extra, 200, 1200
    q = torch.randint(-128, 128, (rows, k), generator=g, device="cuda").to(torch.int8)
    w = torch.randint(-128, 128, (len(counts), n, k), generator=g, device="cuda").to(torch.int8)
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
    one = torch.ones(len(counts), n, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = ops.grouped_qlinear_i8(q, w, torch.ones(1, device="cuda"), one, offsets=offsets, status=status, variant=variant)
    want = np.zeros((rows, n), np.float32)
    at = 0
    for e, c in enumerate(counts):
        want[at:at + c] = (q[at:at + c].cpu().numpy().astype(np.int64) @ w[e].cpu().numpy().astype(np.int64).T)
        at += c
    np.testing.assert_array_equal(y.cpu().numpy(), want)
    assert int(status) == 0


def test_offsets_outside_the_rows_are_clamped(ops):
    g = generator(2)
    q = torch.randint(-128, 128, (40, 64), generator=g, device="cuda").to(torch.int8)
    w = torch.randint(-128, 128, (3, 32, 64), generator=g, device="cuda").to(torch.int8)
    one = torch.ones(3, 32, device="cuda")
    offsets = torch.tensor([-5, 10, 3, 10 ** 6], dtype=torch.int32, device="cuda")
    store = torch.full((44, 32), 7.0, device="cuda")
    from lucid_b200._C._loader import LC_F32, check as ok, lib

    sx = torch.ones(1, device="cuda")
    ok(lib.lc_grouped_qlinear_i8(q.data_ptr(), 0, 64, 40, offsets.data_ptr(), 3, w.data_ptr(), 64, 32 * 64, 32, 64,
                                 sx.data_ptr(), 0, None, None, one.data_ptr(), None, 0, None, 0, store.data_ptr(), LC_F32,
                                 32, None, 0, torch.cuda.current_stream().cuda_stream))
    want = q[:10].cpu().numpy().astype(np.int64) @ w[0].cpu().numpy().astype(np.int64).T
    np.testing.assert_array_equal(store[:3].cpu().numpy(), want[:3].astype(np.float32))
    assert (store[40:] == 7.0).all()  # nothing behind the rows is written


# ---- combination -----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,top_k,n,missing", [(1, 1, 1, 0), (5, 2, 17, 0), (16, 4, 4096, 0), (33, 8, 128, 40),
                                                    (100, 3, 1000, 17), (4, 9, 72, 36)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_combine(F, dtype, tokens, top_k, n, missing, with_residual):
    g = generator(tokens + n)
    rows = tokens * top_k
    positions = torch.randperm(rows, generator=g, device="cuda").int()
    positions[torch.randperm(rows, generator=g, device="cuda")[:missing]] = -1
    positions = positions.view(tokens, top_k)
    weights = torch.rand(tokens, top_k, generator=g, device="cuda")
    r = F.ExpertRouting(weights, torch.zeros_like(positions), torch.tensor([0, rows], dtype=torch.int32, device="cuda"),
                        positions)
    y = torch.randn(rows, n, generator=g, device="cuda").to(dtype)
    res = torch.randn(tokens, n, generator=g, device="cuda").to(dtype) if with_residual else None
    out = F.combine_experts(y, r, residual=res)
    terms = np.where((positions.cpu().numpy() < 0)[..., None], 0.0,
                     f64(y)[positions.cpu().numpy().clip(0)] * f64(weights)[..., None])
    want = terms.sum(1) + (0.0 if res is None else f64(res))
    # one rounding per term and one for the residual, each of a partial sum that the magnitudes bound
    err = (top_k + 1) * U * (np.abs(terms).sum(1) + (0.0 if res is None else np.abs(f64(res))))
    check(out, want, err, dtype)


# ---- the operators together ------------------------------------------------------------------------
def plain_block(x, logits, top_k, gate_up, sgu, down, sd, dtype):
    """The block with the intermediate rows rounded to their type; what the next quantizer may see one step apart
    is allowed for by the caller's bound."""
    weights, chosen, offsets, positions = plain_route(logits, top_k, True)
    out = f64(x).copy()
    scale = np.zeros(out.shape[0])
    for t in range(out.shape[0]):
        for j in range(top_k):
            e = chosen[t, j]
            if e < 0:
                continue
            q, s = plain_codes(x[t:t + 1])
            h, _ = plain_product(q, s, gate_up[e].cpu().numpy(), f64(sgu[e]), None, "swiglu")
            h = torch.tensor(h).to(dtype)
            q, s = plain_codes(h)
            y, _ = plain_product(q, s, down[e].cpu().numpy(), f64(sd[e]), None, None)
            out[t] += weights[t, j] * y[0]
            # one step of the codes' grid and one of the type on every entry of h, against the weight's row
            step = float(s[0]) + torch.finfo(dtype).eps * np.abs(f64(h)).max()
            scale[t] += weights[t, j] * step * (np.abs(f64(down[e])) * f64(sd[e])[:, None]).sum(1).max() * 0.02
            scale[t] += weights[t, j] * torch.finfo(dtype).eps * np.abs(y).max()
    return out, scale


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 12, 150])
def test_block(F, dtype, tokens):
    """Router, both products and the combination as a block uses them.  The intermediate row h agrees with the plain
    one up to its rounding; where that lands next to the middle of two codes the code differs by one.  At most 2 % of
    the entries are let differ at once (a value is that close to a middle with a probability of about 2^-8 for the
    coarsest type), each counted with the largest absolute row sum of the weight."""
    g = generator(tokens)
    e, top_k, k, inter = 6, 2, 256, 192
    x = torch.randn(tokens, k, generator=g, device="cuda").to(dtype)
    logits = torch.randn(tokens, e, generator=g, device="cuda")
    if tokens >= 5:
        logits[tokens - tokens // 5:] = -math.inf
    gate_up, sgu = make_weight(g, e, 2 * inter, k)
    down, sd = make_weight(g, e, k, inter)

    def block():
        r = F.route_experts(logits, top_k)
        h = F.expert_linear(x, gate_up, sgu, r, activation="swiglu")
        y = F.expert_linear(h, down, sd, r, sorted_rows=True)
        return F.combine_experts(y, r, residual=x)

    out = block()
    want, scale = plain_block(x, logits, top_k, gate_up, sgu, down, sd, dtype)
    half = torch.finfo(dtype).eps / 2
    bound = scale[:, None] + half * np.abs(want) + 1e-5 * np.abs(want).max()
    assert (np.abs(f64(out) - want) <= bound).all()
    # the same bits again, from a captured graph with new inputs, and on another stream
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = block()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = block()
    fresh_x = torch.randn(tokens, k, generator=g, device="cuda").to(dtype)
    fresh_l = torch.randn(tokens, e, generator=g, device="cuda")
    x.copy_(fresh_x)
    logits.copy_(fresh_l)
    graph.replay()
    eager = block()
    assert torch.equal(captured, eager) and not torch.equal(captured, out)


def test_two_graphs_in_flight(F):
    """Two captured blocks replayed on two streams at once do not share scratch memory."""
    g = generator(9)
    w, sw = make_weight(g, 2048, 1024)
    xs = [torch.randn(200, 1024, generator=g, device="cuda") for _ in range(2)]
    want = [F.linear(x, w, sw, activation="silu") for x in xs]
    graphs, outs = [], []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(F.linear(x, w, sw, activation="silu"))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("variant", [1, 2, 3, 4, 5, 6])
def test_waits_that_run_out_leave_a_status(ops, variant):
    from lucid_b200._C._loader import LC_QLINEAR_WAIT_TEST, LucidCudaError

    g = generator(4)
    q = torch.randint(-128, 128, (200, 4096), generator=g, device="cuda").to(torch.int8)
    w = torch.randint(-128, 128, (256, 4096), generator=g, device="cuda").to(torch.int8)
    one = torch.ones(256, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.grouped_qlinear_i8(q, w, one[:1], one, status=status, variant=variant | LC_QLINEAR_WAIT_TEST)
    with pytest.raises(LucidCudaError, match="ran out"):
        ops.qlinear_check_status(status)
    y = ops.grouped_qlinear_i8(q, w, one[:1], one, variant=variant)  # the GPU keeps working
    want = (q.cpu().numpy().astype(np.int64) @ w.cpu().numpy().astype(np.int64).T).astype(np.float32)
    np.testing.assert_array_equal(y.cpu().numpy(), want)


# ---- the native form of ordinary calls -----------------------------------------------------------------
def test_native_and_python_forms_agree(F, ops, monkeypatch):
    assert ops.torchcall is not None, "lucid_b200/_C/_torchcall was not built"
    g = generator(21)
    x = torch.randn(48, 96, generator=g, device="cuda").bfloat16()
    w, sw = make_weight(g, 64, 96)
    we, se = make_weight(g, 5, 64, 96)
    res, bias = torch.randn(48, 64, generator=g, device="cuda").bfloat16(), torch.randn(64, generator=g, device="cuda")
    logits = torch.randn(48, 5, generator=g, device="cuda")

    def calls():
        r = F.route_experts(logits, 2, renormalize=False)
        h = F.expert_linear(x, we, se, r, activation="silu", out_dtype=torch.float16)
        y = F.expert_linear(h[:, :64].contiguous(), we[:, :, :64].contiguous(), se, r, sorted_rows=True)
        return [r.weights, r.experts, r.offsets, r.positions, h, y, F.combine_experts(y, r), F.linear(x, w, sw),
                F.linear(x, w, sw, bias, activation="gelu", residual=res),
                F.linear(x, w, sw, activation="swiglu", out_dtype=torch.float32)]

    native = calls()
    monkeypatch.setattr(ops, "torchcall", None)
    for a, b in zip(native, calls()):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)
    monkeypatch.undo()
    t = ops.torchcall
    # calls that are not ordinary are left to the Python form
    assert t.product(x[:, ::2], w[:, :48], sw, None, 0, None, None, None, None) is None      # strided rows
    assert t.product(x, w, sw.double(), None, 0, None, None, None, None) is None             # another type
    assert t.product(x, w, sw, None, 7, None, None, None, None) is None                      # no such activation
    assert t.product(x, w, sw, None, 0, res.float(), None, None, None) is None               # residual of another type
    assert t.product(x, w[:, :90], sw, None, 0, None, None, None, None) is None              # does not contract
    assert t.product(x[:0], w, sw, None, 0, None, None, None, None) is None                  # empty
    assert t.product(x.cpu(), w, sw, None, 0, None, None, None, None) is None
    assert t.route(logits, 6, True) is None and t.route(logits[:0], 2, True) is None
    assert t.combine(native[5][:90], native[0], native[3], None) is None
    with pytest.raises(TypeError):
        t.product(x)


def test_calls_from_another_stream_and_thread(F):
    """Calls of two host threads on two streams at once."""
    import threading

    g = generator(33)
    w, sw = make_weight(g, 512, 1024)
    xs = [torch.randn(40, 1024, generator=g, device="cuda") for _ in range(2)]
    want = [F.linear(x, w, sw, activation="gelu") for x in xs]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i].append(F.linear(xs[i], w, sw, activation="gelu"))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


# ---- calls the documentation allows and nothing above makes --------------------------------------------
def test_offsets_out_of_order_are_made_ascending(ops):
    """Nothing outside is read or written and every row is computed at most once, whatever the offsets hold."""
    g = generator(8)
    rows, n, k = 300, 64, 64
    q = torch.randint(-128, 128, (rows, k), generator=g, device="cuda").to(torch.int8)
    w = torch.randint(-128, 128, (40, n, k), generator=g, device="cuda").to(torch.int8)
    one = torch.ones(40, n, device="cuda")
    raw = torch.randint(-50, 400, (41,), generator=g, device="cuda", dtype=torch.int32)
    ends = torch.cummax(raw.clamp(0, rows), 0).values.tolist()
    for variant in range(7):
        y = ops.grouped_qlinear_i8(q, w, one[0, :1], one, offsets=raw, variant=variant)
        want = np.zeros((rows, n), np.float32)
        for e in range(40):
            a, b = ends[e], ends[e + 1]
            want[a:b] = q[a:b].cpu().numpy().astype(np.int64) @ w[e].cpu().numpy().astype(np.int64).T
        got = y.cpu().numpy()
        np.testing.assert_array_equal(got[ends[0]:], want[ends[0]:])  # (rows before the first group are nobody's)


def test_weights_that_are_views(F):
    g = generator(12)
    base = torch.randint(-128, 128, (6, 48, 96), generator=g, device="cuda").to(torch.int8)
    sw = 0.002 * (0.5 + torch.rand(6, 48, generator=g, device="cuda"))
    r = F.route_experts(torch.randn(20, 6, generator=g, device="cuda"), 2)
    x = torch.randn(20, 64, generator=g, device="cuda")
    for view in (base[:, :, 16:80], base[:, ::2, :64].repeat_interleave(2, 1), base[:1, :, :64].expand(6, 48, 64),
                 base.transpose(0, 1).contiguous().transpose(0, 1)[:, :, :64], base[..., 1:65]):
        got = F.expert_linear(x, view, sw, r)
        assert torch.equal(got, F.expert_linear(x, view.contiguous(), sw, r))


def test_values_that_are_not_numbers(F):
    g = generator(14)
    w, sw = make_weight(g, 64, 128)
    x = torch.randn(4, 128, generator=g, device="cuda")
    x[1, 5] = math.nan
    x[2, 7] = -math.inf
    clean = x.clone()
    clean[1, 5] = 0.0
    for activation in (None, "relu", "gelu", "gelu_tanh", "silu", "swiglu"):
        y = F.linear(x, w, sw, activation=activation)
        assert torch.equal(y[[0, 1, 3]], F.linear(clean, w, sw, activation=activation)[[0, 1, 3]])
        assert y[2].isnan().all()


def test_one_row_in_all_experts_and_many_experts(F):
    g = generator(15)
    w, sw = make_weight(g, 1024, 16, 32)
    x = torch.randn(3, 32, generator=g, device="cuda").half()
    r = F.route_experts(torch.randn(3, 1024, generator=g, device="cuda"), 32)
    y = F.expert_linear(x, w, sw, r)
    q, s = plain_codes(x)
    experts, positions = r.experts.cpu().numpy(), r.positions.cpu().numpy()
    for t in range(3):
        for j in range(32):
            e = experts[t, j]
            want, err = plain_product(q[t:t + 1], s[t:t + 1], w[e].cpu().numpy(), f64(sw[e]), None, None)
            check(y[positions[t, j]][None], want, err, torch.float16)


def test_first_call_of_a_process_inside_a_capture():
    """Nothing the operators set up on their first call disturbs a graph capture."""
    import os
    import subprocess
    import sys

    code = """
import torch
from lucid_b200.nn.quantized.dynamic import functional as F
x = torch.randn(5, 64, device="cuda"); logits = torch.randn(5, 4, device="cuda")
w = torch.randint(-9, 9, (4, 64, 64), device="cuda").to(torch.int8); s = torch.ones(4, 64, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    r = F.route_experts(logits, 2)
    y = F.combine_experts(F.expert_linear(x, w, s, r, activation="silu"), r)
graph.replay()
r2 = F.route_experts(logits, 2)
assert torch.equal(y, F.combine_experts(F.expert_linear(x, w, s, r2, activation="silu"), r2))
print("same")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=root, timeout=300)
    assert done.returncode == 0 and "same" in done.stdout, done.stderr[-2000:]


@pytest.mark.parametrize("rows", [70000])
def test_offsets_beyond_32_bits(F, rows):
    """Elements of the input and the result past 2^31."""
    g = generator(16)
    k, n = 32784, 32
    x = torch.empty(rows, k, dtype=torch.bfloat16, device="cuda")
    assert x.numel() > 2 ** 31
    tail = torch.randn(3, k, generator=g, device="cuda").bfloat16()
    x[:-3] = 0
    x[-3:] = tail
    w, sw = make_weight(g, n, k)
    y = F.linear(x, w, sw)
    assert torch.equal(y[-3:], F.linear(tail, w, sw)) and (y[:-3] == 0).all()
    wide, wsw = make_weight(g, 40960, 64)
    small = torch.randn(53000, 64, generator=g, device="cuda").bfloat16()
    big = F.linear(small, wide, wsw)
    assert big.numel() > 2 ** 31
    assert torch.equal(big[-5:], F.linear(small[-5:], wide, wsw))


def test_refusals_of_the_library_reach_python(F):
    from lucid_b200._C import LucidCudaError

    x, w = torch.zeros(2, 65552, device="cuda"), torch.zeros(16, 65552, dtype=torch.int8, device="cuda")
    with pytest.raises(LucidCudaError, match="overflow"):
        F.linear(x, w, torch.ones(16, device="cuda"))
    with pytest.raises(ValueError, match="residual"):
        F.linear(x[:, :64].contiguous(), w[:, :64], torch.ones(16, device="cuda"), residual=torch.zeros(3, 16, device="cuda"))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        F.linear(torch.zeros(2, 64), w[:, :64].cpu(), torch.ones(16))
    with pytest.raises(RuntimeError, match="different devices"):
        F.linear(x[:, :64].contiguous(), w[:, :64].cpu(), torch.ones(16, device="cuda"))
    ok = F.linear(x[:, :64].contiguous(), w[:, :64], torch.ones(16, device="cuda"))  # and the GPU goes on
    assert (ok == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_rows_of_every_alignment(ops, dtype):
    """Rows whose start, pitch and length are no multiples of a vector."""
    g = generator(40)
    store = torch.randn(64 * 4200, generator=g, device="cuda").to(dtype)
    for cols, ldx in ((1, 1), (7, 7), (9, 13), (31, 33), (255, 257), (1003, 1003), (1021, 1029), (2049, 2051), (4099, 4101)):
        for start in (0, 1, 3, 6):
            rows = min(13, (store.numel() - start) // ldx)
            x = store[start:].as_strided((rows, cols), (ldx, 1))
            q, s = ops.quantize_tokens(x)
            want_q, want_s = plain_codes(x)
            np.testing.assert_array_equal(q.cpu().numpy().astype(np.int64), want_q)
            np.testing.assert_array_equal(f64(s), want_s)
