"""The modules that the expert and fused-epilogue operators serve: host logic on CPU against a plain stand-in for
the kernels, and the same tests on the kernels."""
import types

import pytest
import torch
from torch import nn

import lucid_b200.quantization as Q
from lucid_b200 import _backend
from lucid_b200.nn.quantized import dynamic as nnqd
from lucid_b200.nn.quantized.dynamic import functional as F


# ---- plain stand-ins (64 bits) -----------------------------------------------------------------
def _act(v, name):
    if name == "relu":
        return v.clamp_min(0)
    if name == "gelu":
        return nn.functional.gelu(v)
    if name == "gelu_tanh":
        return nn.functional.gelu(v, approximate="tanh")
    if name == "silu":
        return nn.functional.silu(v)
    if name == "swiglu":
        g, u = v.unflatten(-1, (-1, 2, 8)).unbind(-2)
        return (nn.functional.silu(g) * u).flatten(-2)
    return v


def _codes(x):
    s = (x.float().abs().amax(1) / torch.tensor(127.5)).clamp_min(1e-8)
    return torch.round(x.float() * (1.0 / s)[:, None]).clamp(-128, 127), s


def _fake_grouped(q, wq, sx, sw, bias=None, offsets=None, zx=None, wsum=None, activation=None, residual=None,
                  out_dtype=torch.float32, status=None, variant=0):
    assert offsets is None
    acc = q.double() @ wq.double().t()
    if zx is not None:
        acc = acc - float(zx) * wsum.double()[None]
    y = acc * sx.double().reshape(-1, 1) * sw.double()
    if bias is not None:
        y = y + bias.double()
    y = _act(y, activation)
    return (y if residual is None else y + residual.double()).to(out_dtype)


def _fake_expert_linear(x2d, wq, sw, bias, positions, offsets, rows, activation, residual, width, out_dtype, dev):
    name = F.ACTIVATIONS[activation]
    q, s = _codes(x2d)
    if wq.dim() == 2:
        return _fake_grouped(q, wq, s, sw, bias, activation=name, residual=residual, out_dtype=out_dtype)
    if positions is not None:
        source = torch.zeros(rows, dtype=torch.long)
        flat = positions.reshape(-1).long()
        source[flat[flat >= 0]] = torch.arange(flat.numel())[flat >= 0] // positions.shape[1]
        q, s = q[source], s[source]
    y = torch.zeros(rows, width, dtype=out_dtype)
    for e in range(wq.shape[0]):
        a, b = int(offsets[e]), int(offsets[e + 1])
        y[a:b] = _fake_grouped(q[a:b], wq[e], s[a:b], sw[e], None if bias is None else bias[e], activation=name,
                               out_dtype=out_dtype)
    return y


def _fake_route(logits, top_k, renormalize):
    values, experts = torch.sort(logits.double(), dim=-1, descending=True, stable=True)
    p = torch.softmax(values, -1).nan_to_num(0.0)[:, :top_k]
    if renormalize:
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    gone = values[:, :top_k] == -float("inf")
    experts = torch.where(gone, -1, experts[:, :top_k])
    flat = experts.reshape(-1)
    order = torch.sort(torch.where(flat < 0, logits.shape[1], flat), stable=True).indices
    positions = torch.empty_like(flat)
    positions[order] = torch.arange(flat.numel())
    positions = torch.where(flat < 0, -1, positions).view_as(experts)
    counts = torch.bincount(flat[flat >= 0], minlength=logits.shape[1])
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)])
    return torch.where(gone, 0.0, p).float(), experts.int(), offsets.int(), positions.int()


def _fake_combine(y, weights, positions, residual, dev):
    out = torch.where(positions[..., None] < 0, 0.0, y[positions.clamp_min(0).long()].double() * weights[..., None]).sum(1)
    return (out if residual is None else out + residual.double()).to(y.dtype)


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def device(request, monkeypatch):
    if request.param == "cpu":
        from tests import fake_ops

        fakes = types.SimpleNamespace(**{k: v for k, v in vars(fake_ops).items() if not k.startswith("__")})
        fakes.grouped_qlinear_i8, fakes.expert_linear = _fake_grouped, _fake_expert_linear
        fakes.route_experts, fakes.combine_experts = _fake_route, _fake_combine
        from lucid_b200._C import ops

        fakes.interleave_gate_up = ops.interleave_gate_up
        monkeypatch.setattr(_backend, "ops", lambda: fakes)
        monkeypatch.setattr(_backend, "on_cuda", lambda t: t)
        monkeypatch.setattr(F, "_check_cuda", lambda *a: None)
    return request.param


def _rel(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return float((a - b).abs().max() / a.abs().max())


# ---- the dynamic Linear with an epilogue -----------------------------------------------------------
@pytest.mark.parametrize("scheme", ["tensor_affine", "tensor_symmetric", "token_symmetric"])
@pytest.mark.parametrize("activation", [None, "relu", "gelu", "gelu_tanh", "silu"])
def test_dynamic_linear_epilogue_equals_separate_steps(device, scheme, activation):
    """Same codes, same integer sums: the fused result differs from layer + activation + add in 64 bits by the
    rounding of a few fp32 steps only."""
    torch.manual_seed(0)
    lin = nn.Linear(96, 40)
    m = nnqd.Linear.from_float(lin).set_activation_scheme(scheme)
    x, r = torch.randn(3, 7, 96), torch.randn(3, 7, 40)
    plain = m(x.to(device)).double().cpu()
    want = _act(plain, activation) + r
    m.set_activation(activation)
    got = m(x.to(device), residual=r.to(device))
    assert got.shape == (3, 7, 40) and got.dtype == torch.float32 and got.device.type == device
    # the plain layer's own three roundings and the fused one's, each 2^-24 of |product| + |bias|; 2^-20 for the activation
    torch.testing.assert_close(got.double().cpu(), want, rtol=2.0 ** -20, atol=2.0 ** -20 * float(plain.abs().max()))
    no_residual = m(x.to(device))
    torch.testing.assert_close(no_residual.double().cpu(), _act(plain, activation), rtol=2.0 ** -20,
                               atol=2.0 ** -20 * float(plain.abs().max()))
    if activation is None:
        assert torch.equal(no_residual.double().cpu(), plain)  # without an epilogue the layer is what it was


def test_dynamic_linear_epilogue_checks(device):
    m = nnqd.Linear.from_float(nn.Linear(32, 16))
    with pytest.raises(ValueError, match="activation"):
        m.set_activation("swiglu")
    with pytest.raises(ValueError, match="residual"):
        m(torch.zeros(2, 32).to(device), residual=torch.zeros(2, 15).to(device))
    assert "activation=gelu" in repr(m.set_activation("gelu"))
    assert m(torch.zeros(0, 32).to(device)).shape == (0, 16)


def test_shared_codes_reach_the_epilogue(device):
    torch.manual_seed(1)
    a, b = (nnqd.Linear.from_float(nn.Linear(64, 24)) for _ in range(2))
    a.set_activation("silu")
    x = torch.randn(5, 64).to(device)
    want = a(x), b(x)
    with nnqd.share_quantized_input():
        got = a(x), b(x)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---- the mixture of experts ---------------------------------------------------------------------------
def _float_experts(hidden, inter, experts):
    torch.manual_seed(3)
    mk = lambda i, o: [nn.Linear(i, o, bias=False) for _ in range(experts)]
    return nn.Linear(hidden, experts, bias=False), mk(hidden, inter), mk(hidden, inter), mk(inter, hidden)


def _float_forward(x, router, gates, ups, downs, top_k, renormalize):
    p = torch.softmax(router(x), -1)
    w, e = p.topk(top_k, -1)
    if renormalize:
        w = w / w.sum(-1, keepdim=True)
    out = torch.zeros_like(x)
    for t in range(x.shape[0]):
        for j in range(top_k):
            i = int(e[t, j])
            out[t] += w[t, j] * downs[i](nn.functional.silu(gates[i](x[t])) * ups[i](x[t]))
    return out


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("tokens", [1, 40])
def test_moe_tracks_the_float_model(device, renormalize, tokens):
    parts = _float_experts(64, 48, 6)
    m = nnqd.MoESwiGLU.from_float(*parts, top_k=2, renormalize=renormalize)
    x = torch.randn(tokens, 64)
    with torch.no_grad():
        want = _float_forward(x, *parts, 2, renormalize)
        got = m(x.to(device))
    assert got.shape == x.shape and got.device.type == device and not got.requires_grad
    # two int8 quantizations on each side of both products: half a step of 1/127 each, four in all, of the maximum
    assert _rel(want, got) < 4 * 0.5 / 127 * 2


def test_moe_residual_mask_and_shapes(device):
    m = nnqd.MoESwiGLU.from_float(*_float_experts(64, 48, 6), top_k=3)
    x, r = torch.randn(2, 9, 64).to(device), torch.randn(2, 9, 64).to(device)
    mask = torch.ones(2, 9, dtype=torch.bool)
    mask[1, 5:] = False
    mask = mask.to(device)
    y, z = m(x), m(x, residual=r, token_mask=mask)
    assert z.shape == x.shape
    assert torch.equal(z[~mask], r[~mask])  # a masked token goes nowhere
    torch.testing.assert_close(z[mask], (y + r)[mask], rtol=1e-5, atol=1e-5 * float(y.abs().max()))
    assert (m(x, token_mask=torch.zeros_like(mask)) == 0).all()
    assert m(x[:, :0]).shape == (2, 0, 64)
    with pytest.raises(ValueError, match="features"):
        m(x[..., :32])
    with pytest.raises(ValueError, match="residual"):
        m(x, residual=r[:1])
    with pytest.raises(ValueError, match="token_mask"):
        m(x, token_mask=mask[:1])


def test_moe_state_dict_round_trip(device, tmp_path):
    from lucid_b200.serialization import load_safetensors, save_safetensors

    m = nnqd.MoESwiGLU.from_float(*_float_experts(64, 48, 6), top_k=2)
    x = torch.randn(5, 64).to(device)
    want = m(x)
    save_safetensors(m.state_dict(), tmp_path / "moe.safetensors")
    fresh = nnqd.MoESwiGLU(64, 48, 6, 2).to(device)
    fresh.load_state_dict(load_safetensors(tmp_path / "moe.safetensors"))
    assert torch.equal(fresh(x), want)
    assert fresh.gate_up_int8.shape == (6, 96, 64) and fresh.down_scale.shape == (6, 64)


def test_moe_construction_checks(device):
    with pytest.raises(ValueError, match="multiples of 16"):
        nnqd.MoESwiGLU(60, 48, 4, 2)
    with pytest.raises(ValueError, match="top_k"):
        nnqd.MoESwiGLU(64, 48, 4, 5)
    router, gates, ups, downs = _float_experts(64, 48, 4)
    with pytest.raises(ValueError, match="router outputs"):
        nnqd.MoESwiGLU.from_float(router, gates[:3], ups, downs, top_k=2)
    with pytest.raises(ValueError, match="biases"):
        nnqd.MoESwiGLU.from_float(nn.Linear(64, 4), gates, ups, downs, top_k=2)


@pytest.mark.gpu
def test_moe_is_captured_in_a_graph():
    m = nnqd.MoESwiGLU.from_float(*_float_experts(64, 48, 6), top_k=2)
    m.router.to("cuda")
    x = torch.randn(30, 64, device="cuda")
    m(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m(x, residual=x)
    x.copy_(torch.randn(30, 64, device="cuda"))
    graph.replay()
    assert torch.equal(out, m(x, residual=x))


def test_alias_and_names():
    import lucid

    from lucid.nn.quantized.dynamic import functional as aliased

    assert aliased is F and lucid.nn.quantized.dynamic.MoESwiGLU is nnqd.MoESwiGLU
    assert set(F.__all__) >= {"linear", "route_experts", "expert_linear", "combine_experts"}
    assert Q.qint8.quant_max == 127  # the activation grid these operators use
