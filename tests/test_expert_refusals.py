"""What the functional forms of the dynamic Linear and the expert operators refuse, checked on the host before
anything is launched."""
import ctypes

import pytest
import torch

from lucid_b200.nn.quantized.dynamic import functional as F


def routing(tokens=4, top_k=2, experts=3):
    z = torch.zeros(tokens, top_k, dtype=torch.int32)
    return F.ExpertRouting(torch.zeros(tokens, top_k), z, torch.zeros(experts + 1, dtype=torch.int32), z)


def test_cpu_tensors_are_refused():
    w, s = torch.zeros(16, 32, dtype=torch.int8), torch.ones(16)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        F.linear(torch.zeros(2, 32), w, s)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        F.route_experts(torch.zeros(2, 8), 2)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        F.expert_linear(torch.zeros(4, 32), w.expand(3, 16, 32), s.expand(3, 16), routing())
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        F.combine_experts(torch.zeros(8, 16), routing())


@pytest.mark.parametrize("top_k,experts", [(0, 4), (5, 4), (33, 64), (1, 1025), (-1, 4)])
def test_router_sizes(top_k, experts):
    with pytest.raises(ValueError, match="top_k"):
        F.route_experts(torch.zeros(2, experts), top_k)


def test_router_types():
    with pytest.raises(TypeError):
        F.route_experts(torch.zeros(2, 4, dtype=torch.int32), 1)
    with pytest.raises(ValueError):
        F.route_experts(torch.zeros(4), 1)


def test_routing_is_checked():
    w, i = torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32)
    o = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        F.ExpertRouting(w, i[:3], o, i)
    with pytest.raises(ValueError):
        F.ExpertRouting(w, i, o[:1], i)
    with pytest.raises(TypeError, match="positions"):
        F.ExpertRouting(w, i, o, i.long())
    with pytest.raises(TypeError, match="weights"):
        F.ExpertRouting(w.double(), i, o, i)


def test_weights_are_checked():
    with pytest.raises(TypeError):
        F.pack_weight(torch.zeros(4, 4))
    with pytest.raises(ValueError):
        F.pack_weight(torch.zeros(4, dtype=torch.int8))
    w = torch.randint(-128, 128, (3, 5, 20)).to(torch.int8)
    p = F.pack_weight(w)
    assert torch.equal(p, w) and p.stride(1) % 16 == 0 and p.stride(0) % 16 == 0 and F.pack_weight(p) is p
    aligned = torch.zeros(4, 32, dtype=torch.int8)
    assert F.pack_weight(aligned) is aligned
    assert F.pack_weight(aligned.t()).stride(-1) == 1


@pytest.mark.parametrize("kwargs,error", [
    (dict(activation="tanh"), ValueError), (dict(activation="swiglu"), ValueError),
    (dict(out_dtype=torch.float64), TypeError), (dict(residual=torch.zeros(2, 24)), ValueError),
    (dict(bias=torch.zeros(24)), ValueError)])
def test_linear_arguments(kwargs, error, monkeypatch):
    monkeypatch.setattr(F, "_check_cuda", lambda *a: None)
    with pytest.raises(error):
        F.linear(torch.zeros(2, 32), torch.zeros(25, 32, dtype=torch.int8), torch.ones(25), **kwargs)
    with pytest.raises(ValueError, match="contract"):
        F.linear(torch.zeros(2, 31), torch.zeros(25, 32, dtype=torch.int8), torch.ones(25))
    with pytest.raises(TypeError):
        F.linear(torch.zeros(2, 32, dtype=torch.float64), torch.zeros(25, 32, dtype=torch.int8), torch.ones(25))
    with pytest.raises(TypeError, match="residual"):
        F.linear(torch.zeros(2, 32), torch.zeros(25, 32, dtype=torch.int8), torch.ones(25),
                 residual=torch.zeros(2, 25, dtype=torch.float16))
    with pytest.raises(ValueError, match="weight_scale"):
        F.linear(torch.zeros(2, 32), torch.zeros(25, 32, dtype=torch.int8), torch.ones(24))


def test_expert_linear_arguments(monkeypatch):
    monkeypatch.setattr(F, "_check_cuda", lambda *a: None)
    w, s = torch.zeros(3, 16, 32, dtype=torch.int8), torch.ones(3, 16)
    with pytest.raises(ValueError, match="experts"):
        F.expert_linear(torch.zeros(4, 32), w, s, routing(experts=4))
    with pytest.raises(ValueError, match="input"):
        F.expert_linear(torch.zeros(5, 32), w, s, routing())
    with pytest.raises(ValueError, match="input"):  # sorted rows: one per choice
        F.expert_linear(torch.zeros(4, 32), w, s, routing(), sorted_rows=True)
    with pytest.raises(ValueError, match="weight_scale"):
        F.expert_linear(torch.zeros(4, 32), w, torch.ones(16), routing())
    with pytest.raises(ValueError, match="weight must be"):
        F.expert_linear(torch.zeros(4, 32), w[0], s, routing())


def test_combine_arguments(monkeypatch):
    monkeypatch.setattr(F, "_check_cuda", lambda *a: None)
    with pytest.raises(ValueError):
        F.combine_experts(torch.zeros(7, 16), routing())
    with pytest.raises(ValueError, match="residual"):
        F.combine_experts(torch.zeros(8, 16), routing(), residual=torch.zeros(8, 16))
    with pytest.raises(TypeError, match="residual"):
        F.combine_experts(torch.zeros(8, 16), routing(), residual=torch.zeros(4, 16).half())


def test_c_entry_points_refuse_before_they_launch():
    import lucid_b200._C as capi

    L = capi.lib
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256

    def product(q=p, ldq=32, rows=4, offsets=None, groups=1, w=p, ldw=32, stride=512, n=16, k=32, sx=p, zx=None, wsum=None,
                sw=p, act=0, out=p, dtype=capi.LC_F32, ldo=16, variant=0):
        return L.lc_grouped_qlinear_i8(q, 0, ldq, rows, offsets, groups, w, ldw, stride, n, k, sx, 0, zx, wsum, sw, None,
                                       act, None, 0, out, dtype, ldo, None, variant, None)

    invalid, unsupported = capi.LC_ERR_INVALID_ARG, capi.LC_ERR_UNSUPPORTED
    assert product(rows=0) == 0 and product(n=0) == 0
    assert product(q=None) == invalid and product(sw=None) == invalid and product(k=0) == invalid
    assert product(groups=2) == invalid and "offsets" in capi.last_error()
    assert product(groups=2, offsets=p, stride=16) == invalid
    assert product(groups=1025, offsets=p) == unsupported
    assert product(zx=p) == invalid and product(act=6) == invalid and product(variant=7) == invalid
    assert product(act=5, n=24, ldo=24) == invalid and product(dtype=capi.LC_S8) == unsupported
    assert product(ldw=40) == unsupported and product(q=p + 8) == unsupported and product(ldo=8) == invalid
    assert product(k=65552, ldq=65552, ldw=65552) == unsupported and "overflow" in capi.last_error()
    assert product(variant=capi.LC_QLINEAR_WAIT_TEST) == invalid
    assert L.lc_quantize_tokens(p, capi.LC_S8, 1, 16, 16, None, 1, 1, None, p, 16, p, None) == unsupported
    assert L.lc_quantize_tokens(p, capi.LC_F32, 2, 16, 16, None, 1, 1, None, p, 16, p, None) == invalid
    assert L.lc_quantize_tokens(p, capi.LC_F32, 1, 16, 8, None, 1, 1, None, p, 16, p, None) == invalid
    assert L.lc_route_experts(p, capi.LC_F32, 4, 8, 8, 9, 1, p, p, p, p, None, 0, None) == invalid
    assert L.lc_route_experts(p, capi.LC_F32, 4, 2000, 2000, 2, 1, p, p, p, p, None, 0, None) == unsupported
    assert L.lc_route_experts(p, capi.LC_F32, 4096, 8, 8, 2, 1, p, p, p, p, None, 0, None) == capi.LC_ERR_WORKSPACE
    assert L.lc_route_experts(p, capi.LC_F32, 4096, 8, 8, 2, 1, p, p, p, p, p + 8, 4096, None) == capi.LC_ERR_WORKSPACE
    assert L.lc_combine_experts(p, capi.LC_F32, 4, 8, 8, p, p, 2, 0, None, 0, p, 8, None) == invalid
    assert L.lc_combine_experts(p, capi.LC_U8, 4, 8, 8, p, p, 2, 2, None, 0, p, 8, None) == unsupported
    assert L.lc_expert_linear(p, capi.LC_F32, 4, 32, None, 1, None, 1, 4, p, 32, 0, 16, 32, p, None, 0, None, 0, p,
                              capi.LC_F32, 16, None, 0, None, None) == capi.LC_ERR_WORKSPACE
    assert L.lc_expert_linear(p, capi.LC_F32, 3, 32, p, 2, None, 1, 4, p, 32, 0, 16, 32, p, None, 0, None, 0, p,
                              capi.LC_F32, 16, p, 4096, None, None) == invalid
    assert L.lc_expert_linear_workspace_bytes(4, 20) == 512
