"""Mixture of SwiGLU experts with int8 weights and dynamically quantized activations: the
feed-forward block of :class:`lucid_b200.nn.quantized.WeightOnlySwiGLU` with a router in front of
it.  (The reference has no expert layers; the arithmetic of each product is its dynamic Linear's,
``lucid/nn/quantized/dynamic/linear.py:85-92``, with one activation scale per row.)
"""
from __future__ import annotations

from collections.abc import Sequence

import torch
from torch import nn

from lucid_b200 import _backend
from lucid_b200.nn.quantized.dynamic import functional as F
from lucid_b200.quantization._functional import quantize
from lucid_b200.quantization._qscheme import QDtype, per_channel_symmetric, qint8


def _quantize_rows(weight: torch.Tensor, dtype: QDtype):
    from lucid_b200.quantization.observer import PerChannelMinMaxObserver

    obs = PerChannelMinMaxObserver(ch_axis=0, qscheme=per_channel_symmetric, qdtype=dtype)
    obs(weight)
    scale, zero_point = obs.calculate_qparams()
    return quantize(weight, scale, zero_point, dtype, ch_axis=0), scale


class MoESwiGLU(nn.Module):
    """``sum_j w_j down_e(silu(gate_e(x)) * up_e(x))`` over the ``top_k`` experts a router chooses for
    each token.

    The router is a float ``nn.Linear`` without bias; ``renormalize`` chooses between weights that sum
    to one over the chosen experts and the softmax over all of them.  Gate and up rows are stored
    interleaved (blocks of eight), as :class:`WeightOnlySwiGLU` stores them, and the experts' weights
    as one tensor each: ``gate_up_int8`` [E, 2 * intermediate, hidden] and ``down_int8``
    [E, hidden, intermediate] with one scale per row.  ``hidden`` and ``intermediate`` must be
    multiples of 16 (rows on 16-byte boundaries).

    ``forward(x, residual=None, token_mask=None)``: tokens whose mask is false go to no expert; their
    result is the residual, or zero.  Inference only, like the other dynamically quantized layers."""

    def __init__(self, hidden: int, intermediate: int, num_experts: int, top_k: int, renormalize: bool = True) -> None:
        super().__init__()
        if hidden % 16 or intermediate % 16 or hidden < 16 or intermediate < 16:
            raise ValueError(f"hidden and intermediate must be multiples of 16, got {hidden} and {intermediate}")
        if not 1 <= top_k <= min(num_experts, 32) or num_experts > 1024:
            raise ValueError(f"1 <= top_k <= min(num_experts, 32) and num_experts <= 1024 are required, got "
                             f"top_k = {top_k} of {num_experts}")
        self.hidden, self.intermediate = hidden, intermediate
        self.num_experts, self.top_k, self.renormalize = num_experts, top_k, renormalize
        self.router = nn.Linear(hidden, num_experts, bias=False)
        self.router.requires_grad_(False)
        self.register_buffer("gate_up_int8", torch.zeros((num_experts, 2 * intermediate, hidden), dtype=torch.int8))
        self.register_buffer("gate_up_scale", torch.ones(num_experts, 2 * intermediate))
        self.register_buffer("down_int8", torch.zeros((num_experts, hidden, intermediate), dtype=torch.int8))
        self.register_buffer("down_scale", torch.ones(num_experts, hidden))

    @classmethod
    def from_float(cls, router: nn.Linear, gates: Sequence[nn.Linear], ups: Sequence[nn.Linear],
                   downs: Sequence[nn.Linear], top_k: int, renormalize: bool = True,
                   dtype: QDtype = qint8) -> "MoESwiGLU":
        """Quantizes the experts ``down(silu(gate(x)) * up(x))`` (no biases) row by row."""
        if not len(gates) == len(ups) == len(downs) == router.out_features:
            raise ValueError(f"{router.out_features} router outputs for {len(gates)} gate, {len(ups)} up and "
                             f"{len(downs)} down projections")
        if any(m.bias is not None for m in (router, *gates, *ups, *downs)):
            raise ValueError("MoESwiGLU has no biases")
        ops = _backend.ops()
        m = cls(gates[0].in_features, gates[0].out_features, len(gates), top_k, renormalize)
        gate_up, gate_up_scale, down, down_scale = [], [], [], []
        for g, u, d in zip(gates, ups, downs):
            (wg, sg), (wu, su), (wd, sd) = (_quantize_rows(_backend.on_cuda(l.weight.detach().float()), dtype)
                                            for l in (g, u, d))
            gate_up.append(ops.interleave_gate_up(wg, wu))
            gate_up_scale.append(ops.interleave_gate_up(sg, su))
            down.append(wd)
            down_scale.append(sd)
        m.register_buffer("gate_up_int8", torch.stack(gate_up))
        m.register_buffer("gate_up_scale", torch.stack(gate_up_scale))
        m.register_buffer("down_int8", torch.stack(down))
        m.register_buffer("down_scale", torch.stack(down_scale))
        m.router.weight = nn.Parameter(_backend.on_cuda(router.weight.detach()).clone(), requires_grad=False)
        return m

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None,
                token_mask: torch.Tensor | None = None) -> torch.Tensor:
        if x.shape[-1] != self.hidden:
            raise ValueError(f"input of shape {tuple(x.shape)} does not have {self.hidden} features")
        if residual is not None and residual.shape != x.shape:
            raise ValueError(f"residual has shape {tuple(residual.shape)}, expected {tuple(x.shape)}")
        if token_mask is not None and token_mask.shape != x.shape[:-1]:
            raise ValueError(f"token_mask has shape {tuple(token_mask.shape)}, expected {tuple(x.shape[:-1])}")
        xd = _backend.on_cuda(x)
        x2 = xd.reshape(-1, self.hidden)
        logits = nn.functional.linear(x2, self.router.weight.to(device=x2.device, dtype=x2.dtype)).float()
        if token_mask is not None:
            keep = token_mask.to(x2.device).reshape(-1, 1).bool()
            logits = logits.masked_fill(~keep, float("-inf"))
        routing = F.route_experts(logits, self.top_k, renormalize=self.renormalize)
        h = F.expert_linear(x2, _backend.on_cuda(self.gate_up_int8), _backend.on_cuda(self.gate_up_scale), routing,
                            activation="swiglu")
        y = F.expert_linear(h, _backend.on_cuda(self.down_int8), _backend.on_cuda(self.down_scale), routing,
                            sorted_rows=True)
        if residual is not None:
            residual = residual.to(device=x2.device, dtype=y.dtype).reshape(-1, self.hidden)
        out = F.combine_experts(y, routing, residual=residual).reshape(xd.shape)
        return out if x.is_cuda else out.to(x.device)

    def extra_repr(self) -> str:
        return (f"hidden={self.hidden}, intermediate={self.intermediate}, num_experts={self.num_experts}, "
                f"top_k={self.top_k}, renormalize={self.renormalize}, dynamic=True")
