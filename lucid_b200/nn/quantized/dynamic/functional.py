"""Functional forms of the dynamically quantized product and of what a mixture-of-experts block puts
around it.  Activations are quantized on the fly with one symmetric int8 scale per row
(``s = max(max|x| / 127.5, 1e-8)``, codes ``clamp(rint(x / s), -128, 127)``), weights are int8 codes
with one scale per output row (what ``nnqd.Linear.from_float`` stores), the products are exact in
int32, and everything after them is computed in fp32 and rounded once.

A mixture-of-experts block is four calls::

    routing = route_experts(logits, top_k)
    h = expert_linear(x, gate_up, gate_up_scale, routing, activation="swiglu")
    y = expert_linear(h, down, down_scale, routing, sorted_rows=True)
    out = combine_experts(y, routing, residual=x)

Nothing of the routing is read on the host, so the calls can be captured in a CUDA graph.  Like the
dynamically quantized layers themselves these are inference functions: results carry no gradient.
All tensors are CUDA tensors of one device; calls go to its current stream.  The reference has no
counterpart of this module (its dynamic Linear is ``lucid/nn/quantized/dynamic/linear.py:85-92``).

As in the framework's quantizer a NaN in an activation row counts as zero; an infinity makes the
row's results NaN.
"""
from __future__ import annotations

import torch

from lucid_b200 import _backend

ACTIVATIONS = (None, "relu", "gelu", "gelu_tanh", "silu", "swiglu")
_ACTIVATION_ID = {name: i for i, name in enumerate(ACTIVATIONS)}
_SWIGLU = _ACTIVATION_ID["swiglu"]
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


class ExpertRouting:
    """Which experts each token goes to, and where its rows are in expert order.

    ``weights``    [tokens, top_k] fp32: factor of each choice;
    ``experts``    [tokens, top_k] int32: the chosen experts, -1 where nothing is chosen;
    ``offsets``    [num_experts + 1] int32: expert e owns the rows ``offsets[e] .. offsets[e + 1]``;
    ``positions``  [tokens, top_k] int32: the row of each choice, -1 where nothing is chosen.

    There are ``tokens * top_k`` rows; those behind ``offsets[-1]`` belong to no expert.  Built by
    :func:`route_experts`, or from the results of another router (rows of one expert may be in any
    order, but no row may be named twice)."""

    __slots__ = ("weights", "experts", "offsets", "positions")

    def __init__(self, weights: torch.Tensor, experts: torch.Tensor, offsets: torch.Tensor, positions: torch.Tensor):
        if weights.dim() != 2 or experts.shape != weights.shape or positions.shape != weights.shape:
            raise ValueError("ExpertRouting: weights, experts and positions must share one [tokens, top_k] shape")
        if offsets.dim() != 1 or offsets.numel() < 2:
            raise ValueError("ExpertRouting: offsets must have num_experts + 1 entries")
        if weights.dtype != torch.float32:
            raise TypeError(f"ExpertRouting: weights must be float32, got {weights.dtype}")
        for name, t in (("experts", experts), ("offsets", offsets), ("positions", positions)):
            if t.dtype != torch.int32:
                raise TypeError(f"ExpertRouting: {name} must be int32, got {t.dtype}")
            if t.device != weights.device:
                raise RuntimeError(f"ExpertRouting: tensors on different devices: {weights.device} and {t.device}")
        self.weights, self.experts = weights.contiguous(), experts.contiguous()
        self.offsets, self.positions = offsets.contiguous(), positions.contiguous()

    @property
    def num_experts(self) -> int:
        return self.offsets.shape[0] - 1

    @property
    def top_k(self) -> int:
        return self.positions.shape[1]

    @property
    def tokens(self) -> int:
        return self.positions.shape[0]

    @property
    def rows(self) -> int:
        return self.positions.numel()

    def __repr__(self) -> str:
        return f"ExpertRouting(tokens={self.tokens}, top_k={self.top_k}, num_experts={self.num_experts})"


def pack_weight(codes: torch.Tensor) -> torch.Tensor:
    """The int8 codes ``[..., N, K]`` with rows on 16-byte boundaries, which is what the products read:
    ``codes`` itself when they are already, else a view into a padded copy.  Call it once per weight;
    :func:`linear` and :func:`expert_linear` make the copy on every call for a weight that needs it."""
    if codes.dtype is not torch.int8:
        raise TypeError(f"weight codes must be int8, got {codes.dtype}")
    strides = codes.stride()
    if len(strides) < 2:
        raise ValueError("weight codes must have at least two dimensions [N, K]")
    k = codes.shape[-1]
    if strides[-1] == 1 and strides[-2] >= k and not strides[-2] & 15 and codes.data_ptr() & 15 == 0:
        # (of several matrices: whole ones behind one another)
        if len(strides) == 2 or (len(strides) == 3 and not strides[0] & 15
                                 and (codes.shape[0] == 1 or strides[0] >= codes.shape[1] * strides[1])):
            return codes
    store = codes.new_zeros((*codes.shape[:-1], (k + 15) // 16 * 16))
    store[..., :k] = codes
    return store[..., :k]


def _rows(x: torch.Tensor, what: str) -> torch.Tensor:
    """``x`` as a matrix whose rows are dense (any row pitch)."""
    if x.dtype not in _FLOATS:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {x.dtype}")
    strides = x.stride()
    if len(strides) != 2:
        x = x.reshape(-1, x.shape[-1])
        strides = x.stride()
    return x if strides[1] == 1 and strides[0] >= x.shape[1] else x.contiguous()


def _vector(t: torch.Tensor, shape: tuple, name: str, device: torch.device) -> torch.Tensor:
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")
    if t.device != device:
        raise RuntimeError(f"tensors on different devices: {device} and {t.device}")
    if t.dtype is torch.float32 and t.is_contiguous():
        return t
    return t.float().contiguous()


def _residual(t: torch.Tensor, shape: tuple, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    if t.shape != shape:
        raise ValueError(f"residual has shape {tuple(t.shape)}, expected {shape}")
    if t.dtype is not dtype:
        raise TypeError(f"residual must have the result's type {dtype}, got {t.dtype}")
    if t.device != device:
        raise RuntimeError(f"tensors on different devices: {device} and {t.device}")
    return _rows(t, "residual")


def _activation(name, n: int) -> int:
    code = _ACTIVATION_ID.get(name)
    if code is None:
        raise ValueError(f"activation must be one of {ACTIVATIONS}, got {name!r}")
    if code == _SWIGLU and n % 16:
        raise ValueError("swiglu needs weight rows in interleaved blocks of 8 gate and 8 up rows "
                         f"(a multiple of 16), got {n}")
    return code


def _check_cuda(x: torch.Tensor, device: torch.device) -> None:
    if not x.is_cuda:
        raise RuntimeError("the quantized kernels take CUDA tensors only (there is no CPU fallback); "
                           f"got a tensor on {x.device}")
    if x.device != device:
        raise RuntimeError(f"tensors on different devices: {x.device} and {device}")


def _native():
    """The native forms of the ordinary calls (see ``_C/csrc/torchcall.cpp``), or None.  They return None for a call
    they do not serve -- the Python form then converts or refuses -- and an int for a failed one."""
    return getattr(_backend.ops(), "torchcall", None)


def _done(result):
    if type(result) is int:
        from lucid_b200._C import check

        check(result)
    return result


def _matrix(weight: torch.Tensor) -> tuple:
    shape = weight.shape
    if len(shape) != 2:
        raise ValueError(f"weight must be [N, K], got {tuple(shape)}")
    return shape


def _result_type(out_dtype) -> torch.dtype:
    if out_dtype not in _FLOATS:
        raise TypeError(f"out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
    return out_dtype


def linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor | None = None, *,
           activation: str | None = None, residual: torch.Tensor | None = None,
           out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``activation(x @ (weight * weight_scale)^T + bias) + residual`` with ``x`` quantized row by row.

    ``x`` [..., K] fp32, bf16 or f16; ``weight`` [N, K] int8 codes (see :func:`pack_weight`);
    ``weight_scale`` and ``bias`` [N].  ``activation``: ``None``, ``"relu"``, ``"gelu"``,
    ``"gelu_tanh"``, ``"silu"`` or ``"swiglu"`` (weight rows in interleaved blocks of 8 gate and 8 up
    rows; the result has N / 2 columns).  ``residual`` has the result's shape and is added after the
    activation.  The result has ``out_dtype`` (default: the type of ``x``), which ``residual`` must
    have too."""
    native = _native()
    if native is not None:
        y = native.product(x, weight, weight_scale, bias, _ACTIVATION_ID.get(activation, -1), residual, out_dtype, None, None)
        if y is not None:
            return _done(y)
    n, k = _matrix(weight)
    shape = x.shape
    if not shape or shape[-1] != k:
        raise ValueError(f"input of shape {tuple(shape)} does not contract with a [{n}, {k}] weight")
    device = x.device
    _check_cuda(x, weight.device)
    x2 = _rows(x, "input")
    act = _activation(activation, n)
    dtype = x.dtype if out_dtype is None else _result_type(out_dtype)
    width = n // 2 if act == _SWIGLU else n
    rows = x2.shape[0]
    if residual is not None:
        residual = _residual(residual, (rows, width) if x2 is x else (*shape[:-1], width), dtype, device)
    scale = _vector(weight_scale, (n,), "weight_scale", device)
    if bias is not None:
        bias = _vector(bias, (n,), "bias", device)
    if rows == 0 or n == 0:
        return torch.empty((*shape[:-1], width), dtype=dtype, device=device)
    y = _backend.ops().expert_linear(x2, pack_weight(weight), scale, bias, None, None, rows, act, residual, width, dtype,
                                     device)
    return y if x2 is x else y.view((*shape[:-1], width))


def route_experts(logits: torch.Tensor, top_k: int, *, renormalize: bool = True) -> ExpertRouting:
    """Router: the ``top_k`` largest of each token's ``logits`` [tokens, num_experts] (equal logits: the
    lowest expert first) with softmax weights over the chosen experts (``renormalize``) or over all of
    them, and each choice's row in the order "by expert, then by token".

    A logit of ``-inf`` or NaN is never chosen and carries no weight: a token whose row is all ``-inf``
    (padding) goes nowhere.  Logits of ``+inf`` share the weight evenly.  At most 1024 experts and a
    ``top_k`` of 32."""
    native = _native()
    if native is not None:
        made = native.route(logits, top_k, renormalize)
        if made is not None:
            routing = ExpertRouting.__new__(ExpertRouting)
            routing.weights, routing.experts, routing.offsets, routing.positions = _done(made)
            return routing
    if logits.dim() != 2:
        raise ValueError(f"logits must be [tokens, num_experts], got {tuple(logits.shape)}")
    if logits.dtype not in _FLOATS:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    count = logits.shape[1]
    if not 1 <= top_k <= min(count, 32) or count > 1024:
        raise ValueError(f"route_experts: 1 <= top_k <= min(num_experts, 32) and num_experts <= 1024 are required, "
                         f"got top_k = {top_k} of {count}")
    _check_cuda(logits, logits.device)
    routing = ExpertRouting.__new__(ExpertRouting)
    routing.weights, routing.experts, routing.offsets, routing.positions = _backend.ops().route_experts(
        logits, top_k, renormalize)
    return routing


def expert_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, routing: ExpertRouting,
                  bias: torch.Tensor | None = None, *, activation: str | None = None, sorted_rows: bool = False,
                  out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """The products of a mixture of experts: row r of the result is ``activation(row @ (weight[e] *
    weight_scale[e])^T + bias[e])`` for the expert e that owns row r (see :class:`ExpertRouting`).

    ``x`` holds the tokens, [tokens, K], or with ``sorted_rows`` one row per choice in expert order,
    [tokens * top_k, K] (the result of an earlier ``expert_linear``).  ``weight`` [E, N, K] int8 codes
    (see :func:`pack_weight`), ``weight_scale`` and ``bias`` [E, N]; ``activation`` and ``out_dtype`` as
    for :func:`linear`.  The result has ``tokens * top_k`` rows in expert order; rows that belong to no
    expert are zero, and what ``x`` holds there does not matter."""
    native = _native()
    if native is not None:
        y = native.product(x, weight, weight_scale, bias, _ACTIVATION_ID.get(activation, -1), None, out_dtype,
                           routing.rows if sorted_rows else routing.positions, routing.offsets)
        if y is not None:
            return _done(y)
    if weight.dim() != 3:
        raise ValueError(f"weight must be [num_experts, N, K], got {tuple(weight.shape)}")
    e, n, k = weight.shape
    if routing.num_experts != e:
        raise ValueError(f"routing over {routing.num_experts} experts, weights of {e}")
    if e > 1024:
        raise ValueError(f"expert_linear: at most 1024 experts, got {e}")
    rows = routing.rows
    expected = rows if sorted_rows else routing.tokens
    if x.dim() != 2 or x.shape[0] != expected or x.shape[1] != k:
        raise ValueError(f"input has shape {tuple(x.shape)}, expected ({expected}, {k})")
    device = x.device
    _check_cuda(x, weight.device)
    _check_cuda(x, routing.positions.device)
    x2 = _rows(x, "input")
    act = _activation(activation, n)
    dtype = x.dtype if out_dtype is None else _result_type(out_dtype)
    width = n // 2 if act == _SWIGLU else n
    scale = _vector(weight_scale, (e, n), "weight_scale", device)
    if bias is not None:
        bias = _vector(bias, (e, n), "bias", device)
    if rows == 0 or n == 0:
        return torch.empty((rows, width), dtype=dtype, device=device)
    return _backend.ops().expert_linear(x2, pack_weight(weight), scale, bias, None if sorted_rows else routing.positions,
                                        routing.offsets, rows, act, None, width, dtype, device)


def combine_experts(y: torch.Tensor, routing: ExpertRouting, *, residual: torch.Tensor | None = None) -> torch.Tensor:
    """Brings the experts' rows ``y`` [tokens * top_k, N] back to their tokens: ``out[t] = sum_j
    weights[t, j] * y[positions[t, j]] + residual[t]``, added in the order of j in fp32 and rounded once
    to the type of ``y``, which ``residual`` [tokens, N] must have too."""
    native = _native()
    if native is not None:
        out = native.combine(y, routing.weights, routing.positions, residual)
        if out is not None:
            return _done(out)
    if y.dim() != 2 or y.shape[0] != routing.rows:
        raise ValueError(f"y has shape {tuple(y.shape)}, expected ({routing.rows}, N)")
    device = y.device
    _check_cuda(y, routing.positions.device)
    y = _rows(y, "y")
    shape = (routing.tokens, y.shape[1])
    if residual is not None:
        residual = _residual(residual, shape, y.dtype, device)
    if shape[0] == 0 or shape[1] == 0:
        return torch.empty(shape, dtype=y.dtype, device=device)
    return _backend.ops().combine_experts(y, routing.weights, routing.positions, residual, device)


__all__ = ["ACTIVATIONS", "ExpertRouting", "pack_weight", "linear", "route_experts", "expert_linear", "combine_experts"]
