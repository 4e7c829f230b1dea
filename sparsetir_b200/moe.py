"""A mixture-of-experts layer over the library's operators: the relational product
``y = sum over relations r of A_r x W_r`` with the experts as relations and with ``A`` made on the GPU in every call.

    p = softmax(x router^T),  y[t] = sum over the top_k experts e of token t of  p[t, e] * expert_e(x[t])
    expert_e(x) = (silu(x gate_e^T) * (x up_e^T)) down_e^T

``ExpertLayer`` holds the weights; ``forward`` returns the result and what ``backward`` needs, ``backward`` the gradients of the
input and of all weights, each from the library's own operator.  ``QuantizedExpertLayer`` is the same layer for serving with
weights and activations in 8-bit integers.  Everything runs on torch's current stream, nothing is read back to the host:
how many tokens an expert has is known on the device alone, so that a step can be captured into a CUDA graph.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, Optional, Tuple

import torch
import torch.nn.functional as F

from . import ops


@dataclass
class Routing:
    """Which rows of the experts' order the pairs (token, choice) have (``ops.moe_route``)."""

    logits: torch.Tensor   # [tokens, experts] float32
    gates: torch.Tensor    # [tokens, top_k] float32
    experts: torch.Tensor  # [tokens, top_k] int32, -1: none
    slots: torch.Tensor    # [tokens, top_k] int32, -1: none
    indptr: torch.Tensor   # [experts + 1] int32


@dataclass
class Saved:
    """What a forward pass leaves for the backward pass."""

    x: torch.Tensor
    routing: Routing
    rows: torch.Tensor    # the tokens' rows in the experts' order
    hidden: torch.Tensor  # [pairs, 2 * width]: gate and up projections
    act: torch.Tensor     # silu(gate) * up
    out: torch.Tensor     # the experts' results


def route(logits: torch.Tensor, top_k: int, renormalize: bool = False) -> Routing:
    tokens, experts = logits.shape
    dev = logits.device
    gates = torch.empty(tokens, top_k, device=dev)
    chosen, slots = (torch.empty(tokens, top_k, dtype=torch.int32, device=dev) for _ in range(2))
    indptr = torch.empty(experts + 1, dtype=torch.int32, device=dev)
    ops.moe_route(logits.view(-1), gates.view(-1), chosen.view(-1), slots.view(-1), indptr, experts, top_k,
                  ops.MOE_RENORMALIZE if renormalize else 0)
    return Routing(logits, gates, chosen, slots, indptr)


class _Layer:
    def _logits(self, x: torch.Tensor, padding: Optional[torch.Tensor]) -> torch.Tensor:
        if x.dim() != 2 or x.shape[1] != self.features or not x.is_contiguous():
            raise ValueError(f"x must be a contiguous [tokens, {self.features}] tensor")
        logits = x.float() @ self.router.float().t()
        if padding is not None:  # tokens that no expert takes
            logits.masked_fill_(padding[:, None], float("-inf"))
        return logits


class ExpertLayer(_Layer):
    """``router [experts, features]``, ``gate_up [experts, 2 * width, features]`` (the gate projection's rows first), ``down
    [experts, features, width]``; ``gate_up`` and ``down`` in float16 or bfloat16."""

    def __init__(self, router: torch.Tensor, gate_up: torch.Tensor, down: torch.Tensor, top_k: int, renormalize: bool = False):
        self.experts, self.features = router.shape
        self.width = down.shape[2]
        if tuple(gate_up.shape) != (self.experts, 2 * self.width, self.features) or tuple(down.shape) != (self.experts, self.features, self.width):
            raise ValueError("gate_up must be [experts, 2 * width, features] and down [experts, features, width]")
        self.router, self.gate_up, self.down = router, gate_up.contiguous(), down.contiguous()
        self.top_k, self.renormalize = top_k, renormalize

    def _product(self, x: torch.Tensor, w: torch.Tensor, indptr: torch.Tensor, transposed: bool) -> torch.Tensor:
        """x times every expert's ``w[e]^T`` (its layout is [out, in]), or times ``w[e]``: the gradient's product."""
        fo, fi = (w.shape[2], w.shape[1]) if transposed else (w.shape[1], w.shape[2])
        y = torch.empty(x.shape[0], fo, dtype=x.dtype, device=x.device)
        ops.grouped_mm(x.view(-1), w.view(-1), y.view(-1), indptr, self.experts, fi, fo, 0 if transposed else ops.GROUPED_W_OUT_IN)
        return y

    def _weight_grad(self, x: torch.Tensor, dy: torch.Tensor, w: torch.Tensor, indptr: torch.Tensor) -> torch.Tensor:
        dw = torch.empty_like(w)
        ops.grouped_mm_grad_w(x.view(-1), dy.view(-1), dw.view(-1), indptr, self.experts, w.shape[2], w.shape[1], ops.GROUPED_W_OUT_IN)
        return dw

    def forward(self, x: torch.Tensor, padding: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Saved]:
        r = route(self._logits(x, padding), self.top_k, self.renormalize)
        rows = torch.empty(x.shape[0] * self.top_k, self.features, dtype=x.dtype, device=x.device)
        ops.moe_dispatch(x.view(-1), r.slots.view(-1), rows.view(-1), self.features, self.top_k)
        hidden = self._product(rows, self.gate_up, r.indptr, False)
        # rounded to 16 bits behind silu and behind the product: in 32 bits the two would take three more passes over [pairs, width]
        act = F.silu(hidden[:, :self.width]) * hidden[:, self.width:]
        out = self._product(act, self.down, r.indptr, False)
        y = torch.empty_like(x)
        ops.moe_combine(out.view(-1), r.slots.view(-1), r.gates.view(-1), y.view(-1), self.features, self.top_k)
        return y, Saved(x, r, rows, hidden, act, out)

    def backward(self, dy: torch.Tensor, s: Saved) -> Dict[str, torch.Tensor]:
        r, k = s.routing, self.top_k
        d_out, d_gates = torch.empty_like(s.out), torch.empty_like(r.gates)
        ops.moe_combine_grad(dy.contiguous().view(-1), s.out.view(-1), r.slots.view(-1), r.gates.view(-1), d_out.view(-1),
                             d_gates.view(-1), self.features, k)
        d_down = self._weight_grad(s.act, d_out, self.down, r.indptr)
        d_act = self._product(d_out, self.down, r.indptr, True)
        gate, up = s.hidden[:, :self.width].float(), s.hidden[:, self.width:].float()
        sig = torch.sigmoid(gate)
        d_hidden = torch.cat([d_act * up * sig * (1 + gate * (1 - sig)), d_act * gate * sig], 1).to(s.hidden.dtype)
        d_gate_up = self._weight_grad(s.rows, d_hidden, self.gate_up, r.indptr)
        d_rows = self._product(d_hidden, self.gate_up, r.indptr, True)
        dx = torch.empty(s.x.shape, device=s.x.device)
        ops.moe_combine(d_rows.view(-1), r.slots.view(-1), None, dx.view(-1), self.features, k)
        d_logits = torch.empty_like(r.logits)
        ops.moe_route_grad(r.logits.view(-1), r.gates.view(-1), r.experts.view(-1), d_gates.view(-1), d_logits.view(-1), self.experts,
                           k, ops.MOE_RENORMALIZE if self.renormalize else 0)
        dx += d_logits @ self.router.float()
        return {"x": dx.to(s.x.dtype), "router": d_logits.t() @ s.x.float(), "gate_up": d_gate_up, "down": d_down}

    def __call__(self, x: torch.Tensor, padding: Optional[torch.Tensor] = None) -> torch.Tensor:
        return self.forward(x, padding)[0]

    def quantized(self) -> "QuantizedExpertLayer":
        return QuantizedExpertLayer(self)


def quantize_channels(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Weights [..., out, in] as 8-bit integers with a scale for every output channel."""
    scale = w.float().abs().amax(-1) / 127
    q = torch.round(w.float() / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None])
    return q.to(torch.int8), scale


class QuantizedExpertLayer(_Layer):
    """An ``ExpertLayer`` for serving: weights in 8-bit integers with a scale for every output channel, activations
    quantised on the way with a scale for every row."""

    def __init__(self, layer: ExpertLayer):
        self.router, self.top_k, self.renormalize = layer.router, layer.top_k, layer.renormalize
        self.experts, self.features, self.width = layer.experts, layer.features, layer.width
        self.gate_up, self.gate_up_scale = quantize_channels(layer.gate_up)
        self.down, self.down_scale = quantize_channels(layer.down)

    def _product(self, x: torch.Tensor, slots: Optional[torch.Tensor], rows: int, w: torch.Tensor, w_scale: torch.Tensor,
                 indptr: torch.Tensor) -> torch.Tensor:
        fo, fi = w.shape[1:]
        q, scale = torch.empty(rows, fi, dtype=torch.int8, device=x.device), torch.empty(rows, device=x.device)
        ops.moe_dispatch_i8(x.view(-1), slots, q.view(-1), scale, fi, 1 if slots is None else self.top_k)
        y = torch.empty(rows, fo, dtype=x.dtype, device=x.device)
        ops.grouped_mm_i8(q.view(-1), scale, w.view(-1), w_scale.view(-1), y.view(-1), indptr, self.experts, fi, fo)
        return y

    def __call__(self, x: torch.Tensor, padding: Optional[torch.Tensor] = None) -> torch.Tensor:
        r = route(self._logits(x, padding), self.top_k, self.renormalize)
        pairs = x.shape[0] * self.top_k
        hidden = self._product(x, r.slots.view(-1), pairs, self.gate_up, self.gate_up_scale, r.indptr)
        act = F.silu(hidden[:, :self.width]) * hidden[:, self.width:]
        out = self._product(act, None, pairs, self.down, self.down_scale, r.indptr)
        y = torch.empty_like(x)
        ops.moe_combine(out.view(-1), r.slots.view(-1), r.gates.view(-1), y.view(-1), self.features, self.top_k)
        return y
