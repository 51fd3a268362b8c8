"""The routed experts in training, in bf16, on torch tensors.

forward and backward run the experts of a batch on the router's routes, on weights
[experts, ., .] of one tensor each:

  gate_up [E, 2 F, H] (gate's rows, then up's), down [E, H, F]
  y[t, r]   = down_e . bf16(weights[t, r] act(gate_e . hidden[t], up_e . hidden[t]))
  output[t] = bf16(residual[t] + bf16(sum_r y[t, r]))

with gate/up, the weighted activation and y in bf16. They are the calls of
grouped.py and of gated, gated_backward and combine here, one after the other
(include/k3_moe.h has the formulas); backward's dweights go to
balance.router_backward. torch is used only for device memory and streams. Autograd
does not see these calls: an input that requires a gradient is refused while
gradients are recorded; in an autograd.Function, forward goes in forward and
backward in backward. A batch of no tokens has empty outputs and weight gradients of
zeros.
"""
from dataclasses import dataclass

import torch

from . import grouped
from ._lib import lib
from .fp8 import _BF16, _F32, _I32, _call, _dense
from .synth import ACT_SITU, ACT_SWIGLU


def _gated_args(gate_up, offsets, route_index, weights, activation):
    """(device, addresses of gate_up, offsets, route_index and weights, rows, routes, experts, F)."""
    at = _dense(gate_up, "gate_up", _BF16, 2)
    device = gate_up.get_device()
    o, i = _dense(offsets, "offsets", _I32, 1, device), _dense(route_index, "route_index", _I32, 1, device)
    w = _dense(weights, "weights", _F32, 2, device)
    R, F2 = gate_up.shape
    if F2 % 2 != 0 or route_index.shape[0] != R:
        raise ValueError(f"gate_up {tuple(gate_up.shape)}, route_index {tuple(route_index.shape)}")
    if activation not in (ACT_SITU, ACT_SWIGLU):
        raise ValueError(f"activation: {activation}")
    return device, at, o, i, w, R, weights.numel(), offsets.shape[0] - 1, F2 // 2


def gated(gate_up, offsets, route_index, weights, activation, beta=4.0, linear_beta=25.0, out=None):
    """gate_up bf16 [R, 2 F] -> bf16 [R, F]: row r's activation times weights[route_index[r]] (weights
    f32 [T, top_k], route_index int32 [R] into it). Rows from offsets' last on are left as they were."""
    device, at, o, i, w, R, routes, E, F = _gated_args(gate_up, offsets, route_index, weights, activation)
    if out is None:
        out = gate_up.new_empty((R, F))
        to = out.data_ptr()
    else:
        to = _dense(out, "out", _BF16, 2, device)
        if out.shape != (R, F):
            raise ValueError(f"out: {tuple(out.shape)}, wanted {(R, F)}")
    if R != 0:
        _call(lib().k3_moe_gated_rows_bf16, device, to, at, o, i, w, R, routes, E, F, activation, beta, linear_beta)
    return out


def gated_backward(dh, gate_up, offsets, route_index, weights, activation, beta=4.0, linear_beta=25.0,
                   out=None):
    """The gradient of gated: dh bf16 [R, F] -> (bf16 [R, 2 F] by gate_up, f32 [T, top_k] by weights; 0
    for a route without a row). out may be gate_up itself."""
    device, at, o, i, w, R, routes, E, F = _gated_args(gate_up, offsets, route_index, weights, activation)
    d = _dense(dh, "dh", _BF16, 2, device)
    if dh.shape != (R, F):
        raise ValueError(f"dh: {tuple(dh.shape)}, wanted {(R, F)}")
    if out is None:
        out = gate_up.new_empty(gate_up.shape)
        to = out.data_ptr()
    else:
        to = _dense(out, "out", _BF16, 2, device)
        if out.shape != gate_up.shape:
            raise ValueError(f"out: {tuple(out.shape)}, wanted {tuple(gate_up.shape)}")
    dweights = weights.new_empty(weights.shape)
    if R == 0:
        return out, dweights.zero_()
    _call(lib().k3_moe_gated_rows_backward_bf16, device, to, dweights.data_ptr(), d, at, o, i, w, R, routes, E, F,
          activation, beta, linear_beta)
    return out, dweights


def combine(rows, ids, experts, residual=None, weights=None, out=None):
    """rows bf16 [T top_k, H] in route order -> bf16 [T, H]: a token's rows, times weights (f32 [T, top_k]) if
    given, added up, and the residual. Routes of no expert and repeated ones are left out. out may be
    residual itself."""
    at = _dense(rows, "rows", _BF16, 2)
    device = rows.get_device()
    i = _dense(ids, "ids", _I32, 2, device)
    (T, k), H = ids.shape, rows.shape[1]
    if rows.shape[0] != T * k:
        raise ValueError(f"rows: {rows.shape[0]}, wanted {T * k}")
    w = r = None
    if weights is not None:
        w = _dense(weights, "weights", _F32, 2, device)
        if weights.shape != ids.shape:
            raise ValueError(f"weights: {tuple(weights.shape)}, wanted {tuple(ids.shape)}")
    if residual is not None:
        r = _dense(residual, "residual", _BF16, 2, device)
        if residual.shape != (T, H):
            raise ValueError(f"residual: {tuple(residual.shape)}, wanted {(T, H)}")
    if out is None:
        out = rows.new_empty((T, H))
        to = out.data_ptr()
    else:
        to = _dense(out, "out", _BF16, 2, device)
        if out.shape != (T, H):
            raise ValueError(f"out: {tuple(out.shape)}, wanted {(T, H)}")
    if T != 0:
        _call(lib().k3_moe_combine_bf16, device, to, at, r, i, w, T, k, experts, H)
    return out


@dataclass(frozen=True)
class Saved:
    """What backward needs of a forward pass."""

    plan: grouped.RoutePlan
    hidden: torch.Tensor
    weights: torch.Tensor
    gate_up: torch.Tensor  # the rows' gate/up products
    h: torch.Tensor        # their weighted activation
    activation: int
    beta: float
    linear_beta: float


def forward(hidden, ids, weights, gate_up, down, activation, beta=4.0, linear_beta=25.0, residual=None):
    """hidden bf16 [T, H], ids int32 and weights f32 [T, top_k] -> (output bf16 [T, H], Saved)."""
    E = gate_up.shape[0]
    if down.shape != (E, gate_up.shape[2], gate_up.shape[1] // 2):
        raise ValueError(f"gate_up {tuple(gate_up.shape)}, down {tuple(down.shape)}")
    if ids.shape != weights.shape or ids.shape[0] != hidden.shape[0]:
        raise ValueError(f"hidden {tuple(hidden.shape)}, ids {tuple(ids.shape)}, weights {tuple(weights.shape)}")
    plan = grouped.route_plan(ids, E) if ids.shape[0] != 0 else grouped.no_routes(ids, E)
    gu = grouped.product(hidden, gate_up, plan.offsets, index=plan.token_index)
    h = gated(gu, plan.offsets, plan.route_index, weights, activation, beta, linear_beta)
    y = grouped.product(h, down, plan.offsets, to=plan.route_index)
    out = combine(y, ids, E, residual)
    return out, Saved(plan, hidden, weights, gu, h, activation, beta, linear_beta)


def backward(doutput, saved, gate_up, down, dgate_up=None, ddown=None):
    """doutput bf16 [T, H] -> (dhidden bf16 [T, H], dweights f32 [T, top_k], dgate_up, ddown f32 as the
    weights). dgate_up and ddown, if given, are added to. The residual's gradient is doutput."""
    s, p = saved, saved.plan
    (T, H), E, F = s.hidden.shape, p.experts, s.h.shape[1]
    device = s.hidden.get_device()
    # all before the first call: a token that doutput lacks would be a row of zeros to the plan's
    # indices, and a gradient refused late would leave the other added to
    for t, name, dtypes, shape in ((doutput, "doutput", _BF16, (T, H)), (gate_up, "gate_up", _BF16, (E, 2 * F, H)),
                                   (down, "down", _BF16, (E, H, F)), (dgate_up, "dgate_up", _F32, (E, 2 * F, H)),
                                   (ddown, "ddown", _F32, (E, H, F))):
        if t is None and dtypes is _F32:
            continue
        at = _dense(t, name, dtypes, len(shape), device)
        if t.shape != shape or at % 16 != 0:
            raise ValueError(f"{name}: {tuple(t.shape)} at {at:#x}, wanted {shape} at a multiple of 16 bytes")
    dh = grouped.input_gradient(doutput, down, p.offsets, index=p.token_index)
    ddown = grouped.weight_gradient(doutput, s.h, p.offsets, dy_index=p.token_index, out=ddown,
                                    accumulate=ddown is not None)
    dgu, dweights = gated_backward(dh, s.gate_up, p.offsets, p.route_index, s.weights, s.activation, s.beta,
                                   s.linear_beta)
    dgate_up = grouped.weight_gradient(dgu, s.hidden, p.offsets, x_index=p.token_index, out=dgate_up,
                                       accumulate=dgate_up is not None)
    rows = grouped.input_gradient(dgu, gate_up, p.offsets, to=p.route_index)
    return combine(rows, p.ids, p.experts), dweights, dgate_up, ddown


__all__ = ["gated", "gated_backward", "combine", "Saved", "forward", "backward"]
