"""bf16 products grouped by expert, on torch tensors, and their gradients.

route_plan sorts a batch's routes by expert; product multiplies each expert's rows
with its weights, input_gradient and weight_gradient are its gradients by the rows
and by the weights (include/k3_moe.h has the definitions). torch is used only for
device memory and streams. Autograd does not see these calls: an input that
requires a gradient is refused while gradients are recorded; in an
autograd.Function, product goes in forward and the gradients in backward.

Rows past the last expert's, and rows of an output that `to` sends nothing to, are
left as they were: of an output made here they hold whatever its memory did. Of no rows
at all, outputs are empty and a weight gradient zeros (added up, out as it was), without a
call of the library.
"""
from dataclasses import dataclass

import torch

from ._lib import lib
from .fp8 import _BF16, _F32, _I32, _call, _dense, _scratch

MOST_PICKED = 65535


@dataclass(frozen=True)
class RoutePlan:
    """A batch's routes sorted by expert, stable: row r of the plan is route route_index[r] (token *
    top_k + rank), of token token_index[r], and expert e has rows offsets[e] up to offsets[e + 1].
    Routes of no expert, and a token's repeated ones, have no row: offsets[experts] rows are in
    use. All int32 on the device; ids are the routes themselves, [T, top_k]."""

    ids: torch.Tensor
    experts: int
    counts: torch.Tensor
    offsets: torch.Tensor
    token_index: torch.Tensor
    route_index: torch.Tensor


def route_plan(ids, experts):
    """ids int32 [T, top_k] -> RoutePlan."""
    at = _dense(ids, "ids", _I32, 2)
    T, k = ids.shape
    L, device = lib(), ids.get_device()
    if T == 0 or T > 65535 or k == 0 or k > 32 or not 0 < experts <= 1024:
        raise ValueError(f"ids {tuple(ids.shape)} of {experts} experts")
    n = L.k3_moe_plan_scratch_bytes(T, experts)
    counts, offsets, unique = (ids.new_empty((m,)) for m in (experts, experts + 1, experts))
    summary, token, route = ids.new_empty((4,)), ids.new_empty((T * k,)), ids.new_empty((T * k,))
    keep, room = _scratch(ids, n)
    _call(L.k3_moe_route_plan, device, counts.data_ptr(), offsets.data_ptr(), unique.data_ptr(),
          summary.data_ptr(), token.data_ptr(), route.data_ptr(), at, T, k, experts, room, n)
    return RoutePlan(ids, experts, counts, offsets, token, route)


def no_routes(ids, experts):
    """The plan of no token's routes, ids int32 [0, top_k]."""
    _dense(ids, "ids", _I32, 2)
    none = ids.new_empty((0,))
    return RoutePlan(ids, experts, ids.new_zeros((experts,)), ids.new_zeros((experts + 1,)), none, none)


def _index(t, name, device):
    return None if t is None else _dense(t, name, _I32, 1, device)


def _rows(name, have, index, index_name):
    """Rows of the product by a tensor of `have` rows and an index (or None) of it."""
    if index is None:
        return have
    if index.shape[0] == 0:
        return 0
    if not 0 < have <= MOST_PICKED:
        raise ValueError(f"{name}: {have} rows; {index_name} picks from 1 to {MOST_PICKED}")
    return index.shape[0]


def _experts(offsets, E, device):
    at = _dense(offsets, "offsets", _I32, 1, device)
    if offsets.shape[0] != E + 1:
        raise ValueError(f"offsets: {offsets.shape[0]}, wanted {E + 1}")
    return at


def _by_rows(fn, rows, name, weights, inner, outer, offsets, index, to, out):
    """product and input_gradient: rows [., weights.shape[inner]] -> [., weights.shape[outer]]."""
    at = _dense(rows, name, _BF16, 2)
    device = rows.get_device()
    w = _dense(weights, "weights", _BF16, 3, device)
    E, N, K = weights.shape
    o = _experts(offsets, E, device)
    i, t = _index(index, "index", device), _index(to, "to", device)
    if rows.shape[1] != weights.shape[inner]:
        raise ValueError(f"{name}: {rows.shape[1]} wide, weights {tuple(weights.shape)}")
    R = _rows(name, rows.shape[0], index, "index")
    if to is not None and to.shape[0] != R:
        raise ValueError(f"to: {to.shape[0]} rows, wanted {R}")
    width = weights.shape[outer]
    if out is None:
        out = rows.new_empty((R, width))
        dst = out.data_ptr()
    else:
        dst = _dense(out, "out", _BF16, 2, device)
        if out.shape[1] != width or (to is None and out.shape[0] < R):
            raise ValueError(f"out: {tuple(out.shape)}, wanted {(R, width)}")
    if R != 0:
        _call(fn, device, dst, at, w, o, i, t, R, rows.shape[0], out.shape[0], E, N, K)
    return out


def product(x, weights, offsets, index=None, to=None, out=None):
    """x bf16 [., K] times weights bf16 [E, N, K] -> bf16 [R, N]: row r, of the expert whose rows hold
    it by offsets (int32 [E + 1]), is weights[e] x[index[r]], written at to[r]. index and to (int32
    [R]): x's and the output's rows as they lie where None."""
    return _by_rows(lib().k3_moe_grouped_product_bf16, x, "x", weights, 2, 1, offsets, index, to, out)


def input_gradient(dy, weights, offsets, index=None, to=None, out=None):
    """The gradient of product by its rows: dy bf16 [., N] -> bf16 [R, K]; dy[index[r]] is the
    gradient of row r, whose own is written at to[r]."""
    return _by_rows(lib().k3_moe_grouped_input_gradient_bf16, dy, "dy", weights, 1, 2, offsets, index, to,
                    out)


def weight_gradient(dy, x, offsets, dy_index=None, x_index=None, dtype=torch.float32, out=None,
                    accumulate=False):
    """The gradient of product by its weights: dy bf16 [., N], x bf16 [., K] -> [E, N, K] of dtype
    (float32 or bfloat16). accumulate adds to out, a float32 gradient of earlier batches."""
    at = _dense(dy, "dy", _BF16, 2)
    device = dy.get_device()
    src = _dense(x, "x", _BF16, 2, device)
    if dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"dtype: {dtype}, float32 or bfloat16 is wanted")
    if not isinstance(offsets, torch.Tensor) or offsets.dim() != 1 or offsets.shape[0] < 2:
        raise ValueError("offsets: [experts + 1] is wanted")
    E, N, K = offsets.shape[0] - 1, dy.shape[1], x.shape[1]
    o = _experts(offsets, E, device)
    i, j = _index(dy_index, "dy_index", device), _index(x_index, "x_index", device)
    R = _rows("dy", dy.shape[0], dy_index, "dy_index")
    if _rows("x", x.shape[0], x_index, "x_index") != R:
        raise ValueError(f"dy has {R} rows, x {x.shape[0] if x_index is None else x_index.shape[0]}")
    if out is None:
        if accumulate:
            raise ValueError("accumulate wants an out to add to")
        out = dy.new_empty((E, N, K), dtype=dtype)
        dst = out.data_ptr()
    else:
        dst = _dense(out, "out", (dtype,), 3, device)
        if out.shape != (E, N, K):
            raise ValueError(f"out: {tuple(out.shape)}, wanted {(E, N, K)}")
    if accumulate and dtype != torch.float32:
        raise ValueError("accumulate: a float32 out is wanted")
    if R == 0:
        return out if accumulate else out.zero_()
    _call(lib().k3_moe_grouped_weight_gradient_bf16, device, dst, dtype == torch.float32, accumulate, at, src,
          o, i, j, R, dy.shape[0], x.shape[0], E, N, K)
    return out


__all__ = ["RoutePlan", "route_plan", "no_routes", "product", "input_gradient", "weight_gradient"]
