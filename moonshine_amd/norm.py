"""RMS norm with the residual's addition, on torch tensors, and its gradient.

residual_norm gives the sum (the next residual), its normed rows in bf16 and, where
asked for, in FP8-128 for fp8.product_encoded; residual_norm_backward the gradient
by the sum and by the norm's weight (include/k3_moe.h has the formulas). torch is
used only for device memory and streams. Autograd does not see these calls: an
input that requires a gradient is refused while gradients are recorded; in an
autograd.Function, residual_norm goes in forward and the gradient in backward. Of no rows,
outputs are empty and the weight's gradient zeros.
"""
from typing import NamedTuple, Optional

import torch

from ._lib import lib
from .fp8 import _BF16, _F32, BLOCK, _call, _dense, _scratch


class Normed(NamedTuple):
    """total bf16 [rows, cols] (x itself without a residual); rstd f32 [rows]; normed bf16 [rows,
    cols], and codes float8_e4m3fn [rows, cols] with scales f32 [rows, cols / 128]: None where not
    asked for."""

    total: torch.Tensor
    rstd: torch.Tensor
    normed: Optional[torch.Tensor]
    codes: Optional[torch.Tensor]
    scales: Optional[torch.Tensor]


def _like(t, name, like, device):
    at = _dense(t, name, _BF16, 2, device)
    if t.shape != like.shape:
        raise ValueError(f"{name}: {tuple(t.shape)}, wanted {tuple(like.shape)}")
    return at


def _weight(weight, cols, device):
    at = _dense(weight, "weight", _BF16, 1, device)
    if weight.shape[0] != cols:
        raise ValueError(f"weight: {weight.shape[0]}, wanted {cols}")
    return at


def residual_norm(x, weight, epsilon, residual=None, normed=True, encode=False, total=None):
    """x, residual bf16 [rows, cols], weight bf16 [cols] -> Normed. normed and encode say in which forms
    the rows are wanted; total, if given, receives the sum and may be x or residual itself."""
    at = _dense(x, "x", _BF16, 2)
    device = x.get_device()
    rows, cols = x.shape
    w = _weight(weight, cols, device)
    r = t = n = c = s = None
    if residual is not None:
        r = _like(residual, "residual", x, device)
        if total is None:
            total = x.new_empty(x.shape)
            t = total.data_ptr()
        else:
            t = _like(total, "total", x, device)
    elif total is not None:
        raise ValueError("total: without a residual the sum is x itself")
    if encode and cols % BLOCK != 0:
        raise ValueError(f"x: {cols} columns, blocks of {BLOCK} are wanted")
    out = codes = scales = None
    if normed:
        out = x.new_empty(x.shape)
        n = out.data_ptr()
    if encode:
        codes = x.new_empty(x.shape, dtype=torch.float8_e4m3fn)
        scales = x.new_empty((rows, cols // BLOCK), dtype=torch.float32)
        c, s = codes.data_ptr(), scales.data_ptr()
    rstd = x.new_empty((rows,), dtype=torch.float32)
    if rows != 0:
        _call(lib().k3_moe_residual_norm_bf16, device, t, n, c, s, rstd.data_ptr(), at, r, w, rows, cols, epsilon)
    return Normed(x if residual is None else total, rstd, out, codes, scales)


def residual_norm_backward(dnormed, total, weight, rstd, dtotal=None, out=None):
    """(gradient bf16 [rows, cols] by the sum, which is x's and the residual's; gradient f32 [cols] by
    weight). dtotal is the sum's gradient from elsewhere; out may be dnormed, total or dtotal itself."""
    at = _dense(dnormed, "dnormed", _BF16, 2)
    device = dnormed.get_device()
    rows, cols = dnormed.shape
    s, w = _like(total, "total", dnormed, device), _weight(weight, cols, device)
    r = _dense(rstd, "rstd", _F32, 1, device)
    if rstd.shape[0] != rows:
        raise ValueError(f"rstd: {rstd.shape[0]} rows, wanted {rows}")
    d = None if dtotal is None else _like(dtotal, "dtotal", dnormed, device)
    if out is None:
        out = dnormed.new_empty(dnormed.shape)
        to = out.data_ptr()
    else:
        to = _like(out, "out", dnormed, device)
    dweight = dnormed.new_empty((cols,), dtype=torch.float32)
    if rows == 0:
        return out, dweight.zero_()
    L = lib()
    n = L.k3_moe_residual_norm_scratch_bytes(rows, cols)
    keep, room = _scratch(dnormed, n)
    _call(L.k3_moe_residual_norm_backward_bf16, device, to, dweight.data_ptr(), at, s, w, r, d, rows, cols, room,
          n)
    return out, dweight


__all__ = ["Normed", "residual_norm", "residual_norm_backward"]
