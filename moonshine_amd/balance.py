"""The router in training, on torch tensors (include/k3_moe.h has the formulas).

balance_loss gives the balance loss of a batch with its per-expert counts and
mean scores; router_backward the gradient of that loss, and of the route
weights, by the router's logits. torch is used only for device memory and
streams; each call takes its scratch from torch's allocator for itself. Autograd
does not see them: logits that require a gradient are refused while gradients are
recorded, rather than a loss returned that has none. In an autograd.Function,
balance_loss goes in forward and router_backward, with dloss, in backward.
"""
import torch

from ._lib import lib
from .fp8 import _F32, _I32, _call, _dense, _scratch

_MASK = (torch.uint8, torch.bool)


def _batch(logits, ids, segments, mask):
    """(device, addresses of logits, ids and mask, T, E, k) of checked arguments."""
    x = _dense(logits, "logits", _F32, 2)
    device = logits.get_device()
    i = _dense(ids, "ids", _I32, 2, device)
    T, E = logits.shape
    if ids.shape[0] != T:
        raise ValueError(f"ids: {ids.shape[0]} rows, {T} tokens")
    if segments <= 0 or T == 0 or T % segments != 0:
        raise ValueError(f"{T} tokens are not {segments} equal segments")
    m = None
    if mask is not None:
        m = _dense(mask, "mask", _MASK, 1, device)
        if mask.shape[0] != T:
            raise ValueError(f"mask: {mask.shape[0]} tokens, wanted {T}")
    return device, x, i, m, T, E, ids.shape[1]


def balance_loss(logits, ids, coefficient, segments=1, mask=None):
    """logits f32 [T, E], ids int32 [T, k] -> (loss [], counts int32 [segments, E], mean_scores
    f32 [segments, E], live_tokens int32 [segments]). T is `segments` sequences of one length;
    mask (uint8 or bool [T]) marks the live tokens of a padded batch."""
    device, x, i, m, T, E, k = _batch(logits, ids, segments, mask)
    loss, mean = logits.new_empty(()), logits.new_empty((segments, E))
    counts, live = ids.new_empty((segments, E)), ids.new_empty((segments,))
    L = lib()
    n = L.k3_moe_balance_scratch_bytes(segments, T // segments, E)
    keep, room = _scratch(logits, n)
    _call(L.k3_moe_balance_loss_f32, device, loss.data_ptr(), counts.data_ptr(), mean.data_ptr(),
          live.data_ptr(), x, i, m, segments, T // segments, E, k, coefficient, room, n)
    return loss, counts, mean, live


def router_backward(logits, ids, counts, live_tokens, coefficient, segments=1, mask=None,
                    dloss=None, dweights=None, scaling_factor=1.0, out=None):
    """The gradient by the logits, f32 [T, E]: of dloss (f32 [] on the device, or None for 1) times
    the loss, plus that of the route weights (scores of the ids, renormalized, times
    scaling_factor) with gradient dweights f32 [T, k], or None for the loss alone. out may be
    logits itself."""
    device, x, i, m, T, E, k = _batch(logits, ids, segments, mask)
    c, n = _dense(counts, "counts", _I32, 2, device), _dense(live_tokens, "live_tokens", _I32, 1, device)
    if counts.shape != (segments, E) or live_tokens.shape != (segments,):
        raise ValueError(f"counts {tuple(counts.shape)}, live_tokens {tuple(live_tokens.shape)}, "
                         f"wanted {(segments, E)}, {(segments,)}")
    dl = None if dloss is None else _dense(dloss, "dloss", _F32, 0, device)
    dw = None
    if dweights is not None:
        dw = _dense(dweights, "dweights", _F32, 2, device)
        if dweights.shape != (T, k):
            raise ValueError(f"dweights: {tuple(dweights.shape)}, wanted {(T, k)}")
    if out is None:
        out = logits.new_empty((T, E))
        to = out.data_ptr()
    else:
        to = _dense(out, "out", _F32, 2, device)
        if out.shape != (T, E):
            raise ValueError(f"out: {tuple(out.shape)}, wanted {(T, E)}")
    _call(lib().k3_moe_router_backward_f32, device, to, x, i, c, n, m, dl, dw, segments, T // segments,
          E, k, coefficient, scaling_factor)
    return out


__all__ = ["balance_loss", "router_backward"]
