"""The router in training, on torch tensors (include/k3_moe.h has the formulas).

balance_loss gives the balance loss of a batch with its per-expert counts and
mean scores; router_backward the gradient of that loss, and of the route
weights, by the router's logits. torch is used only for device memory and
streams; each call takes its scratch from torch's allocator for itself.
"""
import torch

from ._lib import lib
from .fp8 import _dense, _need, _On, _scratch


def _batch(logits, ids, segments, mask):
    """(T, E, k, length) of checked arguments."""
    _dense(logits, "logits", (torch.float32,), 2)
    _dense(ids, "ids", (torch.int32,), 2, logits.device)
    T, E = logits.shape
    _need(ids.shape[0] == T, f"ids: {ids.shape[0]} rows, {T} tokens")
    _need(segments > 0 and T > 0 and T % segments == 0, f"{T} tokens are not {segments} equal segments")
    if mask is not None:
        _dense(mask, "mask", (torch.uint8, torch.bool), 1, logits.device)
        _need(mask.shape[0] == T, f"mask: {mask.shape[0]} tokens, wanted {T}")
    return T, E, ids.shape[1], T // segments


def balance_loss(logits, ids, coefficient, segments=1, mask=None):
    """logits f32 [T, E], ids int32 [T, k] -> (loss [], counts int32 [segments, E], mean_scores
    f32 [segments, E], live_tokens int32 [segments]). T is `segments` sequences of one length;
    mask (uint8 or bool [T]) marks the live tokens of a padded batch."""
    T, E, k, length = _batch(logits, ids, segments, mask)
    new = lambda shape, dtype: torch.empty(shape, dtype=dtype, device=logits.device)  # noqa: E731
    loss, counts = new((), torch.float32), new((segments, E), torch.int32)
    mean, live = new((segments, E), torch.float32), new((segments,), torch.int32)
    L = lib()
    n = L.k3_moe_balance_scratch_bytes(segments, length, E)
    keep, at = _scratch(n, logits.device)
    with _On(logits.device) as st:
        if not L.k3_moe_balance_loss_f32(loss.data_ptr(), counts.data_ptr(), mean.data_ptr(),
                                         live.data_ptr(), logits.data_ptr(), ids.data_ptr(),
                                         None if mask is None else mask.data_ptr(), segments, length,
                                         E, k, coefficient, at, n, st):
            raise RuntimeError("k3_moe_balance_loss_f32 rejected its arguments or failed to launch")
    return loss, counts, mean, live


def router_backward(logits, ids, counts, live_tokens, coefficient, segments=1, mask=None,
                    dloss=None, dweights=None, scaling_factor=1.0, out=None):
    """The gradient by the logits, f32 [T, E]: of dloss (f32 [] on the device, or None for 1) times
    the loss, plus that of the route weights (scores of the ids, renormalized, times
    scaling_factor) with gradient dweights f32 [T, k], or None for the loss alone."""
    T, E, k, length = _batch(logits, ids, segments, mask)
    for t, name, shape in ((counts, "counts", (segments, E)), (live_tokens, "live_tokens", (segments,))):
        _dense(t, name, (torch.int32,), len(shape), logits.device)
        _need(t.shape == shape, f"{name}: {tuple(t.shape)}, wanted {shape}")
    if dloss is not None:
        _dense(dloss, "dloss", (torch.float32,), 0, logits.device)
    if dweights is not None:
        _dense(dweights, "dweights", (torch.float32,), 2, logits.device)
        _need(dweights.shape == (T, k), f"dweights: {tuple(dweights.shape)}, wanted {(T, k)}")
    if out is None:
        out = torch.empty_like(logits)
    else:
        _dense(out, "out", (torch.float32,), 2, logits.device)
        _need(out.shape == logits.shape, f"out: {tuple(out.shape)}, wanted {tuple(logits.shape)}")
    with _On(logits.device) as st:
        if not lib().k3_moe_router_backward_f32(
                out.data_ptr(), logits.data_ptr(), ids.data_ptr(), counts.data_ptr(),
                live_tokens.data_ptr(), None if mask is None else mask.data_ptr(),
                None if dloss is None else dloss.data_ptr(),
                None if dweights is None else dweights.data_ptr(), segments, length, E, k,
                coefficient, scaling_factor, st):
            raise RuntimeError("k3_moe_router_backward_f32 rejected its arguments or failed to launch")
    return out


__all__ = ["balance_loss", "router_backward"]
