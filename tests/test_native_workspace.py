"""Workspace sizes of the K3-native block by its static weights' kinds (CPU)."""
import ctypes

import pytest

from moonshine_amd import _lib
from moonshine_amd._lib import K3MoeNativeShape, K3MoeNativeWeights, K3MoeStaticWeight
from moonshine_amd.native import K3_NATIVE_LAYER, STATIC_BF16, STATIC_FP8, STATIC_Q8, routed_shape

CFG = K3_NATIVE_LAYER
SHAPE = K3MoeNativeShape(routed_shape(CFG), CFG.hidden, CFG.shared, CFG.eps)
SIZES = dict(routed_down=(CFG.latent, CFG.hidden), routed_up=(CFG.hidden, CFG.latent),
             shared_gate=(CFG.shared, CFG.hidden), shared_up=(CFG.shared, CFG.hidden),
             shared_down=(CFG.hidden, CFG.shared))
SIDE = ("routed_down", "shared_gate", "shared_up")
TOKENS = (1, 2, 5, 8, 16, 64, 512, 4096, 65535)


def weights(kinds):
    w = K3MoeNativeWeights()
    for name, (rows, cols) in SIZES.items():
        setattr(w, name, K3MoeStaticWeight(kinds.get(name, STATIC_Q8), rows, cols, None, None))
    return w


def plain(tokens):
    return _lib.lib().k3_moe_native_workspace_bytes(ctypes.byref(SHAPE), tokens)


def of(kinds, tokens):
    return _lib.lib().k3_moe_native_weights_workspace_bytes(ctypes.byref(weights(kinds)), ctypes.byref(SHAPE),
                                                            tokens)


@pytest.mark.parametrize("tokens", TOKENS)
def test_no_scratch_for_weights_that_take_none(tokens):
    """The block's rows, routes, logits of up to 16 slices and its experts' workspace, as programs
    with bf16 and Q8-128 weights have held it."""
    H, D, S, E, k = CFG.hidden, CFG.latent, CFG.shared, CFG.experts, CFG.top_k
    rows = 2 * tokens * (3 * D + 3 * H + 3 * S) + 8 * tokens * k + 4 * E + 64 * tokens * E
    experts = _lib.lib().k3_moe_workspace_bytes(ctypes.byref(SHAPE.routed), tokens)
    assert experts < plain(tokens) <= experts + rows + 16 * 256
    assert of({}, tokens) == plain(tokens)
    assert of(dict.fromkeys(SIZES, STATIC_BF16), tokens) == plain(tokens)


@pytest.mark.parametrize("tokens", TOKENS)
def test_scratch_of_each_streams_fp8_weights(tokens):
    scratch = {n: _lib.lib().k3_moe_fp8_128_scratch_bytes(tokens, *SIZES[n]) for n in SIZES}
    assert all(n % 256 == 0 for n in scratch.values())
    for name in SIZES:
        assert of({name: STATIC_FP8}, tokens) == plain(tokens) + scratch[name]
    side = max(scratch[n] for n in SIDE)
    main = max(scratch[n] for n in SIZES if n not in SIDE)
    assert of(dict.fromkeys(SIZES, STATIC_FP8), tokens) == plain(tokens) + side + main
    assert of(dict.fromkeys(SIDE, STATIC_FP8), tokens) == plain(tokens) + side


def test_sizes_refuse():
    f = _lib.lib().k3_moe_native_weights_workspace_bytes
    w = weights({})
    assert f(None, ctypes.byref(SHAPE), 4) == 0 and f(ctypes.byref(w), None, 4) == 0
    assert f(ctypes.byref(w), ctypes.byref(SHAPE), 0) == 0
    assert f(ctypes.byref(w), ctypes.byref(SHAPE), 65536) == 0
