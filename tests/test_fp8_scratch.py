"""Scratch of the FP8-128 product (CPU): the encoded rows, and room for parts of K only where K
can be cut."""
import ctypes

import pytest

from moonshine_amd import _lib
from moonshine_amd._lib import K3MoeNativeShape, K3MoeNativeWeights, K3MoeShape, K3MoeStaticWeight

MIB = 1 << 20


def rows_bytes(tokens, cols):
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    return up(tokens * cols) + up(4 * tokens * ((cols // 128 + 3) // 4 * 4))


def scratch(tokens, rows, cols):
    return _lib.lib().k3_moe_fp8_128_scratch_bytes(tokens, rows, cols)


@pytest.mark.parametrize("tokens", [9, 20, 64, 300, 4096, 65535])
@pytest.mark.parametrize("cols", [128, 384, 512])
def test_no_parts_of_few_columns(tokens, cols):
    """Parts are of four blocks of 128 columns at least: up to 512 columns are one."""
    assert scratch(tokens, 65536, cols) == rows_bytes(tokens, cols)


@pytest.mark.parametrize("tokens,most", [(9, 12), (16, 12), (32, 12), (33, 24), (64, 24), (65, 32), (4096, 32)])
@pytest.mark.parametrize("rows,cols", [(7168, 7168), (6144, 7168), (20000, 16384), (1 << 24, 1 << 24)])
def test_parts_of_few_tokens(tokens, most, rows, cols):
    """768 blocks of 128 rows at most, of 32 or 64 tokens where there are no more: 12 and 24 MiB."""
    assert scratch(tokens, rows, cols) <= rows_bytes(tokens, cols) + most * MIB


@pytest.mark.parametrize("tokens", [20, 64])
def test_parts_of_few_rows(tokens):
    """16 parts of a tile of 256 rows."""
    height = 32 if tokens <= 32 else 64
    assert scratch(tokens, 256, 8192) == rows_bytes(tokens, 8192) + 4 * height * 256 * 16


def test_grows_with_the_tokens():
    steps = [*range(1, 300), *range(300, 4200, 61), 8191, 40000, 65535]
    for rows in (1, 130, 256, 1030, 4096, 7168, 50000, 1 << 22):
        for cols in (128, 640, 1664, 2176, 4096, 8192, 65536, 1 << 24):
            sizes = [scratch(t, rows, cols) for t in steps]
            assert sizes == sorted(sizes), (rows, cols)


def test_outputs_past_a_launch_are_refused_with_the_sizes():
    """2^38 outputs are the most; the size is 0 as for every size that the product refuses."""
    assert scratch(16384, 1 << 24, 128) > 0 and scratch(65535, 1 << 22, 128) > 0
    for tokens, rows in ((16385, 1 << 24), (65535, 1 << 24), (65535, (1 << 22) + 65), (32768, (1 << 23) + 1)):
        assert scratch(tokens, rows, 128) == 0, (tokens, rows)


def test_block_refuses_such_an_output_with_its_size():
    """The native block asks before its first launch, by the same rule."""
    shape = K3MoeNativeShape(K3MoeShape(512, 8, 2, 256, 1.0, 0, 1.0, 1.0), 1024, 1 << 24, 1e-5)
    w = K3MoeNativeWeights()
    for name, rows, cols in (("routed_down", 512, 1024), ("routed_up", 1024, 512),
                             ("shared_gate", 1 << 24, 1024), ("shared_up", 1 << 24, 1024),
                             ("shared_down", 1024, 1 << 24)):
        setattr(w, name, K3MoeStaticWeight(2, rows, cols, 1 << 20, 1 << 20))
    size = lambda t: _lib.lib().k3_moe_native_weights_workspace_bytes(  # noqa: E731
        ctypes.byref(w), ctypes.byref(shape), t)
    assert size(16384) > 0 and size(16385) == 0


@pytest.mark.parametrize("experts", [1, 8, 64, 128, 200, 512, 896, 1024])
def test_layer_workspace_for_more_tokens_serves_fewer(experts):
    """The router's part grows in K slices that end at 512 tiles: at each row of tiles, and everywhere."""
    for top_k, hidden, ffn in ((1, 128, 128), (8, 2048, 4096), (32, 8320, 128)):
        if top_k > experts:
            continue
        s = ctypes.byref(K3MoeShape(hidden, experts, top_k, ffn, 1.0, 0, 4.0, 25.0))
        steps = [*range(1, 2100), *range(2100, 65536, 29), *(128 * m + 1 for m in range(16, 512)), 65535]
        sizes = {t: _lib.lib().k3_moe_fp8_workspace_bytes(s, t) for t in steps}
        ordered = [sizes[t] for t in sorted(sizes)]
        assert ordered == sorted(ordered), (experts, top_k)
        for t in (1, 100, 512, 2049):
            assert sizes[t] > _lib.lib().k3_moe_router_scratch_bytes(t, experts) > 0
