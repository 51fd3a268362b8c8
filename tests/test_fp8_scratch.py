"""Scratch of the FP8-128 product (CPU): the encoded rows, and room for parts of K only where K
can be cut."""
import pytest

from moonshine_amd import _lib

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
    for rows in (1, 130, 256, 1030, 4096, 7168, 50000, 1 << 24):
        for cols in (128, 640, 1664, 2176, 4096, 8192, 65536, 1 << 24):
            sizes = [scratch(t, rows, cols) for t in steps]
            assert sizes == sorted(sizes), (rows, cols)
