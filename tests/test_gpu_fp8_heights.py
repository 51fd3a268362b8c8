"""FP8-128 experts whose last row tile is short: one row, and fewer 32-row steps than the tile's
shortest loop runs. Bounds as in tests/_fp8.py."""
import pytest
import torch

from moonshine_amd.synth import ACT_SITU, ACT_SWIGLU
from test_gpu_fp8 import check_experts, make_store

pytestmark = pytest.mark.gpu


def height(n):
    many = -(-n // 256)
    return 32 * -(-(-(-n // 32)) // many) if n > 128 else n


@pytest.mark.parametrize("rows,last", [(1344, 224), (1345, 65), (1537, 193), (1761, 225), (1793, 1), (1824, 32),
                                       (1857, 65), (2049, 1)])
@pytest.mark.parametrize("act", [ACT_SWIGLU, ACT_SITU])
def test_short_last_tiles(cuda, rows, last, act):
    """`rows` tokens at expert 1, none or an invalid id beside it."""
    assert rows - height(rows) * (-(-rows // height(rows)) - 1) == last
    store = make_store(cuda, 3, 128, 256, 3)
    ids = torch.full((rows, 2), 1, dtype=torch.int32)
    ids[:, 1] = 3
    ids[: rows // 40, 1] = 2
    check_experts(cuda, store, rows, 2, act, rows, ids=ids, residual=act == ACT_SITU)
