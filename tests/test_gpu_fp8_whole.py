"""FP8-128 experts as a whole against the 64-bit form, without a residual: beside one that is far larger
than the experts' sum, an error of the whole stage is lost in a norm. The bounds of tests/_fp8.py are
worst cases per element; here the norm of the difference is held to 0.02 of the experts' own sum. The form
has the kernels' codes, but for activations next to a tie, so bf16's steps are what is left: two roundings
of 2^-8 at most each, 0.008."""
import pytest
import torch

from moonshine_amd.synth import ACT_SITU, ACT_SWIGLU
from test_gpu_fp8 import check_experts, make_store

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 2, 70, 256, 1025])
@pytest.mark.parametrize("E,H,F,k", [(6, 128, 128, 4), (64, 128, 128, 8), (8, 256, 384, 3), (16, 1024, 512, 4)])
def test_routes_of_the_router(cuda, T, E, H, F, k):
    check_experts(cuda, make_store(cuda, E, H, F, 4), T, k, ACT_SITU, T + E, residual=False)


@pytest.mark.parametrize("T", [255, 300, 1024, 1025])
@pytest.mark.parametrize("E,k", [(6, 4), (40, 32), (1024, 3)])
def test_any_ids(cuda, T, E, k):
    ids = torch.randint(-1, E + 1, (T, k), generator=torch.Generator().manual_seed(T + E), dtype=torch.int32)
    ids[3] = E
    check_experts(cuda, make_store(cuda, E, 128, 128, 4), T, k, ACT_SWIGLU, T, ids=ids, residual=False)


@pytest.mark.parametrize("rows", [31, 96, 129, 257, 385, 513, 1025])
def test_rows_of_one_expert(cuda, rows):
    ids = torch.full((rows, 3), 1, dtype=torch.int32)
    ids[:, 1:] = -5
    ids[: rows // 3, 1] = 0
    check_experts(cuda, make_store(cuda, 5, 256, 384, 3), rows, 3, ACT_SITU, rows, ids=ids, residual=False)
