"""FP8-128 calls' scratch and stream: products in scratch of exactly their size give the bits of a
call with room to spare and write nothing behind it."""
import pytest
import torch

from moonshine_amd import fp8
from moonshine_amd._lib import lib
from test_gpu_fp8 import normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [9, 20, 32, 33, 64, 65, 128, 129, 300])
@pytest.mark.parametrize("rows,cols", [(130, 16384), (513, 4736), (4100, 2176), (1030, 640), (7168, 1152)])
def test_exact_scratch(cuda, T, rows, cols):
    x = normal((T, cols), T).to(cuda)
    codes, scales = fp8.quantize_weight(normal((rows, cols), 3, 0.02).to(cuda))
    need = lib().k3_moe_fp8_128_scratch_bytes(T, rows, cols)
    room = torch.full((need + 4096,), 0x5a, dtype=torch.uint8, device=cuda)
    out = torch.empty((T, rows), dtype=torch.bfloat16, device=cuda)

    def run(n):
        return lib().k3_moe_fp8_128_gemm_bf16(out.data_ptr(), codes.data_ptr(), scales.data_ptr(), x.data_ptr(),
                                              T, rows, cols, room.data_ptr(), n,
                                              torch.cuda.current_stream().cuda_stream)

    assert run(need)
    assert torch.equal(out, fp8.product(x, codes, scales)) and (room[need:] == 0x5a).all()
    if need > 0:
        assert not run(need - 1)


def test_public_stream_is_the_one_asked_for_directly(cuda):
    device = torch.cuda.current_device()
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            assert fp8._public_stream(device) == fp8._stream(device) == stream.cuda_stream
