"""Scratch and stream of the FP8-128 and balance calls: in memory of exactly their size they give the
bits of a call with room to spare, and write nothing behind it."""
import ctypes

import pytest
import torch

from moonshine_amd import balance, fp8
from moonshine_amd._lib import lib
from moonshine_amd.synth import ACT_SWIGLU
from test_gpu_fp8 import make_store, normal

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


@pytest.mark.parametrize("T", [1, 2, 9, 64, 65, 300, 1024, 1025])
@pytest.mark.parametrize("E,H,F,k", [(8, 256, 384, 3), (64, 128, 128, 8), (40, 384, 256, 9)])
def test_exact_workspace_of_experts(cuda, T, E, H, F, k):
    """Any ids, in a workspace of exactly the call's size and in one for more tokens."""
    store = make_store(cuda, E, H, F, 4)
    g = torch.Generator().manual_seed(T + E)
    ids = torch.randint(-1, E + 1, (T, k), generator=g, dtype=torch.int32).to(cuda)
    w = torch.rand((T, k), generator=g).to(cuda)
    x, r = normal((T, H), T).to(cuda), normal((T, H), T + 1).to(cuda)
    sh = fp8.shape(H, E, k, F, 1.0, ACT_SWIGLU)
    want = fp8.experts(x, ids, w, store.table, sh, r)
    size = lambda t: lib().k3_moe_fp8_workspace_bytes(ctypes.byref(sh), t)  # noqa: E731
    room = torch.full((size(T + 700) + 4096,), 0xff, dtype=torch.uint8, device=cuda)
    out = torch.zeros_like(x)

    def run(n):
        return lib().k3_moe_fp8_experts_bf16(out.data_ptr(), x.data_ptr(), r.data_ptr(), ids.data_ptr(),
                                             w.data_ptr(), store.table.data_ptr(), ctypes.byref(sh), T,
                                             room.data_ptr(), n, torch.cuda.current_stream().cuda_stream)

    need = size(T)
    assert not run(need - 1)
    assert run(need)
    assert torch.equal(out, want) and (room[need:] == 0xff).all()
    out.zero_()
    assert run(size(T + 700)) and torch.equal(out, want)


@pytest.mark.parametrize("segments,length,E", [(1, 1, 1), (1, 700, 64), (3, 333, 130), (1, 4096, 896),
                                               (600, 9, 24), (40, 100, 1024)])
def test_exact_scratch_of_the_balance_loss(cuda, segments, length, E):
    T = segments * length
    logits = torch.randn((T, E), generator=torch.Generator().manual_seed(T)).to(cuda)
    ids = logits.topk(1, 1).indices.to(torch.int32)
    loss, counts, mean, live = balance.balance_loss(logits, ids, 0.4, segments=segments)
    need = lib().k3_moe_balance_scratch_bytes(segments, length, E)
    room = torch.full((need + 4096,), 0xff, dtype=torch.uint8, device=cuda)
    got = [torch.zeros_like(t) for t in (loss, counts, mean, live)]

    def run(n):
        return lib().k3_moe_balance_loss_f32(*(t.data_ptr() for t in got), logits.data_ptr(), ids.data_ptr(), None,
                                             segments, length, E, 1, 0.4, room.data_ptr(), n,
                                             torch.cuda.current_stream().cuda_stream)

    assert not run(need - 1)
    assert run(need)
    for a, b in zip(got, (loss, counts, mean, live)):
        assert torch.equal(a, b)
    assert (room[need:] == 0xff).all()
