"""Outputs that share memory with an input: the buffer itself where the call allows it, any other
overlap refused before a launch, neighbours allowed. (A refused call's memory is all its own, so
the call would only race.)"""
import pytest
import torch

from moonshine_amd import balance, fp8
from moonshine_amd._lib import lib
from moonshine_amd.synth import ACT_SWIGLU
from test_gpu_fp8 import layer, make_store, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [2, 40, 300])
@pytest.mark.parametrize("rows", [1, -1])
def test_experts_refuse_an_output_over_part_of_the_residual(cuda, T, rows):
    E, H, F, k = 4, 128, 128, 2
    store = make_store(cuda, E, H, F, 2)
    x = normal((T, H), 1).to(cuda)
    ids = torch.arange(k, dtype=torch.int32, device=cuda).repeat(T, 1)
    w = torch.ones((T, k), device=cuda)
    sh = fp8.shape(H, E, k, F, 1.0, ACT_SWIGLU)
    room = normal((2 * T + 2, H), 3).to(cuda)
    before = room.clone()
    r = room[1:T + 1]
    with pytest.raises(RuntimeError):
        fp8.experts(x, ids, w, store.table, sh, r, out=room[1 + rows:T + 1 + rows])
    with pytest.raises(RuntimeError):  # half a row
        flat = room.view(-1)[H + H // 2:]
        fp8.experts(x, ids, w, store.table, sh, r, out=flat[:T * H].view(T, H))
    moe, y = layer(cuda, T, E=4, H=128, F=128, k=2)
    with pytest.raises(RuntimeError):
        moe.forward(y, r, out=room[1 + rows:T + 1 + rows])
    assert torch.equal(room, before)
    want = fp8.experts(x, ids, w, store.table, sh, r)
    fp8.experts(x, ids, w, store.table, sh, r, out=room[T + 1:2 * T + 1])  # right behind it
    assert torch.equal(room[T + 1:2 * T + 1], want) and torch.equal(r, before[1:T + 1])
    fp8.experts(x, ids, w, store.table, sh, r, out=r)
    assert torch.equal(r, want)


@pytest.mark.parametrize("T", [2, 40, 300])
def test_experts_over_the_hidden_rows(cuda, T):
    """Every hidden row has been read before an output is written: any overlap is as good."""
    E, H, F, k = 4, 128, 128, 2
    store = make_store(cuda, E, H, F, 2)
    ids = torch.arange(k, dtype=torch.int32, device=cuda).repeat(T, 1)
    w = torch.ones((T, k), device=cuda)
    sh = fp8.shape(H, E, k, F, 1.0, ACT_SWIGLU)
    for at in (0, 1, 2):
        room = normal((T + 2, H), 3).to(cuda)
        x = room[1:T + 1]
        want = fp8.experts(x, ids, w, store.table, sh)
        fp8.experts(x, ids, w, store.table, sh, out=room[at:T + at])
        assert torch.equal(room[at:T + at], want)


@pytest.mark.parametrize("T,E", [(2, 8), (70, 200)])
def test_router_gradient_refuses_part_of_the_logits(cuda, T, E):
    g = torch.Generator().manual_seed(T)
    room = torch.randn(2 * T * E + 2 * E, generator=g).to(cuda)
    logits = room[E:E + T * E].view(T, E)
    ids = logits.topk(2, 1).indices.to(torch.int32)
    before = room.clone()
    _, counts, _, live = balance.balance_loss(logits, ids, 0.3)

    def gradient(at):
        return balance.router_backward(logits, ids, counts, live, 0.3, out=room[at:at + T * E].view(T, E))

    for at in (0, E - 1, E + 1, 2 * E, T * E):
        with pytest.raises(RuntimeError):
            gradient(at)
    assert torch.equal(room, before)
    want = balance.router_backward(logits, ids, counts, live, 0.3)
    assert torch.equal(gradient(E + T * E), want) and torch.equal(logits, before[E:E + T * E].view(T, E))
    assert torch.equal(gradient(E), want)


@pytest.mark.parametrize("entry", ["k3_moe_fp8_128_quantize_rows_bf16", "k3_moe_fp8_128_quantize_weight_bf16"])
def test_quantizers_refuse_codes_or_scales_over_the_values(cuda, entry):
    """Blocks of 128 values end before others are read: codes in the values' place would be read
    as values."""
    rows, cols = 200, 256
    src = normal((rows, cols), 1).to(cuda)
    n = 2 * rows * cols
    room = torch.zeros(4 * n, dtype=torch.uint8, device=cuda)
    room[n:2 * n] = src.view(torch.uint8).view(-1)
    before, base = room.clone(), room.data_ptr()
    run = lambda codes, scales, x=base + n: getattr(lib(), entry)(  # noqa: E731
        codes, scales, x, rows, cols, torch.cuda.current_stream().cuda_stream)
    away = base + 3 * n
    for codes, scales in ((base + n, away), (base + n + n // 2, away), (base + n // 2 + 8, away),
                          (base, base + n + 64), (base, base + n - 4), (base, base + 64)):
        assert not run(codes, scales), (codes - base, scales - base)
    assert torch.equal(room, before)
    assert run(base + n // 2, away) and run(base + 2 * n, away)  # right before and behind the values
    f = fp8.quantize_rows if "rows" in entry else fp8.quantize_weight
    codes, scales = f(src)
    for at in (n // 2, 2 * n):
        assert torch.equal(room[at:at + n // 2], codes.view(torch.uint8).view(-1))
    assert torch.equal(room[3 * n:3 * n + 4 * scales.numel()], scales.view(torch.uint8).view(-1))
