"""The K3-native block with FP8-128 and mixed static weights: in a workspace of exactly its size, and
captured (the FP8-128 layer too)."""
import ctypes

import pytest
import torch

from moonshine_amd import native as N
from moonshine_amd._lib import lib
from test_gpu_fp8 import layer, normal

pytestmark = pytest.mark.gpu
NAMES = ("routed_down", "routed_up", "shared_gate", "shared_up", "shared_down")


def block(cuda, T, fp8):
    """A block whose weights named in `fp8` are FP8-128, the others Q8-128."""
    cfg = N.NativeConfig("native-mixed", T, 1024, 512, 64, 4, 256, 768, static_kind=N.STATIC_Q8, seed=2100)
    blk = N.NativeLayer(cfg, device=cuda)
    other = N.NativeLayer(N.NativeConfig("native-mixed", T, 1024, 512, 64, 4, 256, 768,
                                         static_kind=N.STATIC_FP8, seed=2100), device=cuda, store=blk.store)
    for name in fp8:
        setattr(blk, name, getattr(other, name))
        setattr(blk.weights, name, getattr(blk, name).c_struct())
    return blk


@pytest.mark.parametrize("fp8", [(), ("routed_down",), ("shared_down",), ("shared_gate", "routed_up"), NAMES])
@pytest.mark.parametrize("T", [1, 5, 40, 300])
@pytest.mark.parametrize("shared_stream", [False, True])
def test_exact_workspace(cuda, fp8, T, shared_stream):
    """The same bits as with room to spare, nothing written behind it, and no byte less is taken."""
    blk = block(cuda, T, fp8)
    x, r = normal((T, 1024), T).to(cuda), normal((T, 1024), T + 1).to(cuda)
    side = torch.cuda.Stream()
    stream = side.cuda_stream if shared_stream else None
    room = torch.full((1 << 28,), 0x5a, dtype=torch.uint8, device=cuda)
    blk._ws = room
    want = blk.forward(x, r, shared_stream=stream)
    torch.cuda.synchronize()
    need = lib().k3_moe_native_weights_workspace_bytes(ctypes.byref(blk.weights), ctypes.byref(blk.shape), T)
    assert 0 < need < room.numel() - 4096
    if not fp8:
        assert need == lib().k3_moe_native_workspace_bytes(ctypes.byref(blk.shape), T)
    room.fill_(0x5a)
    blk._ws = room[:need]
    out = blk.forward(x, r, shared_stream=stream)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and (room[need:need + 4096] == 0x5a).all()
    blk.workspace = lambda tokens: room[:need - 256]
    with pytest.raises(RuntimeError):
        blk.forward(x, r, shared_stream=stream)


@pytest.mark.parametrize("T", [1, 5, 100])
@pytest.mark.parametrize("shared_stream", [False, True])
def test_replayed(cuda, T, shared_stream):
    """The block captured on one or two streams: every replay is the eager call, which runs between."""
    blk = block(cuda, T, NAMES)
    x, r = normal((T, 1024), T).to(cuda), normal((T, 1024), T + 1).to(cuda)
    ids, w = torch.zeros((T, 4), dtype=torch.int32, device=cuda), torch.zeros((T, 4), device=cuda)
    side = torch.cuda.Stream()
    stream = side.cuda_stream if shared_stream else None
    blk.forward(x, r, shared_stream=stream)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = blk.forward(x, r, ids=ids, weights=w, shared_stream=stream)
    for n in range(4):
        v = normal((T, 1024), 50 + n).to(cuda)
        x.copy_(v)
        g.replay()
        got = out.clone(), ids.clone(), w.clone()
        eager = torch.zeros_like(ids), torch.zeros_like(w)
        want = blk.forward(v, r, ids=eager[0], weights=eager[1], shared_stream=stream)
        torch.cuda.synchronize()
        for a, b in zip(got, (want, *eager)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T", [1, 40, 200])
def test_layer_replayed_with_its_routes(cuda, T):
    """The FP8-128 layer's copies of the routes are part of the graph."""
    moe, x = layer(cuda, T)
    ids = torch.zeros((T, moe.cfg.top_k), dtype=torch.int32, device=cuda)
    w = torch.zeros((T, moe.cfg.top_k), device=cuda)
    moe.forward(x, x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = moe.forward(x, x, ids=ids, weights=w)
    for n in range(4):
        v = normal(x.shape, 60 + n).to(cuda)
        x.copy_(v)
        g.replay()
        got = out.clone(), ids.clone(), w.clone()
        eager = torch.zeros_like(ids), torch.zeros_like(w)
        want = moe.forward(v, v, ids=eager[0], weights=eager[1])
        torch.cuda.synchronize()
        for a, b in zip(got, (want, *eager)):
            assert torch.equal(a, b)
