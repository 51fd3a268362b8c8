"""What moonshine_amd.fp8 and moonshine_amd.balance refuse by themselves, on CPU
tensors that stand in for the GPU's: nothing is launched."""
import pytest
import torch

from moonshine_amd import fp8
from moonshine_amd.synth import Config

E, F, H = 2, 128, 256


@pytest.fixture
def anywhere(monkeypatch):
    """Layout checks without the one for the device."""
    monkeypatch.setattr(fp8, "_dense", lambda t, *args: t.data_ptr())


def matrices():
    make = lambda rows, cols: (torch.zeros((E, rows, cols), dtype=torch.uint8),  # noqa: E731
                               torch.ones((E, rows // 128, cols // 128)))
    return dict(gate=make(F, H), down=make(H, F), up=make(F, H))


def view_of_blob(t, at):
    """A contiguous view of t's size, `at` bytes into a buffer."""
    room = torch.zeros(t.numel() + 64, dtype=torch.uint8)
    start = -room.data_ptr() % 16 + at
    return room[start:start + t.numel()].view(t.shape)


@pytest.mark.parametrize("name", ["gate", "down", "up"])
@pytest.mark.parametrize("at", [1, 4, 8])
@pytest.mark.parametrize("dtype", [torch.uint8, torch.float8_e4m3fn])
def test_store_refuses_codes_off_a_boundary_of_16_bytes(anywhere, name, at, dtype):
    m = matrices()
    fp8.Fp8ExpertStore(**m)
    codes, scales = m[name]
    m[name] = view_of_blob(codes, 16).view(dtype), scales
    fp8.Fp8ExpertStore(**m)
    m[name] = view_of_blob(codes, at).view(dtype), scales
    with pytest.raises(ValueError, match=name):
        fp8.Fp8ExpertStore(**m)


def test_layer_refuses_a_store_on_another_device(anywhere):
    m = matrices()
    store = fp8.Fp8ExpertStore(**m)
    router = torch.zeros((E, H), dtype=torch.bfloat16), torch.zeros(E)
    cfg = Config("small", 1, H, E, 1, F)
    fp8.Fp8RoutedMoE(cfg, *router, store)
    store.table = store.table.to("meta")
    with pytest.raises(ValueError, match="meta"):
        fp8.Fp8RoutedMoE(cfg, *router, store)
