"""What moonshine_amd.fp8 and moonshine_amd.balance refuse by themselves, on CPU
tensors that stand in for the GPU's: nothing is launched."""
import importlib.util
from types import SimpleNamespace

import pytest
import torch

from moonshine_amd import balance, fp8
from moonshine_amd.synth import Config

E, F, H = 2, 128, 256


@pytest.fixture
def anywhere(monkeypatch):
    """Layout checks without the one for the device."""
    monkeypatch.setattr(fp8, "_layout", lambda t, *args: t.data_ptr())


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


class Called(Exception):
    pass


@pytest.fixture
def stopped(anywhere, monkeypatch):
    """A call whose checks pass ends where it would take memory or launch."""
    def stop(*args, **kwargs):
        raise Called

    for module in (fp8, balance):
        monkeypatch.setattr(module, "_call", stop)
        monkeypatch.setattr(module, "_scratch", lambda like, n: (None, None))


def calls(leaf):
    """Each call of the wrappers by its name, `leaf` among its inputs where it has that name."""
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    m = matrices()
    store = fp8.Fp8ExpertStore(**m)
    x = dict(x=bf(3, H), hidden=bf(3, H), residual=bf(3, H), ids=torch.zeros((3, 1), dtype=torch.int32),
             weights=torch.ones((3, 1)), logits=torch.zeros((4, E)), dweights=torch.zeros((4, 1)),
             dloss=torch.ones(()), router_weight=bf(E, H), router_bias=torch.zeros(E),
             scales=torch.ones((1, 2)))
    if leaf is not None:
        x[leaf].requires_grad_()
    sh = fp8.shape(H, E, 1, F, 1.0, 0)
    layer = fp8.Fp8RoutedMoE(Config("small", 3, H, E, 1, F), x["router_weight"], x["router_bias"], store)
    route = torch.zeros((4, 1), dtype=torch.int32)
    counts, live = torch.zeros((1, E), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    return {
        "product": lambda: fp8.product(x["x"], torch.zeros((128, H), dtype=torch.uint8), x["scales"]),
        "experts": lambda: fp8.experts(x["hidden"], x["ids"], x["weights"], store.table, sh, x["residual"]),
        "layer": lambda: layer.forward(x["hidden"], x["residual"]),
        "loss": lambda: balance.balance_loss(x["logits"], route, 1.0),
        "backward": lambda: balance.router_backward(x["logits"], route, counts, live, 1.0,
                                                    dloss=x["dloss"], dweights=x["dweights"]),
        "quantize": lambda: fp8.quantize_weight(x["x"]),
    }


@pytest.mark.parametrize("call,leaves", [
    ("product", ["x", "scales"]), ("experts", ["hidden", "weights", "residual"]),
    ("layer", ["hidden", "residual", "router_weight", "router_bias"]), ("loss", ["logits"]),
    ("backward", ["logits", "dloss", "dweights"])])
def test_an_input_that_requires_a_gradient_is_refused(stopped, call, leaves):
    """Autograd would go on without it. Not refused: no gradient recorded, or wanted."""
    with pytest.raises(Called):
        calls(None)[call]()
    for leaf in leaves:
        with pytest.raises(ValueError, match=f"^{leaf} requires a gradient"):
            calls(leaf)[call]()
        with torch.no_grad(), pytest.raises(Called):
            calls(leaf)[call]()


def test_a_weight_that_requires_a_gradient_is_encoded(stopped):
    with pytest.raises(Called):
        calls("x")["quantize"]()


def test_imports_without_torchs_private_names(monkeypatch):
    """The package loads, and asks for device and stream by torch's public functions."""
    for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
        monkeypatch.delattr(torch._C, name, raising=False)
    spec = importlib.util.spec_from_file_location("moonshine_amd._fp8_again", fp8.__file__)
    again = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(again)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: SimpleNamespace(cuda_stream=7 + device))
    assert again._device is torch.cuda.current_device and again._stream(3) == 10
