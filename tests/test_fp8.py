"""FP8-128 and balance entry points on the CPU: sizes, refusals before any
launch, and the test reference's own encoder against torch's e4m3 cast."""
import ctypes

import numpy as np
import pytest
import torch

import _fp8 as R
from moonshine_amd import _lib, balance, fp8
from moonshine_amd._lib import K3MoeNativeShape
from moonshine_amd.native import NativeConfig, routed_shape
from moonshine_amd.synth import ACT_SITU, ACT_SWIGLU

P = ctypes.c_void_p(1 << 20)  # never dereferenced: the checks fail first


def test_reference_encoder_is_the_e4m3_cast():
    """Every bf16 within +-448, and values around every tie of the format."""
    bits = np.arange(1 << 16, dtype=np.uint32) << 16
    v = bits.view(np.float32)
    v = v[np.abs(v) <= 448]
    pos = R.values(np.arange(0x7f, dtype=np.uint8)).numpy()
    ties = ((pos[1:] + pos[:-1]) / 2).astype(np.float32)
    v = np.concatenate([v, ties, -ties, np.nextafter(ties, np.float32(0)),
                        np.nextafter(ties, np.float32(500)), np.float32([448 * (1 + 2 ** -23)])])
    want = torch.from_numpy(v).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(R.encode(v), want)


@pytest.mark.parametrize("T,N,K", [(1, 1, 128), (65535, 7168, 7168), (37, 4100, 2048)])
def test_scratch_holds_the_encoded_rows(T, N, K):
    n = _lib.lib().k3_moe_fp8_128_scratch_bytes(T, N, K)
    assert n % 256 == 0
    assert n == 0 or n >= T * K + T * K // 32


def test_scratch_refuses():
    f = _lib.lib().k3_moe_fp8_128_scratch_bytes
    for bad in ((0, 1, 128), (65536, 1, 128), (1, 0, 128), (20, (1 << 24) + 1, 128),
                (20, 1, (1 << 24) + 128), (1, 1, 0), (1, 1, 64), (1, 1, 192)):
        assert f(*bad) == 0


def test_quantizers_refuse():
    L = _lib.lib()
    for f in (L.k3_moe_fp8_128_quantize_rows_bf16, L.k3_moe_fp8_128_quantize_weight_bf16):
        for bad in ((None, P, P, 1, 128), (P, None, P, 1, 128), (P, P, None, 1, 128),
                    (P, P, P, 0, 128), (P, P, P, 1, 0), (P, P, P, 1, 64), (P, P, P, 1, 200),
                    (P, P, P.value + 8, 1, 128), (P.value + 4, P, P, 1, 128),
                    (P, P.value + 2, P, 1, 128)):
            assert not f(*bad, None)


def test_product_refuses():
    L = _lib.lib()
    big = 1 << 40
    good = [P, P, P, P, 5, 64, 256, P, big]
    for at, bad in ((0, None), (1, None), (2, None), (3, None), (4, 0), (4, 65536), (5, 0),
                    (5, (1 << 24) + 1), (6, 0),
                    (6, 64), (6, 200), (0, P.value + 1), (1, P.value + 8), (2, P.value + 2),
                    (3, P.value + 8)):
        args = list(good)
        args[at] = bad
        assert not L.k3_moe_fp8_128_gemm_bf16(*args, None), (at, bad)
    for at in (P.value + 16, P.value - 2, P.value + 2 * 5 * 256 - 2):  # an output over the input
        assert not L.k3_moe_fp8_128_gemm_bf16(at, P, P, P, 5, 64, 256, P, big, None), at
    need = L.k3_moe_fp8_128_scratch_bytes(300, 640, 256)
    assert need > 0
    for at, n in ((None, need), (P, need - 1), (P.value + 128, need)):
        assert not L.k3_moe_fp8_128_gemm_bf16(P, P, P, P, 300, 640, 256, at, n, None)


def test_experts_refuse():
    L = _lib.lib()
    good = dict(hidden=256, experts=8, top_k=2, ffn=128, scaling_factor=1.0, activation=ACT_SWIGLU)
    size = lambda T=5, **kw: L.k3_moe_fp8_workspace_bytes(  # noqa: E731
        ctypes.byref(fp8.shape(**{**good, **kw})), T)
    assert size() > 0 and size() % 256 == 0 and size(T=65535) > 0
    for kw in (dict(hidden=0), dict(hidden=192), dict(ffn=64), dict(ffn=0), dict(experts=0),
               dict(experts=1025), dict(top_k=0), dict(top_k=9), dict(experts=64, top_k=33),
               dict(scaling_factor=0.0), dict(activation=2), dict(T=0), dict(T=65536),
               dict(activation=ACT_SITU, beta=0.0), dict(activation=ACT_SITU, linear_beta=-1.0)):
        assert size(**kw) == 0, kw
    s, n = ctypes.byref(fp8.shape(**good)), size()
    args = [P, P, P, P, P, P, s, 5, P, n]
    for at, bad in ((0, None), (1, None), (3, None), (4, None), (5, None), (6, None), (7, 0),
                    (8, None), (9, n - 1), (0, P.value + 8), (1, P.value + 8), (2, P.value + 8),
                    (3, P.value + 2), (4, P.value + 2), (5, P.value + 4), (8, P.value + 128)):
        a = list(args)
        a[at] = bad
        assert not L.k3_moe_fp8_experts_bf16(*a, None), (at, bad)
    args = [P, P, P, P, P, P, s, 5, None, None, P, n]
    for at, bad in ((0, None), (1, None), (3, None), (4, None), (5, None), (6, None), (7, 0),
                    (10, None), (11, n - 1), (3, P.value + 8), (5, P.value + 4), (10, P.value + 64)):
        a = list(args)
        a[at] = bad
        assert not L.k3_moe_fp8_forward_bf16(*a, None), (at, bad)


def test_balance_refuses():
    L = _lib.lib()
    size = L.k3_moe_balance_scratch_bytes
    assert size(1, 1, 1) > 0 and size(1, 1 << 24, 1024) > 0 and size(65535, 256, 8) > 0
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, 1025), (65536, 1, 8), (1, (1 << 24) + 1, 8),
                (4096, 4097, 8)):
        assert size(*bad) == 0
    n = size(3, 40, 16)
    good = [P, P, P, P, P, P, None, 3, 40, 16, 4, 0.5, P, n]
    for at, bad in ((0, None), (1, None), (2, None), (3, None), (4, None), (5, None), (7, 0),
                    (8, 0), (9, 0), (9, 1025), (10, 0), (10, 17), (12, None), (13, n - 1),
                    (12, P.value + 128)):
        a = list(good)
        a[at] = bad
        assert not L.k3_moe_balance_loss_f32(*a, None), (at, bad)
    a = list(good)
    a[9], a[10], a[13] = 64, 33, 1 << 30
    assert not L.k3_moe_balance_loss_f32(*a, None)
    good = [P, P, P, P, P, None, None, P, 3, 40, 16, 4, 0.5, 1.0]
    for at, bad in ((0, None), (1, None), (2, None), (3, None), (4, None), (8, 0), (9, 0), (10, 0),
                    (10, 1025), (11, 0), (11, 17), (13, 0.0), (13, float("nan"))):
        a = list(good)
        a[at] = bad
        assert not L.k3_moe_router_backward_f32(*a, None), (at, bad)


def test_wrappers_refuse_tensors_that_are_not_on_the_gpu():
    x = torch.zeros((2, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        fp8.quantize_rows(x)
    with pytest.raises(ValueError):
        fp8.product(x, x, x)
    with pytest.raises(ValueError):
        balance.balance_loss(torch.zeros((2, 8)), torch.zeros((2, 1), dtype=torch.int32), 1.0)


def test_scratch_for_more_serves_fewer():
    """Sizes grow with the tokens: memory for the most tokens is enough for any."""
    L = _lib.lib()
    steps = list(range(1, 80)) + list(range(80, 1200, 7)) + [4096, 8191, 20000, 65535]
    for n, k in ((16, 128), (576, 2048), (4096, 7168), (4100, 7168), (7168, 7168), (20000, 512)):
        sizes = [L.k3_moe_fp8_128_scratch_bytes(t, n, k) for t in steps]
        assert sizes == sorted(sizes), (n, k)
    for kw in (dict(hidden=256, experts=8, top_k=2, ffn=128), dict(hidden=128, experts=64, top_k=6, ffn=2048),
               dict(hidden=7168, experts=128, top_k=8, ffn=2048),
               dict(hidden=8320, experts=4, top_k=4, ffn=256)):
        s = ctypes.byref(fp8.shape(scaling_factor=1.0, activation=ACT_SWIGLU, **kw))
        sizes = [L.k3_moe_fp8_workspace_bytes(s, t) for t in steps]
        assert sizes == sorted(sizes), kw
    for cfg in (NativeConfig("a", 1, 1024, 512, 64, 4, 256, 768),
                NativeConfig("b", 1, 7168, 3584, 64, 4, 256, 4096)):
        s = ctypes.byref(K3MoeNativeShape(routed_shape(cfg), cfg.hidden, cfg.shared, cfg.eps))
        sizes = [L.k3_moe_native_workspace_bytes(s, t) for t in steps]
        assert sizes == sorted(sizes), cfg
    for segments in (1, 3, 40, 600):
        sizes = [L.k3_moe_balance_scratch_bytes(segments, t, 64) for t in range(1, 9000, 13)]
        assert sizes == sorted(sizes), segments
