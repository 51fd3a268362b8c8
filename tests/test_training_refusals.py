"""What the training operators and the residual norm refuse (CPU): by the C entry points, on addresses
that nothing reads, and by the wrappers, on CPU tensors that stand in for the GPU's."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

from moonshine_amd import experts, fp8, grouped, norm
from moonshine_amd._lib import lib
from moonshine_amd.synth import ACT_SITU, ACT_SWIGLU

AT = 1 << 40  # addresses far apart, one for each argument


def address(i, off=0):
    return ctypes.c_void_p(AT + (i << 36) + off)


# ---- C entry points: each refused change of a call that is otherwise in order ------------------

ROWS = dict(output=address(1), input=address(2), weights=address(3), offsets=address(4), index=address(5),
            to=address(6), rows=8, input_rows=4, output_rows=8, experts=3, n=16, k=24)


def by_rows(name, **change):
    a = dict(ROWS, **change)
    return getattr(lib(), name)(*a.values(), None)


@pytest.mark.parametrize("name", ["k3_moe_grouped_product_bf16", "k3_moe_grouped_input_gradient_bf16"])
@pytest.mark.parametrize("change", [
    dict(output=None), dict(input=None), dict(weights=None), dict(offsets=None),
    dict(output=address(1, 8)), dict(input=address(2, 8)), dict(weights=address(3, 8)), dict(offsets=address(4, 2)),
    dict(index=address(5, 1)), dict(to=address(6, 2)),
    dict(rows=0), dict(rows=65535 * 32 + 1, index=None, input_rows=1 << 22, to=None, output_rows=1 << 21),
    dict(input_rows=0), dict(input_rows=65536), dict(index=None, input_rows=7),
    dict(output_rows=0), dict(to=None, output_rows=7), dict(output_rows=65535 * 32 + 1),
    dict(experts=0), dict(experts=1025),
    dict(n=0), dict(n=12), dict(n=32776), dict(k=0), dict(k=20), dict(k=32776),
    dict(output=address(2, 16)), dict(output=address(3, 16)), dict(input=address(1, 128)),
    dict(output=address(4)), dict(output=address(5, 16)), dict(output=address(6)), dict(to=address(1, 252)),
])
def test_products_refuse(name, change):
    assert not by_rows(name, **change)


WEIGHT = dict(output=address(1), f32=True, accumulate=False, dy=address(2), x=address(3), offsets=address(4),
              dy_index=address(5), x_index=address(6), rows=8, dy_rows=4, x_rows=4, experts=3, n=16, k=24)


@pytest.mark.parametrize("change", [
    dict(output=None), dict(dy=None), dict(x=None), dict(offsets=None), dict(output=address(1, 8)),
    dict(dy=address(2, 4)), dict(x=address(3, 8)), dict(offsets=address(4, 1)), dict(dy_index=address(5, 2)),
    dict(x_index=address(6, 3)), dict(f32=False, accumulate=True), dict(rows=0), dict(dy_rows=0), dict(x_rows=65536),
    dict(dy_index=None, dy_rows=7), dict(x_index=None, x_rows=7), dict(experts=0), dict(experts=1025), dict(n=4),
    dict(k=4), dict(n=40000), dict(k=40000), dict(output=address(2, 16)), dict(output=address(3, 32)),
    dict(output=address(4)), dict(output=address(5)), dict(output=address(6, 16)), dict(offsets=address(1, 400)),
])
def test_weight_gradient_refuses(change):
    assert not lib().k3_moe_grouped_weight_gradient_bf16(*dict(WEIGHT, **change).values(), None)


GATED = dict(output=address(1), gate_up=address(2), offsets=address(3), route=address(4), weights=address(5),
             rows=8, routes=8, experts=3, ffn=16, act=ACT_SITU, beta=4.0, linear=25.0)
GATED_CHANGES = [
    dict(gate_up=None), dict(offsets=None), dict(gate_up=address(2, 8)), dict(offsets=address(3, 1)),
    dict(route=address(4, 2)), dict(weights=address(5, 1)), dict(rows=0), dict(rows=65535 * 32 + 1), dict(routes=0),
    dict(experts=0), dict(experts=1025), dict(ffn=0), dict(ffn=12), dict(ffn=32776), dict(act=2), dict(beta=0.0),
    dict(beta=float("nan")), dict(linear=-1.0), dict(output=address(3)), dict(output=address(4, 16)),
    dict(output=address(5, 16))]


@pytest.mark.parametrize("change", GATED_CHANGES + [dict(output=None), dict(output=address(1, 4)),
                                                    dict(output=address(2)), dict(output=address(2, 64))])
def test_gated_refuses(change):
    assert not lib().k3_moe_gated_rows_bf16(*dict(GATED, **change).values(), None)


@pytest.mark.parametrize("change", GATED_CHANGES + [
    dict(output=None), dict(output=address(1, 4)), dict(output=address(2, 16)), dict(output=address(7)),
    dict(dweights=address(8, 2)), dict(dweights=address(1, 64)), dict(dweights=address(2, 4)),
    dict(dweights=address(7, 8)), dict(dweights=address(5)), dict(dweights=address(3, 8)),
    dict(dweights=address(4, 28)), dict(dh=None), dict(dh=address(7, 8))])
def test_gated_backward_refuses(change):
    a = dict(output=GATED["output"], dweights=address(8), dh=address(7))
    a.update({k: v for k, v in GATED.items() if k != "output"})
    assert not lib().k3_moe_gated_rows_backward_bf16(*dict(a, **change).values(), None)


@pytest.mark.parametrize("change", [
    dict(output=None), dict(rows=None), dict(ids=None), dict(output=address(1, 8)), dict(rows=address(2, 2)),
    dict(residual=address(3, 4)), dict(ids=address(4, 1)), dict(weights=address(5, 2)), dict(T=0), dict(T=65536),
    dict(k=0), dict(k=33), dict(E=0), dict(H=0), dict(H=12), dict(H=65544), dict(output=address(2, 16)),
    dict(output=address(3, 16)), dict(output=address(4)), dict(output=address(5, 16))])
def test_combine_refuses(change):
    a = dict(output=address(1), rows=address(2), residual=address(3), ids=address(4), weights=address(5), T=4, k=2,
             E=3, H=16)
    assert not lib().k3_moe_combine_bf16(*dict(a, **change).values(), None)


@pytest.mark.parametrize("change", [
    dict(x=None), dict(weight=None), dict(total=None), dict(residual=None), dict(scales=None), dict(codes=None),
    dict(total=address(1, 8)), dict(normed=address(2, 2)), dict(codes=address(3, 4)), dict(scales=address(4, 2)),
    dict(rstd=address(5, 1)), dict(x=address(6, 8)), dict(residual=address(7, 8)), dict(weight=address(8, 8)),
    dict(rows=0), dict(rows=65535 * 32 + 1), dict(cols=0), dict(cols=132), dict(cols=136), dict(cols=32896),
    dict(eps=-1.0), dict(eps=float("nan")), dict(normed=address(1)), dict(normed=address(1, 16)),
    dict(total=address(6, 16)), dict(normed=address(7, 16)), dict(codes=address(6)), dict(scales=address(7)),
    dict(rstd=address(2, 32)), dict(total=address(8, 16)), dict(codes=address(4, 8))])
def test_norm_refuses(change):
    a = dict(total=address(1), normed=address(2), codes=address(3), scales=address(4), rstd=address(5), x=address(6),
             residual=address(7), weight=address(8), rows=4, cols=128, eps=1e-5)
    assert not lib().k3_moe_residual_norm_bf16(*dict(a, **change).values(), None)


def test_norm_refuses_a_call_for_nothing():
    assert not lib().k3_moe_residual_norm_bf16(None, None, None, None, None, address(6), None, address(8), 4, 128,
                                               1e-5, None)


@pytest.mark.parametrize("change", [
    dict(dx=None), dict(dweight=None), dict(dn=None), dict(total=None), dict(weight=None), dict(rstd=None),
    dict(scratch=None), dict(scratch=address(8, 16)), dict(bytes=100), dict(rows=0), dict(cols=12), dict(cols=40000),
    dict(dx=address(1, 8)), dict(dt=address(7, 2)), dict(dweight=address(2, 2)), dict(rstd=address(6, 1)),
    dict(dx=address(3, 16)), dict(dx=address(4, 16)), dict(dx=address(7, 16)), dict(dx=address(5)),
    dict(dweight=address(1, 16)), dict(dweight=address(8)), dict(dweight=address(3, 4)), dict(dweight=address(4)),
    dict(dweight=address(5, 128)), dict(dweight=address(6, 12)), dict(dweight=address(7)), dict(scratch=address(1)),
    dict(scratch=address(3)), dict(scratch=address(4, 256)), dict(scratch=address(5)), dict(scratch=address(6)),
    dict(scratch=address(7, 512)), dict(dx=address(8, 256))])
def test_norm_backward_refuses(change):
    a = dict(dx=address(1), dweight=address(2), dn=address(3), total=address(4), weight=address(5), rstd=address(6),
             dt=address(7), rows=4, cols=128, scratch=address(8), bytes=1 << 20)
    assert not lib().k3_moe_residual_norm_backward_bf16(*dict(a, **change).values(), None)


def test_norm_scratch_grows_with_the_rows():
    size = lib().k3_moe_residual_norm_scratch_bytes
    for cols in (8, 512, 520, 2048, 2056, 7168, 32768):
        sizes = [size(rows, cols) for rows in (1, 2, 5, 300, 767, 768, 769, 5000, 65535 * 32)]
        assert sizes == sorted(sizes) and sizes[0] > 0
    assert size(0, 128) == size(65535 * 32 + 1, 128) == size(4, 12) == size(4, 32776) == 0


@pytest.mark.parametrize("change", [
    dict(output=None), dict(codes=None), dict(scales=None), dict(x=None), dict(xs=None), dict(x=address(4, 8)),
    dict(xs=address(5, 2)), dict(T=0), dict(T=65536), dict(cols=64), dict(output=address(4, 16)),
    dict(output=address(5)), dict(bytes=0), dict(scratch=None)])
def test_encoded_product_refuses(change):
    a = dict(output=address(1), codes=address(2), scales=address(3), x=address(4), xs=address(5), T=1000, rows=4096,
             cols=1024, scratch=address(6), bytes=1 << 30)
    assert not lib().k3_moe_fp8_128_encoded_gemm_bf16(*dict(a, **change).values(), None)


def test_refused_calls_launch_nothing():
    """Without a GPU a call that goes through fails as well, at its launch: the runtime's log tells the two
    apart. In a process that sees no GPU."""
    env = dict(os.environ, HIP_VISIBLE_DEVICES="-1", AMD_LOG_LEVEL="3")
    launch = "__hipPushCallConfiguration"

    def log(*command):
        run = subprocess.run([sys.executable, *command], env=env, cwd=os.path.dirname(os.path.abspath(__file__)),
                             capture_output=True, text=True, timeout=300)
        return run.returncode, run.stdout + run.stderr

    code, text = log("-c", "import conftest, test_training_refusals as t\n"
                           "assert not t.by_rows('k3_moe_grouped_product_bf16')")
    assert code == 0 and launch in text
    code, text = log("-m", "pytest", "-q", "-s", "-p", "no:cacheprovider", "-k", "refuse and not wrappers and not launch",
                     os.path.basename(__file__))
    assert code == 0 and launch not in text, text[-2000:]


# ---- wrappers -----------------------------------------------------------------------------------


class Called(Exception):
    pass


@pytest.fixture
def stopped(monkeypatch):
    """Layout checks without the one for the device; a call whose checks pass ends where it would
    take memory or launch."""
    def stop(*args, **kwargs):
        raise Called

    monkeypatch.setattr(fp8, "_layout", lambda t, *args: t.data_ptr())
    for module in (grouped, experts, norm, fp8):
        monkeypatch.setattr(module, "_call", stop)
        if hasattr(module, "_scratch"):
            monkeypatch.setattr(module, "_scratch", lambda like, n: (None, None))


def bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


E, N, K, T, k, F = 3, 16, 24, 4, 2, 8
R = T * k


def calls(**x):
    a = dict(x=bf(T, K), weights=bf(E, N, K), dy=bf(R, N), offsets=ints(E + 1), index=ints(R), to=ints(R), ids=ints(T, k),
             gate_up=bf(R, 2 * F), dh=bf(R, F), route=ints(R), w=torch.ones(T, k), rows=bf(R, K), residual=bf(T, K),
             out=None, weight=bf(128), h=bf(T, 128), r=bf(T, 128), dn=bf(T, 128), rstd=torch.ones(T), dt=bf(T, 128))
    a.update(x)
    return {
        "plan": lambda: grouped.route_plan(a["ids"], E),
        "product": lambda: grouped.product(a["x"], a["weights"], a["offsets"], a["index"], a["to"], a["out"]),
        "input": lambda: grouped.input_gradient(a["dy"], a["weights"], a["offsets"], to=a["to"], out=a["out"]),
        "weight": lambda: grouped.weight_gradient(a["dy"], a["x"], a["offsets"], x_index=a["index"], out=a["out"]),
        "gated": lambda: experts.gated(a["gate_up"], a["offsets"], a["route"], a["w"], ACT_SWIGLU, out=a["out"]),
        "gated_backward": lambda: experts.gated_backward(a["dh"], a["gate_up"], a["offsets"], a["route"], a["w"],
                                                         ACT_SWIGLU, out=a["out"]),
        "combine": lambda: experts.combine(a["rows"], a["ids"], E, a["residual"], a["w"], a["out"]),
        "norm": lambda: norm.residual_norm(a["h"], a["weight"], 1e-5, residual=a["r"], encode=True, total=a["out"]),
        "norm_backward": lambda: norm.residual_norm_backward(a["dn"], a["r"], a["weight"], a["rstd"], a["dt"],
                                                             a["out"]),
    }


@pytest.mark.parametrize("name", sorted(calls()))
def test_calls_in_order_pass(stopped, name):
    with pytest.raises(Called):
        calls()[name]()


@pytest.mark.parametrize("name,leaves", [
    ("product", ["x", "weights"]), ("input", ["dy", "weights"]), ("weight", ["dy", "x"]), ("gated", ["gate_up", "w"]),
    ("gated_backward", ["dh", "gate_up", "w"]), ("combine", ["rows", "w", "residual"]), ("norm", ["h", "r", "weight"]),
    ("norm_backward", ["dn", "r", "weight", "rstd", "dt"])])
def test_an_input_that_requires_a_gradient_is_refused(stopped, name, leaves):
    for leaf in leaves:
        value = {"w": torch.ones(T, k), "rstd": torch.ones(T), "weights": bf(E, N, K), "dy": bf(R, N), "x": bf(T, K),
                 "gate_up": bf(R, 2 * F), "dh": bf(R, F), "rows": bf(R, K), "residual": bf(T, K),
                 "weight": bf(128)}.get(leaf, bf(T, 128)).requires_grad_()
        with pytest.raises(ValueError, match="requires a gradient"):
            calls(**{leaf: value})[name]()
        with torch.no_grad(), pytest.raises(Called):
            calls(**{leaf: value})[name]()


@pytest.mark.parametrize("name,change", [
    ("plan", dict(ids=ints(0, 2))), ("plan", dict(ids=ints(3, 33))),
    ("product", dict(x=bf(T, K + 8))), ("product", dict(offsets=ints(E))), ("product", dict(to=ints(R - 1))),
    ("product", dict(x=bf(65536, K))), ("product", dict(out=bf(R, N + 8))), ("product", dict(to=None, out=bf(R - 1, N))),
    ("input", dict(dy=bf(R, N + 8))), ("input", dict(dy=bf(R + 1, N))), ("input", dict(out=bf(R, N))),
    ("weight", dict(x=bf(65536, K))), ("weight", dict(dy=bf(R + 1, N))), ("weight", dict(offsets=ints(1))),
    ("weight", dict(out=torch.zeros(E, K, N))),
    ("gated", dict(gate_up=bf(R, 2 * F + 1))), ("gated", dict(route=ints(R + 1))), ("gated", dict(out=bf(R, 2 * F))),
    ("gated_backward", dict(dh=bf(R, 2 * F))), ("gated_backward", dict(out=bf(R, F))),
    ("combine", dict(rows=bf(R + 1, K))), ("combine", dict(w=torch.ones(T, k + 1))), ("combine", dict(residual=bf(T, N))),
    ("combine", dict(out=bf(R, K))),
    ("norm", dict(weight=bf(127))), ("norm", dict(r=bf(T + 1, 128))), ("norm", dict(out=bf(T, 256))),
    ("norm", dict(h=bf(T, 64), r=bf(T, 64), weight=bf(64))),
    ("norm_backward", dict(rstd=torch.ones(T + 1))), ("norm_backward", dict(weight=bf(8))),
    ("norm_backward", dict(dt=bf(T, 64))), ("norm_backward", dict(out=bf(1, 128)))])
def test_wrappers_refuse(stopped, name, change):
    with pytest.raises(ValueError):
        calls(**change)[name]()


def test_other_refusals(stopped):
    with pytest.raises(ValueError, match="accumulate"):
        grouped.weight_gradient(bf(R, N), bf(R, K), ints(E + 1), accumulate=True)
    with pytest.raises(ValueError, match="accumulate"):
        grouped.weight_gradient(bf(R, N), bf(R, K), ints(E + 1), dtype=torch.bfloat16, out=bf(E, N, K), accumulate=True)
    with pytest.raises(ValueError, match="dtype"):
        grouped.weight_gradient(bf(R, N), bf(R, K), ints(E + 1), dtype=torch.float16)
    with pytest.raises(ValueError, match="activation"):
        experts.gated(bf(R, 2 * F), ints(E + 1), ints(R), torch.ones(T, k), 2)
    with pytest.raises(ValueError, match="total"):
        norm.residual_norm(bf(T, 128), bf(128), 1e-5, total=bf(T, 128))
    with pytest.raises(ValueError, match="product of"):
        fp8.product_encoded(torch.zeros((T, 256), dtype=torch.uint8), torch.ones(T, 1),
                            torch.zeros((64, 256), dtype=torch.uint8), torch.ones(1, 2))
