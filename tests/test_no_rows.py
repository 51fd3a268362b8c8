"""Batches of no rows, as a rank has that got no tokens: outputs are empty, the weights' gradients zeros, and
what is added to stays, without a call of the library (CPU; on the GPU the same)."""
import pytest
import torch

from moonshine_amd import experts, fp8, grouped, norm
from moonshine_amd.synth import ACT_SWIGLU
from test_training_refusals import stopped  # noqa: F401

E, N, K, k, F = 3, 16, 24, 2, 8


def check(device):
    bf = lambda *shape: torch.ones(shape, dtype=torch.bfloat16, device=device)  # noqa: E731
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=device)  # noqa: E731
    o, none, w = ints(E + 1), ints(0), bf(E, N, K)
    f32 = torch.zeros((0, k), device=device)
    for index, to in ((None, None), (none, None), (None, none), (none, none)):
        assert grouped.product(bf(0, K), w, o, index=index, to=to).shape == (0, N)
        assert grouped.input_gradient(bf(0, N), w, o, index=index, to=to).shape == (0, K)
    assert grouped.product(bf(5, K), w, o, index=none).shape == (0, N)
    kept = bf(4, N)
    assert grouped.product(bf(0, K), w, o, to=none, out=kept) is kept and (kept == 1).all()
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.ones((E, N, K), dtype=dtype, device=device)
        assert grouped.weight_gradient(bf(0, N), bf(0, K), o, dtype=dtype, out=out) is out and not out.any()
        made = grouped.weight_gradient(bf(0, N), bf(0, K), o, none, none, dtype=dtype)
        assert made.shape == (E, N, K) and made.dtype == dtype and not made.any()
    out = torch.ones((E, N, K), device=device)
    assert grouped.weight_gradient(bf(0, N), bf(7, K), o, x_index=none, out=out, accumulate=True) is out
    assert (out == 1).all()
    assert experts.gated(bf(0, 2 * F), o, none, f32, ACT_SWIGLU).shape == (0, F)
    d, dw = experts.gated_backward(bf(0, F), bf(0, 2 * F), o, none, torch.ones((4, k), device=device), ACT_SWIGLU)
    assert d.shape == (0, 2 * F) and dw.shape == (4, k) and not dw.any()
    assert experts.combine(bf(0, K), ints(0, k), E, residual=bf(0, K)).shape == (0, K)
    n = norm.residual_norm(bf(0, 256), bf(256), 1e-5, residual=bf(0, 256), encode=True)
    assert n.total.shape == n.normed.shape == n.codes.shape == (0, 256) and n.scales.shape == (0, 2)
    assert n.rstd.shape == (0,)
    dx, dweight = norm.residual_norm_backward(bf(0, 256), n.total, bf(256), n.rstd, dtotal=bf(0, 256))
    assert dx.shape == (0, 256) and dweight.shape == (256,) and not dweight.any()
    codes = torch.zeros((48, 256), dtype=torch.uint8, device=device)
    scales = torch.ones((1, 2), device=device)
    assert fp8.product_encoded(n.codes, n.scales, codes, scales).shape == (0, 48)
    # a layer in training
    gate_up, down = bf(E, 2 * F, K), bf(E, K, F)
    out, saved = experts.forward(bf(0, K), ints(0, k), f32, gate_up, down, ACT_SWIGLU, residual=bf(0, K))
    assert out.shape == (0, K)
    dhidden, dweights, dgate_up, ddown = experts.backward(bf(0, K), saved, gate_up, down)
    assert dhidden.shape == (0, K) and dweights.shape == (0, k)
    assert dgate_up.shape == gate_up.shape and not dgate_up.any()
    assert ddown.shape == down.shape and not ddown.any()
    sums = [torch.ones(t.shape, device=device) for t in (gate_up, down)]
    again = experts.backward(bf(0, K), saved, gate_up, down, *sums)
    assert again[2] is sums[0] and again[3] is sums[1] and all((t == 1).all() for t in sums)


def test_without_a_call(stopped):  # noqa: F811
    check("cpu")


def test_no_rows_are_still_checked(stopped):  # noqa: F811
    bf = lambda *shape: torch.ones(shape, dtype=torch.bfloat16)  # noqa: E731
    o, none = torch.zeros(E + 1, dtype=torch.int32), torch.zeros(0, dtype=torch.int32)
    for bad in (lambda: grouped.product(bf(0, K + 8), bf(E, N, K), o), lambda: grouped.product(bf(0, K), bf(E, N, K), none),
                lambda: grouped.weight_gradient(bf(0, N), bf(3, K), o),
                lambda: grouped.weight_gradient(bf(0, N), bf(0, K), o, out=torch.zeros(E, K, N)),
                lambda: experts.gated(bf(0, 2 * F), o, none, torch.zeros(0, k), 7),
                lambda: norm.residual_norm(bf(0, 256), bf(128), 1e-5),
                lambda: experts.forward(bf(1, K), torch.zeros((0, k), dtype=torch.int32), torch.zeros(0, k),
                                        bf(E, 2 * F, K), bf(E, K, F), ACT_SWIGLU)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.gpu
def test_on_the_gpu(cuda):
    check(cuda)
