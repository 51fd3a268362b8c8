"""The router's gradient where fp32 nearly ends: scores down to 2^-126 and loss gradients of a
loss scale, against the formula in 64 bits.

u = 2^-24. A score and 1 - score are within (8 + 2 |x|) u of themselves: 184 u for |x| <= 88. Z adds
up to 64 of them (22 u more): 206 u. A share sigma / Z is within 392 u, f times it, summed, 30 u more.
The gradient is a difference of two terms, share f and share sum f sigma / Z, each times sigma
(1 - sigma) / Z: 422 + 2 x 184 + 206 and under 28 roundings: 1024 u of their sizes.
"""
import pytest
import torch

from moonshine_amd import balance
from test_gpu_balance import U, forward64, weights64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("level", [-86.5, -80.0, -40.0, 0.0])
@pytest.mark.parametrize("dloss", [1.0, 65536.0, -1e30])
@pytest.mark.parametrize("routes", [False, True])
def test_gradient_of_low_scores(cuda, level, dloss, routes):
    T, E, k, coef, scale = 5, 40, 3, 0.7, 2.5
    g = torch.Generator().manual_seed(7)
    logits = level + torch.randn((T, E), generator=g).clamp(-0.8, 0.8)
    ids = logits.topk(k, 1).indices.to(torch.int32)
    dw = torch.randn((T, k), generator=g) if routes else None
    x = logits.double().requires_grad_()
    loss, counts, _, n, _, ok, sig = forward64(x, ids, coef, 1, None)
    total = loss * dloss
    if routes:
        total = total + (weights64(sig, ids, ok, scale) * dw.double()).sum()
    (want,) = torch.autograd.grad(total, x)
    own = balance.balance_loss(logits.to(cuda), ids.to(cuda), coef)
    assert torch.equal(own[1].cpu().double(), counts)
    got = balance.router_backward(logits.to(cuda), ids.to(cuda), own[1], own[3], coef,
                                  dloss=torch.tensor(dloss, device=cuda),
                                  dweights=None if dw is None else dw.to(cuda),
                                  scaling_factor=scale).cpu().double()
    sig = sig.detach()
    f, z = counts * E / (k * T), sig.sum(1, keepdim=True)
    size = abs(coef * dloss) / T / z * (f + (f * sig).sum(1, keepdim=True) / z)
    if routes:
        picked = sig.gather(1, ids.long())
        den = 1e-20 + picked.sum(1, keepdim=True)
        part = scale / den * (dw.double().abs() + (dw.double().abs() * picked).sum(1, keepdim=True) / den)
        size = size.scatter_add(1, ids.long(), part)
    off = (got - want).abs()
    bound = 1024 * U * size * sig * (1 - sig) + 1e-38
    assert torch.isfinite(got).all() and (off <= bound).all(), (off / bound).max()
