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


def test_in_an_autograd_function(cuda):
    """balance_loss and router_backward as a Function: the gradient that autograd hands on is the
    call's own, and without the Function logits that require a gradient are refused."""
    class Balance(torch.autograd.Function):
        @staticmethod
        def forward(ctx, logits, ids, coef):
            loss, counts, _, live = balance.balance_loss(logits, ids, coef)
            ctx.save_for_backward(logits, ids, counts, live)
            ctx.coef = coef
            return loss

        @staticmethod
        def backward(ctx, dloss):
            logits, ids, counts, live = ctx.saved_tensors
            return balance.router_backward(logits, ids, counts, live, ctx.coef, dloss=dloss), None, None

    g = torch.Generator().manual_seed(3)
    logits = torch.randn((50, 24), generator=g).to(cuda).requires_grad_()
    ids = logits.detach().topk(3, 1).indices.to(torch.int32)
    with pytest.raises(ValueError, match="requires a gradient"):
        balance.balance_loss(logits, ids, 0.4)
    (1.5 * Balance.apply(logits, ids, 0.4)).backward()
    x = logits.detach()
    _, counts, _, live = balance.balance_loss(x, ids, 0.4)
    want = balance.router_backward(x, ids, counts, live, 0.4, dloss=torch.tensor(1.5, device=cuda))
    assert torch.equal(logits.grad, want) and want.abs().max() > 0


def test_where_scores_end(cuda):
    """Scores just over 2^-126 have their shares; under it they are 0, and so is all that follows."""
    E, k = 8, 2
    ids = torch.arange(k, dtype=torch.int32, device=cuda).repeat(3, 1)
    for level, ends in ((-87.3, False), (-87.4, True), (-88.5, True), (-120.0, True)):
        logits = torch.full((3, E), level, device=cuda)
        loss, counts, mean, live = balance.balance_loss(logits, ids, 1.0)
        grad = balance.router_backward(logits, ids, counts, live, 1.0, dweights=torch.ones((3, k), device=cuda))
        if ends:
            assert loss.item() == 0 and (mean == 0).all() and (grad == 0).all()
        else:  # equal scores: shares of 1 / E, within 392 u
            assert ((mean.cpu().double() - 1 / E).abs() <= 392 * U / E).all()
