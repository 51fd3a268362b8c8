"""The routed experts' forward and backward as one, from the norm before them to the router's gradient, on the
GPU against 64-bit autograd.

The 64-bit form takes the bf16 roundings that the operators make (gate/up rows, the weighted
activation, each route's row, the gradients of h and of gate/up, and the outputs) as errors: each is
2^-8 of its value, and they add up along the way. A value is held to the sum of the terms that it is made
of, in magnitudes, times the number of roundings on its way (six at most) and 2^-8, with as much again
for how they meet.
"""
import pytest
import torch

import _grouped as R
from moonshine_amd import balance, experts, norm
from moonshine_amd.synth import ACT_SITU, ACT_SWIGLU

pytestmark = pytest.mark.gpu

EPS = 1e-5


def activation(g, u, act):
    s = torch.sigmoid(g)
    if act == ACT_SWIGLU:
        return g * s * u
    return 4.0 * torch.tanh(g / 4.0) * s * 25.0 * torch.tanh(u / 25.0)


def problem(T, k, E, H, F, seed):
    x, res = R.normal((T, H), seed), R.normal((T, H), seed + 1)
    gu, down = R.normal((E, 2 * F, H), seed + 2, H ** -0.5), R.normal((E, H, F), seed + 3, F ** -0.5)
    ids = R.routes(T, k, E, seed, 0.5)
    w = torch.rand((T, k), generator=torch.Generator().manual_seed(seed)) + 0.1
    return x, res, gu, down, ids, w, R.normal((T, H), seed + 4, 1e-2)


def live_routes(ids, E):
    T, k = ids.shape
    keep = torch.zeros((T, k), dtype=torch.bool)
    for t in range(T):
        seen = set()
        for r in range(k):
            e = int(ids[t, r])
            keep[t, r] = 0 <= e < E and e not in seen
            seen.add(e)
    return keep


def formula(x, w, gu, down, ids, act, E):
    """sum over live routes of w down_e(act(gate_e x, up_e x)), in 64 bits."""
    keep = live_routes(ids, E)
    out = torch.zeros_like(x)
    F = down.shape[2]
    for e in range(E):
        t, r = torch.where((ids == e) & keep)
        if len(t):
            z = x[t] @ gu[e].t()
            out = out.index_add(0, t, w[t, r][:, None] * activation(z[:, :F], z[:, F:], act) @ down[e].t())
    return out


def relative(got, want):
    return float((got.cpu().double() - want).norm() / want.norm())


@pytest.mark.parametrize("act", [ACT_SITU, ACT_SWIGLU])
@pytest.mark.parametrize("T,k,E,H,F", [(1, 2, 4, 64, 32), (7, 3, 5, 72, 40), (150, 2, 6, 264, 136), (600, 4, 8, 256, 128)])
def test_forward_and_backward(cuda, act, T, k, E, H, F):
    x, res, gu, down, ids, w, dout = problem(T, k, E, H, F, T)
    ids = ids.clone()
    if T > 1:
        ids[0, 1], ids[1, 0] = ids[0, 0], E  # a repeated route, and one of no expert
    on = [t.to(cuda) for t in (x, ids, w, gu, down)]
    out, saved = experts.forward(*on, act, residual=res.to(cuda))
    dx, dw, dgu, ddown = experts.backward(dout.to(cuda), saved, on[3], on[4])
    leaves = [t.double().requires_grad_() for t in (x, w, gu, down)]
    want = formula(*leaves, ids, act, E)
    grads = torch.autograd.grad((want * dout.double()).sum(), leaves)
    # roundings: gate/up, h, y, the sum, the output; and dh, dgate/up, the rows' gradients, their sum
    most = 6 * 2.0 ** -8
    assert relative(out, want.detach() + res.double()) <= most
    for got, g in zip((dx, dw, dgu, ddown), grads):
        assert got.shape == g.shape and relative(got, g) <= most
    assert (dw.cpu()[~live_routes(ids, E)] == 0).all()
    # a second batch adds to the gradients
    again = experts.backward(dout.to(cuda), saved, on[3], on[4], dgate_up=dgu.clone(), ddown=ddown.clone())
    assert torch.equal(again[2], 2 * dgu) and torch.equal(again[3], 2 * ddown)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


def test_gradient_by_differences(cuda):
    """The formula's own gradient, which the kernels are held to, by central differences."""
    x, _, gu, down, ids, w, dout = (t.double() if t.is_floating_point() else t for t in problem(3, 2, 4, 16, 8, 5))
    leaves = [t.clone().requires_grad_() for t in (x, w, gu, down)]
    value = lambda *a: float((formula(*a, ids, ACT_SITU, 4) * dout).sum())  # noqa: E731
    grads = torch.autograd.grad((formula(*leaves, ids, ACT_SITU, 4) * dout).sum(), leaves)
    for i, g in enumerate(grads):
        at = g.abs().reshape(-1).argmax()
        step = [t.detach().clone() for t in leaves], [t.detach().clone() for t in leaves]
        step[0][i].view(-1)[at] += 1e-5
        step[1][i].view(-1)[at] -= 1e-5
        assert abs((value(*step[0]) - value(*step[1])) / 2e-5 - float(g.view(-1)[at])) < 1e-7


def test_a_training_step(cuda):
    """Norm, router, experts and back to the router's logits and the norm's inputs, in a graph too."""
    T, k, E, H, F = 96, 2, 8, 256, 128
    x, res, gu, down, _, _, dout = problem(T, k, E, H, F, 3)
    weight = (1 + R.normal((H,), 1, 0.1).float()).to(torch.bfloat16)
    router = R.normal((E, H), 2, H ** -0.5)
    logits64 = None
    on = {n: t.to(cuda) for n, t in dict(x=x, res=res, gu=gu, down=down, weight=weight, dout=dout).items()}
    total = (x.float() + res.float()).to(torch.bfloat16).double()
    normed64 = total / torch.sqrt(total.pow(2).mean(1, keepdim=True) + EPS) * weight.double()
    logits64 = normed64 @ router.double().t()
    logits = logits64.float().to(cuda)  # the router's own product is not under test
    ids = logits64.topk(k, dim=1).indices.to(torch.int32)

    def step():
        n = norm.residual_norm(on["x"], on["weight"], EPS, residual=on["res"])
        score = torch.sigmoid(logits).gather(1, ids.to(cuda).long())
        weights = (2.5 * score / score.sum(1, keepdim=True)).contiguous()
        out, saved = experts.forward(n.normed, ids.to(cuda), weights, on["gu"], on["down"], ACT_SWIGLU,
                                     residual=n.total)
        dnormed, dweights, dgu, ddown = experts.backward(on["dout"], saved, on["gu"], on["down"])
        _, counts, _, live = balance.balance_loss(logits, ids.to(cuda), 0.01)
        dlogits = balance.router_backward(logits, ids.to(cuda), counts, live, 0.01,
                                          dloss=torch.zeros((), device=cuda), dweights=dweights, scaling_factor=2.5)
        dx, dweight = norm.residual_norm_backward(dnormed, n.total, on["weight"], n.rstd, dtotal=on["dout"])
        return out, dgu, ddown, dlogits, dx, dweight

    got = step()
    leaves = [t.double().requires_grad_() for t in (gu, down, logits64, total, weight)]
    g64, d64, l64, t64, w64 = leaves
    n = t64 / torch.sqrt(t64.pow(2).mean(1, keepdim=True) + EPS) * w64
    score = torch.sigmoid(l64).gather(1, ids.long())
    out64 = t64 + formula(n, 2.5 * score / score.sum(1, keepdim=True), g64, d64, ids, ACT_SWIGLU, E)
    grads = torch.autograd.grad((out64 * dout.double()).sum(), leaves)
    assert relative(got[0], out64.detach()) <= 7 * 2.0 ** -8
    for a, b in zip(got[1:], grads):
        assert a.shape == b.shape and relative(a, b) <= 7 * 2.0 ** -8
    # captured (with the ids and the copies that the capture cannot make already there)
    ids_on = ids.to(cuda)
    score = torch.sigmoid(logits).gather(1, ids_on.long())
    weights = (2.5 * score / score.sum(1, keepdim=True)).contiguous()

    def captured():
        n = norm.residual_norm(on["x"], on["weight"], EPS, residual=on["res"])
        out, saved = experts.forward(n.normed, ids_on, weights, on["gu"], on["down"], ACT_SWIGLU, residual=n.total)
        dnormed, dweights, dgu, ddown = experts.backward(on["dout"], saved, on["gu"], on["down"])
        return (out, dweights, dgu, ddown,
                *norm.residual_norm_backward(dnormed, n.total, on["weight"], n.rstd, dtotal=on["dout"]))

    captured()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = captured()
    for turn in range(3):
        on["x"].copy_(R.normal((T, H), 30 + turn).to(cuda))
        want = [t.clone() for t in captured()]
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_no_row_at_all(cuda):
    """A batch whose routes all are of no expert: outputs are the residual, gradients 0."""
    x, res, gu, down, ids, w, dout = problem(5, 2, 3, 64, 32, 1)
    ids = torch.full_like(ids, 3).to(cuda)
    out, saved = experts.forward(x.to(cuda), ids, w.to(cuda), gu.to(cuda), down.to(cuda), ACT_SWIGLU,
                                 residual=res.to(cuda))
    assert torch.equal(out.cpu(), res)
    dx, dw, dgu, ddown = experts.backward(dout.to(cuda), saved, gu.to(cuda), down.to(cuda))
    assert not dx.any() and not dw.any() and not dgu.any() and not ddown.any()


def slopes(g, u, act):
    """The activation with its first and second derivatives, in 64 bits: v, (by g, by u), (gg, gu, uu)."""
    g, u = g.clone().requires_grad_(), u.clone().requires_grad_()
    v = activation(g, u, act)
    by_g, by_u = torch.autograd.grad(v.sum(), (g, u), create_graph=True)
    gg, gu = torch.autograd.grad(by_g.sum(), (g, u), retain_graph=True)
    uu, = torch.autograd.grad(by_u.sum(), u, materialize_grads=True)  # SwiGLU's is 0
    return v.detach(), (by_g.detach(), by_u.detach()), (gg, gu, uu)


@pytest.mark.parametrize("act", [ACT_SITU, ACT_SWIGLU])
@pytest.mark.parametrize("T,k,E,H,F", [(1, 2, 4, 64, 32), (7, 3, 5, 72, 40), (150, 2, 6, 264, 136), (600, 4, 8, 256, 128),
                                       (90, 16, 896, 128, 64)])
def test_each_value_within_its_roundings(cuda, act, T, k, E, H, F):
    """Each value of a layer's outputs and gradients against the formula step by step in 64 bits. An error of
    an input goes on by the magnitudes of the terms that it is in, and each step adds half a bf16 step of its
    own value and Z fp32 steps of its terms' magnitudes (tests/_grouped.py; the activation, which
    is within 2^-12 of its terms for these values, counts as a bf16 step more). Twice the sum, for the
    products of errors."""
    x, res, gu, down, ids, w, dout = problem(T, k, E, H, F, T + 1)
    ids = ids.clone()
    if T > 1:
        ids[0, 1], ids[1, 0] = ids[0, 0], E
    on = [t.to(cuda) for t in (x, ids, w, gu, down)]
    out, saved = experts.forward(*on, act, residual=res.to(cuda))
    got = dict(zip(("dx", "dw", "dgu", "ddown"), experts.backward(dout.to(cuda), saved, on[3], on[4])), out=out)
    half, step = 2.0 ** -8, 2.0 ** -23
    x, res, gu, down, w, dout = (t.double() for t in (x, res, gu, down, w, dout))
    keep = live_routes(ids, E)
    zeros = lambda *s: torch.zeros(s, dtype=torch.float64)  # noqa: E731
    want = {n: zeros(*s) for n, s in dict(y=(T, H), dx=(T, H), dw=(T, k), dgu=(E, 2 * F, H), ddown=(E, H, F)).items()}
    err = {n: torch.zeros_like(t) for n, t in want.items()}
    for e in range(E):
        t, r = torch.where((ids == e) & keep)
        if len(t) == 0:
            continue
        n, wr = len(t), w[t, r][:, None]
        z = x[t] @ gu[e].t()
        ez = half * z.abs() + H * step * (x[t].abs() @ gu[e].abs().t())
        (g, u), (eg, eu) = z.chunk(2, 1), ez.chunk(2, 1)
        v, (by_g, by_u), (gg, gu_, uu) = slopes(g, u, act)
        ev = by_g.abs() * eg + by_u.abs() * eu + half * v.abs()
        h, eh = wr * v, wr * ev + half * (wr * v).abs()
        y, ey = h @ down[e].t(), eh @ down[e].abs().t() + F * step * (h.abs() @ down[e].abs().t())
        want["y"].index_add_(0, t, y)
        err["y"].index_add_(0, t, ey + half * y.abs())
        d = dout[t]
        dh = d @ down[e]
        edh = half * dh.abs() + H * step * (d.abs() @ down[e].abs())
        want["dw"][t, r] = (dh * v).sum(1)
        err["dw"][t, r] = (edh * v.abs() + dh.abs() * ev + F * step * (dh * v).abs()).sum(1)
        dz = torch.cat([wr * dh * by_g, wr * dh * by_u], 1)
        edz = torch.cat([wr * (edh * by_g.abs() + dh.abs() * (gg.abs() * eg + gu_.abs() * eu)),
                         wr * (edh * by_u.abs() + dh.abs() * (gu_.abs() * eg + uu.abs() * eu))], 1)
        edz = edz + 2 * half * dz.abs()
        want["dgu"][e], want["ddown"][e] = dz.t() @ x[t], d.t() @ h
        err["dgu"][e] = edz.t() @ x[t].abs() + n * step * (dz.abs().t() @ x[t].abs())
        err["ddown"][e] = d.abs().t() @ eh + n * step * (d.abs().t() @ h.abs())
        rows, size = dz @ gu[e], dz.abs() @ gu[e].abs()
        want["dx"].index_add_(0, t, rows)
        err["dx"].index_add_(0, t, edz @ gu[e].abs() + 2 * F * step * size + half * rows.abs())
    for name in ("y", "dx"):  # the sum's own rounding
        err[name] += (half + k * step) * want[name].abs()
    want["out"] = want["y"] + res
    err["out"] = err["y"] + half * want["out"].abs()
    for name, value in got.items():
        off, most = (value.cpu().double() - want[name]).abs(), 2 * err[name] + 2.0 ** -130
        assert (off <= most).all(), (name, float((off / most).max()))
