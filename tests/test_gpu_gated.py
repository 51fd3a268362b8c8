"""The gated activation of expert rows with its gradient, and the sum of a token's rows, on the GPU against
64-bit forms.

Bounds: u = 2^-24. exp2 and the reciprocal of the hardware are within 1 ulp (2 u), the exponent's
argument within 2 u |g|, tanh within 16 u; a product of up to eight such factors and their
products' roundings is within (64 + 4 |g| + 4 |u|) u of its terms' magnitudes. Scores under
2^-126 are 0. A bf16 output adds 2^-8 of itself, a sum of F terms F u of their magnitudes.
"""
import pytest
import torch

import _grouped as R
from moonshine_amd import experts, grouped
from moonshine_amd.synth import ACT_SITU, ACT_SWIGLU

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BETA, LINEAR = 4.0, 25.0


def values(g, u, act, beta=BETA, linear=LINEAR):
    """act, its slopes by g and u, and the magnitudes of the three's terms, in 64 bits."""
    s, rest = torch.sigmoid(g), torch.sigmoid(-g)
    if act == ACT_SWIGLU:
        v = g * s * u
        return v, s * (1 + g * rest) * u, g * s, v.abs(), s * (1 + (g * rest).abs()) * u.abs(), (g * s).abs()
    a, c = beta * torch.tanh(g / beta), linear * torch.tanh(u / linear)
    sg, su = 1 / torch.cosh(g / beta) ** 2, 1 / torch.cosh(u / linear) ** 2
    by_g = s * (sg + a * rest) * c
    return a * s * c, by_g, a * s * su, (a * s * c).abs(), s * (sg + (a * rest).abs()) * c.abs(), (a * s * su).abs()


def check(got, want, size, g, u, scale):
    got, slack = got.cpu().double(), (64 + 4 * g.abs() + 4 * u.abs()) * U * size * scale
    slack = slack + 2.0 ** -120 * scale * (1 + g.abs()) * (1 + u.abs())
    bound = slack + 2.0 ** -8 * (want.abs() + slack) + 2.0 ** -133
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("act", [ACT_SITU, ACT_SWIGLU])
@pytest.mark.parametrize("T,k,E,F", [(1, 1, 1, 8), (3, 2, 4, 24), (37, 6, 40, 1024), (130, 3, 8, 520), (5, 2, 3, 4104)])
def test_rows_and_gradients(cuda, act, T, k, E, F):
    ids = R.routes(T, k, E, T)
    p = grouped.route_plan(ids.to(cuda), E)
    _, _, route = R.plan(ids, E)
    rows = T * k
    gu, dh = R.normal((rows, 2 * F), 1, 3.0), R.normal((rows, F), 2, 1e-3)
    weights = torch.rand((T, k), generator=torch.Generator().manual_seed(3)) * 2
    g, u = gu.double()[:, :F], gu.double()[:, F:]
    w = weights.double().view(-1)[route.long()][:, None]
    v, by_g, by_u, vs, gs, us = values(g, u, act)
    h = experts.gated(gu.to(cuda), p.offsets, p.route_index, weights.to(cuda), act, BETA, LINEAR)
    check(h, w * v, vs, g, u, w)
    dgu, dw = experts.gated_backward(dh.to(cuda), gu.to(cuda), p.offsets, p.route_index, weights.to(cuda), act, BETA,
                                     LINEAR)
    d = dh.double()
    check(dgu[:, :F], d * w * by_g, gs, g, u, (d * w).abs())
    check(dgu[:, F:], d * w * by_u, us, g, u, (d * w).abs())
    want = torch.zeros(rows, dtype=torch.float64)
    want[route.long()] = (d * v).sum(1)
    size = torch.zeros(rows, dtype=torch.float64)
    size[route.long()] = (d.abs() * vs * (F + 128 + 4 * g.abs() + 4 * u.abs())).sum(1) * U
    assert ((dw.cpu().double().view(-1) - want).abs() <= size + 2.0 ** -120).all()


@pytest.mark.parametrize("act", [ACT_SITU, ACT_SWIGLU])
def test_every_magnitude(cuda, act):
    """From the smallest bf16 values to large ones of both signs, where the slopes nearly vanish too."""
    m = torch.cat([2.0 ** torch.arange(-40.0, 7.0, 0.5), torch.tensor([0.0, 1.278, 1.2785, 20.0, 87.0, 89.0, 100.0])])
    m = torch.cat([m, -m]).to(torch.bfloat16)
    n = len(m)
    F = -(-n // 8) * 8
    grid = torch.zeros((n, 2 * F), dtype=torch.bfloat16)
    grid[:, :n], grid[:, F:F + n] = m[:, None], m[None, :]
    o = torch.tensor([0, n], dtype=torch.int32, device=cuda)
    r = torch.arange(n, dtype=torch.int32, device=cuda)
    ones = torch.ones((n, 1), device=cuda)
    g, u = grid.double()[:, :F], grid.double()[:, F:]
    v, by_g, by_u, vs, gs, us = values(g, u, act)
    check(experts.gated(grid.to(cuda), o, r, ones, act, BETA, LINEAR), v, vs, g, u, 1.0)
    dh = torch.ones((n, F), dtype=torch.bfloat16)
    dgu, _ = experts.gated_backward(dh.to(cuda), grid.to(cuda), o, r, ones, act, BETA, LINEAR)
    check(dgu[:, :F], by_g, gs, g, u, 1.0)
    check(dgu[:, F:], by_u, us, g, u, 1.0)


@pytest.mark.parametrize("act", [ACT_SITU, ACT_SWIGLU])
def test_slopes_are_the_differences_of_the_values(cuda, act):
    """Of the 64-bit form that the kernels are held to, by central differences."""
    g, u = (R.normal((4, 64), s, 3.0).double() for s in (1, 2))
    e = 1e-5
    _, by_g, by_u, _, _, _ = values(g, u, act)
    d = lambda dg, du: values(g + dg, u + du, act)[0]  # noqa: E731
    torch.testing.assert_close((d(e, 0) - d(-e, 0)) / (2 * e), by_g, rtol=1e-7, atol=1e-7)
    torch.testing.assert_close((d(0, e) - d(0, -e)) / (2 * e), by_u, rtol=1e-7, atol=1e-7)


def test_dropped_routes(cuda):
    """Repeated ids and ids of no expert: no row, gradient 0, and rows behind the last as they were."""
    E, F, T, k = 4, 16, 6, 3
    ids = torch.tensor([[0, 0, 1], [3, 9, 3], [-1, -1, -1], [2, 1, 0], [1, 1, 1], [0, 3, 2]], dtype=torch.int32)
    p = grouped.route_plan(ids.to(cuda), E)
    offsets, token, route = R.plan(ids, E)
    used = len(route)
    assert used < T * k and torch.equal(p.offsets.cpu(), offsets)
    assert torch.equal(p.route_index.cpu()[:used], route) and torch.equal(p.token_index.cpu()[:used], token)
    gu, dh = R.normal((T * k, 2 * F), 1), R.normal((T * k, F), 2)
    gu[used:] = float("nan")
    weights = torch.rand((T, k)).to(cuda)
    out = torch.full((T * k, F), 7.0, dtype=torch.bfloat16, device=cuda)
    experts.gated(gu.to(cuda), p.offsets, p.route_index, weights, ACT_SWIGLU, out=out)
    assert (out[used:] == 7).all() and out[:used].isfinite().all()
    back = torch.full((T * k, 2 * F), 7.0, dtype=torch.bfloat16, device=cuda)
    _, dw = experts.gated_backward(dh.to(cuda), gu.to(cuda), p.offsets, p.route_index, weights, ACT_SWIGLU, out=back)
    assert (back[used:] == 7).all() and back[:used].isfinite().all()
    live = torch.zeros(T * k, dtype=torch.bool)
    live[route.long()] = True
    dw = dw.cpu().view(-1)
    assert (dw[~live] == 0).all() and (dw[live] != 0).all()
    # in the place of gate/up
    room = gu.to(cuda)
    experts.gated_backward(dh.to(cuda), room, p.offsets, p.route_index, weights, ACT_SWIGLU, out=room)
    assert torch.equal(room[:used], back[:used]) and room[used:].isnan().all()
    # the sum leaves them out, whatever their rows hold
    y = R.normal((T * k, 24), 3)
    y[~live] = float("nan")
    res = R.normal((T, 24), 4)
    for w in (None, weights):
        got = experts.combine(y.to(cuda), ids.to(cuda), E, residual=res.to(cuda), weights=w)
        v = y.float().view(T, k, -1).clone()
        v[~live.view(T, k)] = 0
        total = torch.zeros((T, 24))
        for r in range(k):  # in rank order, each step rounded to fp32
            total = total + v[:, r] * (1.0 if w is None else w.cpu()[:, r, None])
        assert torch.equal(got.cpu(), (res.float() + total.to(torch.bfloat16).float()).to(torch.bfloat16))
    none = experts.combine(y.to(cuda), torch.full_like(ids, E).to(cuda), E)
    assert (none == 0).all()


def test_infinities_and_nan_stay_in_their_row(cuda):
    F = 32
    gu = R.normal((4, 2 * F), 1)
    gu[1, 3], gu[2, F + 5], gu[2, 7] = float("nan"), float("inf"), -float("inf")
    o = torch.tensor([0, 4], dtype=torch.int32, device=cuda)
    r, w = torch.arange(4, dtype=torch.int32, device=cuda), torch.ones((4, 1), device=cuda)
    h = experts.gated(gu.to(cuda), o, r, w, ACT_SWIGLU).cpu()
    want = (gu.double()[:, :F] * torch.sigmoid(gu.double()[:, :F]) * gu.double()[:, F:])
    assert torch.equal(h.isnan(), want.isnan()) and torch.equal(h.isinf(), want.isinf())
    assert h[0].isfinite().all() and h[3].isfinite().all()


def test_past_32_bits(cuda):
    """Rows past 4 GiB have the bits that they have alone: gated rows, their gradient, and their sum."""
    rows, F, last = 65600, 32768, 2
    offsets = torch.tensor([0, rows], dtype=torch.int32, device=cuda)
    alone = torch.tensor([0, last], dtype=torch.int32, device=cuda)
    gu = torch.zeros((rows, 2 * F), dtype=torch.bfloat16, device=cuda)
    gu[-last:] = R.normal((last, 2 * F), 1).to(cuda)
    route = torch.arange(rows, dtype=torch.int32, device=cuda)
    w = torch.rand((rows, 1), generator=torch.Generator().manual_seed(2)).to(cuda)
    want = experts.gated(gu[-last:].clone(), alone, route[:last], w[-last:].clone(), ACT_SITU)
    h = experts.gated(gu, offsets, route, w, ACT_SITU)
    assert torch.equal(h[-last:], want) and not h[:-last].any()
    dgu, dw = experts.gated_backward(want, gu[-last:].clone(), alone, route[:last], w[-last:].clone(), ACT_SITU)
    big, bdw = experts.gated_backward(h, gu, offsets, route, w, ACT_SITU, out=gu)
    assert torch.equal(big[-last:], dgu) and not big[:-last].any()
    assert torch.equal(bdw[-last:], dw) and not bdw[:-last].any()
    del gu, big
    ids = torch.tensor([[0, 1]], dtype=torch.int32, device=cuda).expand(rows // 2, 2).contiguous()
    out = experts.combine(h, ids, 2)
    assert torch.equal(out[-1:], experts.combine(want, ids[:1].clone(), 2)) and not out[:-1].any()
