"""Forms of the training operators and the norm that only the C entry points reach (what may be NULL is), and
other bounds of the activation than the layer's, on the GPU.

Bounds: as in test_gpu_gated.py, with what other bounds of SiTU add: y = g / beta is within 2 u of itself,
and the exponent of 1 - tanh(y)^2, -2 |y| log2(e), so within 4 u: the slope, which goes by e^(-2 |y|), is
within 8 |y| u of itself more.
"""
import pytest
import torch

import _grouped as R
from moonshine_amd import experts, norm
from moonshine_amd._lib import lib
from moonshine_amd.synth import ACT_SITU, ACT_SWIGLU
from test_gpu_gated import U, values

pytestmark = pytest.mark.gpu

EPS = 1e-5


def at(t):
    return None if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def gated(gu, offsets, route, weights, routes, act, beta=4.0, linear=25.0):
    out = torch.full((gu.shape[0], gu.shape[1] // 2), 7.0, dtype=torch.bfloat16, device=gu.device)
    assert lib().k3_moe_gated_rows_bf16(at(out), at(gu), at(offsets), at(route), at(weights), gu.shape[0], routes,
                                        offsets.shape[0] - 1, out.shape[1], act, beta, linear, stream())
    return out


def gated_backward(dh, gu, offsets, route, weights, routes, act, dweights=None):
    out = torch.full_like(gu, 7.0)
    assert lib().k3_moe_gated_rows_backward_bf16(at(out), at(dweights), at(dh), at(gu), at(offsets), at(route),
                                                 at(weights), gu.shape[0], routes, offsets.shape[0] - 1, dh.shape[1],
                                                 act, 4.0, 25.0, stream())
    return out


@pytest.mark.parametrize("act", [ACT_SITU, ACT_SWIGLU])
def test_gated_without_an_index_or_weights(cuda, act):
    """No index is the rows' order, no weights are ones: the bits of the call that spells them out."""
    rows, F, used = 37, 520, 33
    gu, dh = R.normal((rows, 2 * F), 1, 3.0).to(cuda), R.normal((rows, F), 2).to(cuda)
    o = torch.tensor([0, 5, 5, used], dtype=torch.int32, device=cuda)
    order = torch.arange(rows, dtype=torch.int32, device=cuda)
    w = torch.rand((rows, 1), generator=torch.Generator().manual_seed(3)).to(cuda)
    for weights in (w, torch.ones_like(w)):
        full = experts.gated(gu, o, order, weights, act)[:used]
        back, dw = experts.gated_backward(dh, gu, o, order, weights, act)
        for route in (order, None):
            for given in (weights, None) if weights is not w else (weights,):
                routes = rows if given is not None or route is not None else 0
                got = gated(gu, o, route, given, routes, act)
                assert torch.equal(got[:used], full) and (got[used:] == 7).all()
                got = gated_backward(dh, gu, o, route, given, routes, act)  # no gradient by the weights
                assert torch.equal(got[:used], back[:used]) and (got[used:] == 7).all()
                dweights = torch.full((rows,), 7.0, device=cuda)
                got = gated_backward(dh, gu, o, route, given, rows, act, dweights)
                assert torch.equal(got[:used], back[:used]) and torch.equal(dweights, dw.view(-1))
                assert not dweights[used:].any() and dweights[:used].all()


def test_gated_routes_out_of_range(cuda):
    """A route that is none of `routes` has weight 0, and no gradient is written for it."""
    rows, F, routes = 9, 64, 5
    gu, dh = R.normal((rows, 2 * F), 1).to(cuda), R.normal((rows, F), 2).to(cuda)
    o = torch.tensor([0, rows], dtype=torch.int32, device=cuda)
    route = torch.tensor([0, 5, 1, -1, 2, 1 << 30, 3, 6, 4], dtype=torch.int32, device=cuda)
    bad = (route < 0) | (route >= routes)
    room = torch.full((routes + 8,), 7.0, device=cuda)
    w = room[4:4 + routes].clone().uniform_(0.5, 1.5)
    got = gated(gu, o, route, w, routes, ACT_SITU)
    assert not got[bad].any() and got[~bad].any(1).all()
    got = gated_backward(dh, gu, o, route, w, routes, ACT_SITU, room[4:4 + routes])
    assert not got[bad].any() and got[~bad].any(1).all()
    assert (room[:4] == 7).all() and (room[4 + routes:] == 7).all()
    want, dw = experts.gated_backward(dh[~bad].contiguous(), gu[~bad].contiguous(),
                                      torch.tensor([0, routes], dtype=torch.int32, device=cuda), route[~bad].contiguous(),
                                      w.view(-1, 1), ACT_SITU)
    assert torch.equal(got[~bad], want) and torch.equal(room[4:4 + routes], dw.view(-1))


@pytest.mark.parametrize("beta,linear", [(0.5, 2.0), (1.0, 1.0), (30.0, 0.25), (2.0 ** -10, 2.0 ** 10), (1e20, 1e-3)])
def test_other_bounds_of_the_activation(cuda, beta, linear):
    n, F = 64, 256
    gu, dh = R.normal((n, 2 * F), 1, 3.0), R.normal((n, F), 2)
    g, u, d = gu.double()[:, :F], gu.double()[:, F:], dh.double()
    o = torch.tensor([0, n], dtype=torch.int32, device=cuda)
    r, ones = torch.arange(n, dtype=torch.int32, device=cuda), torch.ones((n, 1), device=cuda)
    b, c = (float(torch.tensor(v, dtype=torch.float32)) for v in (beta, linear))
    v, by_g, by_u, vs, gs, us = values(g, u, ACT_SITU, b, c)
    terms = 64 + 4 * g.abs() + 4 * u.abs() + 8 * g.abs() / b + 8 * u.abs() / c

    def check(got, want, size):
        slack = terms * U * size + 2.0 ** -120 * (1 + g.abs()) * (1 + u.abs())
        bound = slack + 2.0 ** -8 * (want.abs() + slack) + 2.0 ** -133
        assert ((got.cpu().double() - want).abs() <= bound).all()

    check(experts.gated(gu.to(cuda), o, r, ones, ACT_SITU, beta, linear), v, vs)
    dgu, dw = experts.gated_backward(dh.to(cuda), gu.to(cuda), o, r, ones, ACT_SITU, beta, linear)
    check(dgu[:, :F], d * by_g, d.abs() * gs)
    check(dgu[:, F:], d * by_u, d.abs() * us)
    size = (d.abs() * vs * (F + terms)).sum(1) * U
    assert ((dw.cpu().double()[:, 0] - (d * v).sum(1)).abs() <= size + 2.0 ** -120).all()


@pytest.mark.parametrize("rows,cols", [(5, 128), (9, 2048), (6, 4096), (61, 7168), (3, 16384), (2, 32768)])
def test_norm_of_parts(cuda, rows, cols):
    """Each output alone, the others NULL, has the bits that it has among all."""
    x, res = R.normal((rows, cols), 1).to(cuda), R.normal((rows, cols), 2).to(cuda)
    w = (1 + R.normal((cols,), 3, 0.2).float()).to(torch.bfloat16).to(cuda)
    for residual in (res, None):
        full = norm.residual_norm(x, w, EPS, residual=residual, encode=True)
        for wanted in ("normed", "codes", "rstd", "total"):
            if wanted == "total" and residual is None:
                continue
            total = None if residual is None else torch.empty_like(x)
            normed = torch.empty_like(x) if wanted == "normed" else None
            codes, scales = (torch.empty_like(t) for t in (full.codes, full.scales)) if wanted == "codes" else (None, None)
            rstd = torch.empty_like(full.rstd) if wanted == "rstd" else None
            assert lib().k3_moe_residual_norm_bf16(at(total), at(normed), at(codes), at(scales), at(rstd), at(x),
                                                   at(residual), at(w), rows, cols, EPS, stream())
            for got, want in ((total, full.total), (normed, full.normed), (codes, full.codes), (scales, full.scales),
                              (rstd, full.rstd)):
                assert got is None or torch.equal(got.view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("E,k", [(7, 3), (70, 9), (896, 16), (1024, 32)])
@pytest.mark.parametrize("residual", [True, False])
def test_combine_of_many_routes(cuda, E, k, residual):
    """Up to 32 routes of a token, in rank order, each step rounded to fp32: bit for bit."""
    T, H = 5, 1032
    ids = R.routes(T, k, E, k)
    ids[1, k - 1] = ids[1, 0]
    ids[2, 0] = E
    ids[3, k // 2] = -1
    live = (ids >= 0) & (ids < E)
    live[1, k - 1] = False
    y = R.normal((T * k, H), 1)
    y[~live.view(-1)] = float("nan")
    res = R.normal((T, H), 2) if residual else None
    w = torch.rand((T, k), generator=torch.Generator().manual_seed(3))
    for weights in (None, w):
        total = torch.zeros((T, H))
        for r in range(k):
            term = y.float().view(T, k, H)[:, r] * (1.0 if weights is None else weights[:, r, None])
            total = torch.where(live[:, r, None], total + term, total)
        want = total.to(torch.bfloat16)
        if residual:
            want = (res.float() + want.float()).to(torch.bfloat16)
        got = experts.combine(y.to(cuda), ids.to(cuda), E, residual=None if res is None else res.to(cuda),
                              weights=None if weights is None else weights.to(cuda))
        assert torch.equal(got.cpu(), want)
