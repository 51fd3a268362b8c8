"""Products grouped by expert and their gradients on the GPU, against 64-bit forms
(tests/_grouped.py, where the bounds are derived)."""
import pytest
import torch

import _grouped as R
from moonshine_amd import grouped

pytestmark = pytest.mark.gpu

# (tokens, top_k, experts, N, K, skew): one row, one tile of each class and its edges, widths that
# are no whole tiles or stages, experts without rows, many experts
SHAPES = [
    (1, 1, 1, 8, 8, 0.0),
    (1, 4, 64, 1024, 2048, 0.0),
    (2, 1, 3, 256, 64, 0.0),
    (33, 2, 5, 264, 72, 0.0),
    (65, 1, 2, 40, 520, 3.0),
    (129, 3, 4, 512, 136, 0.0),
    (300, 1, 1, 328, 200, 0.0),
    (513, 2, 2, 256, 256, 0.0),
    (700, 4, 40, 144, 1000, 2.0),
    (257, 8, 896, 64, 128, 0.5),
    (1345, 1, 1, 8, 456, 0.0),
]


def laid_out(T, k, E, skew, seed, cuda):
    ids = R.routes(T, k, E, seed, skew)
    p = grouped.route_plan(ids.to(cuda), E)
    return ids, p, R.plan(ids, E)


def equal(got, want):
    torch.testing.assert_close(got.cpu().double(), want.to(got.dtype).double(), rtol=0, atol=0)


@pytest.mark.parametrize("T,k,E,N,K,skew", SHAPES)
def test_plan_and_exact_sums(cuda, T, k, E, N, K, skew):
    """Every direction, with and without indices, on whole numbers: bit for bit."""
    ids, p, (offsets, token, route) = laid_out(T, k, E, skew, T + N, cuda)
    rows = T * k
    assert torch.equal(p.offsets.cpu(), offsets)
    assert torch.equal(p.token_index.cpu(), token) and torch.equal(p.route_index.cpu(), route)
    w = R.whole((E, N, K), 1)
    x, xr = R.whole((T, K), 2), R.whole((rows, K), 3)
    dy, dyr = R.whole((T, N), 4), R.whole((rows, N), 5)
    wc = w.to(cuda)
    print("product", flush=True)
    equal(grouped.product(x.to(cuda), wc, p.offsets, index=p.token_index),
          R.by_rows(x, w, offsets, token, False)[0])
    want = R.by_rows(xr, w, offsets, None, False)[0]
    slots = torch.empty_like(want)
    slots[route.long()] = want
    equal(grouped.product(xr.to(cuda), wc, p.offsets, to=p.route_index), slots)
    print("input gradient", flush=True)
    equal(grouped.input_gradient(dy.to(cuda), wc, p.offsets, index=p.token_index),
          R.by_rows(dy, w, offsets, token, True)[0])
    want = R.by_rows(dyr, w, offsets, None, True)[0]
    slots = torch.empty_like(want)
    slots[route.long()] = want
    equal(grouped.input_gradient(dyr.to(cuda), wc, p.offsets, to=p.route_index), slots)
    for dtype in (torch.float32, torch.bfloat16):
        print("weight gradient", dtype, flush=True)
        equal(grouped.weight_gradient(dyr.to(cuda), x.to(cuda), p.offsets, x_index=p.token_index, dtype=dtype),
              R.by_weights(dyr, x, offsets, None, token)[0])
        equal(grouped.weight_gradient(dy.to(cuda), xr.to(cuda), p.offsets, dy_index=p.token_index, dtype=dtype),
              R.by_weights(dy, xr, offsets, token, None)[0])


@pytest.mark.parametrize("T,k,E,N,K,skew", [(61, 2, 8, 264, 1096, 1.0), (900, 4, 16, 512, 2048, 2.0)])
def test_within_the_bound(cuda, T, k, E, N, K, skew):
    ids, p, (offsets, token, route) = laid_out(T, k, E, skew, 7, cuda)
    w, x, dy = R.normal((E, N, K), 1, 0.02), R.normal((T, K), 2), R.normal((T * k, N), 3, 1e-3)
    got = grouped.product(x.to(cuda), w.to(cuda), p.offsets, index=p.token_index)
    out, size = R.by_rows(x, w, offsets, token, False)
    assert ((got.cpu().double() - out).abs() <= R.bound(out, size, K, torch.bfloat16)).all()
    got = grouped.input_gradient(dy.to(cuda), w.to(cuda), p.offsets)
    out, size = R.by_rows(dy, w, offsets, None, True)
    assert ((got.cpu().double() - out).abs() <= R.bound(out, size, N, torch.bfloat16)).all()
    longest = int((offsets[1:] - offsets[:-1]).max())
    for dtype in (torch.float32, torch.bfloat16):
        got = grouped.weight_gradient(dy.to(cuda), x.to(cuda), p.offsets, x_index=p.token_index, dtype=dtype)
        out, size = R.by_weights(dy, x, offsets, None, token)
        assert ((got.cpu().double() - out).abs() <= R.bound(out, size, longest, dtype)).all()
