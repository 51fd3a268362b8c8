"""Balance loss, per-expert counts and the router's gradient on the GPU, against
the formulas in 64 bits and their differences.

u = 2^-24. A score (exp2 and the reciprocal 1 ulp each, the exponent's rounding
|x| u, three roundings) is within (8 + 2 |x|) u of itself, and so is 1 - score;
|x| <= 20 here: 48 u. Z adds at most 1024 of them (16 a lane, then 6 levels: 22 u),
a share 1 more division: 48 + 48 + 22 + 2 = 120 u. A mean adds up to 4096 tokens in
runs (at most 64 + 8 + 16 + 16 additions): 230 u of itself; the loss sums
16 positive terms a lane of 6 roundings: 260 u.
"""
import pytest
import torch

from moonshine_amd import balance

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def forward64(logits, ids, coef, segments, mask):
    """loss, counts, mean scores, live tokens; differentiable."""
    T, E = logits.shape
    k = ids.shape[1]
    live = torch.ones(T, dtype=torch.float64) if mask is None else (mask.cpu() != 0).double()
    first = torch.stack([(ids[:, r:r + 1] != ids[:, :r]).all(1) for r in range(k)], 1)
    ok = first & (ids >= 0) & (ids < E)
    hits = torch.zeros((T, E), dtype=torch.float64)
    for r in range(k):
        t = torch.where(ok[:, r])[0]
        hits[t, ids[t, r].long()] = 1
    sig = torch.sigmoid(logits)
    z = sig.sum(1, keepdim=True)
    p = torch.where(z > 0, sig / z.clamp_min(1e-300), torch.zeros_like(sig))
    n = live.view(segments, -1).sum(1)
    d = n.clamp_min(1)[:, None]
    mean = (p * live[:, None]).view(segments, -1, E).sum(1) / d
    counts = (hits * live[:, None]).view(segments, -1, E).sum(1)
    f = torch.where(n[:, None] > 0, counts * E / (k * d), 0.0)
    return coef / segments * (f * mean).sum(), counts, mean, n, live, ok, sig


def weights64(sig, ids, ok, scale):
    picked = torch.where(ok, sig.gather(1, ids.long().clamp(0, sig.shape[1] - 1)), 0.0)
    return scale * picked / (1e-20 + picked.sum(1, keepdim=True))


def case(T, E, k, seed, std=1.7):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn((T, E), generator=g) * std).clamp(-20, 20)
    ids = torch.sigmoid(logits).topk(k, 1).indices.to(torch.int32)
    return logits, ids, torch.randn((T, k), generator=g)


def check(cuda, logits, ids, dw, segments, mask, coef=0.3, scale=2.5, dloss=None):
    d = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    x = logits.double().requires_grad_()
    loss, counts, mean, n, live, ok, sig = forward64(x, ids, coef, segments, mask)
    got = balance.balance_loss(d(logits), d(ids), coef, segments=segments, mask=d(mask))
    assert torch.equal(got[1].cpu().double(), counts)
    assert torch.equal(got[3].cpu().double(), n)
    off = (got[2].cpu().double() - mean).abs()
    assert (off <= 230 * U * mean + 1e-38).all(), (off / mean).max() / U
    assert abs(got[0].item() - loss.item()) <= 260 * U * abs(loss.item()) + 1e-38
    total = loss * (1.0 if dloss is None else dloss)
    if dw is not None:
        total = total + (weights64(sig, ids, ok, scale) * dw.double() * live[:, None]).sum()
    (want,) = torch.autograd.grad(total, x)
    grad = balance.router_backward(
        d(logits), d(ids), got[1], got[3], coef, segments=segments, mask=d(mask),
        dloss=None if dloss is None else torch.tensor(dloss, device=cuda), dweights=d(dw),
        scaling_factor=scale).cpu().double()
    assert (grad[live == 0] == 0).all()
    # size of the terms that the gradient is the difference of, each to 400 u (the scores' 48 in
    # each of up to 4 factors, Z's and the mean's 120, the products' and the sums' roundings)
    T, E = logits.shape
    k = ids.shape[1]
    sig = sig.detach()
    f = counts.repeat_interleave(T // segments, 0) * E / (k * n.clamp_min(1)).repeat_interleave(T // segments)[:, None]
    share = abs(coef * (1.0 if dloss is None else dloss)) / segments / n.clamp_min(1).repeat_interleave(T // segments)
    z = sig.sum(1, keepdim=True).clamp_min(1e-300)
    size = share[:, None] / z * (f + (f * sig).sum(1, keepdim=True) / z)
    if dw is not None:
        picked = torch.where(ok, sig.gather(1, ids.long().clamp(0, E - 1)), 0.0)
        den = 1e-20 + picked.sum(1, keepdim=True)
        part = scale / den * (dw.double().abs() + (dw.double().abs() * picked).sum(1, keepdim=True) / den)
        for r in range(k):
            t = torch.where(ok[:, r])[0]
            size[t, ids[t, r].long()] += part[t, r]
    bound = 400 * U * size * sig * (1 - sig) + 1e-38
    off = (grad - want.detach()).abs() * live[:, None]
    assert (off <= bound).all(), (off / bound).max()
    return got, grad


@pytest.mark.parametrize("E,k", [(1, 1), (8, 3), (63, 4), (64, 4), (65, 2), (128, 8), (200, 32),
                                 (512, 5), (896, 16), (1024, 32)])
@pytest.mark.parametrize("T", [1, 2, 7, 40, 300])
def test_one_segment(cuda, T, E, k):
    logits, ids, dw = case(T, E, k, T + E)
    check(cuda, logits, ids, dw, 1, None)


@pytest.mark.parametrize("segments,length,E,k", [(3, 17, 64, 4), (2, 1, 16, 2), (40, 9, 130, 6),
                                                 (300, 5, 24, 3), (5, 333, 64, 4), (30, 144, 1000, 8),
                                                 (70, 40, 64, 6)])
def test_masked_segments(cuda, segments, length, E, k):
    """Padded sequences: one whole, one empty, one of holes; a loss for each."""
    T = segments * length
    logits, ids, dw = case(T, E, k, T + E)
    g = torch.Generator().manual_seed(T)
    lens = torch.randint(0, length + 1, (segments, 1), generator=g)
    lens[0], lens[-1] = length, 0
    mask = (torch.arange(length)[None] < lens).to(torch.uint8)
    mask[0, ::3] = 0 if length > 2 else 1
    mask = mask.reshape(-1) * 5      # any value but 0 is live
    check(cuda, logits, ids, dw, segments, mask, dloss=-0.7)
    check(cuda, logits, ids, None, segments, mask)
    check(cuda, logits, ids, dw, segments, mask.bool())


def test_long_batch(cuda):
    logits, ids, dw = case(4096, 256, 8, 5)
    check(cuda, logits, ids, dw, 1, None)
    check(cuda, logits, ids, dw, 4, None)


def test_invalid_and_repeated_ids(cuda):
    logits, ids, dw = case(50, 32, 4, 9)
    ids[::3, 2] = ids[::3, 0]
    ids[::4, 1] = 32
    ids[::5, 3] = -1
    ids[7] = 100
    check(cuda, logits, ids, dw, 1, None)


def test_all_masked_and_dead_rows(cuda):
    """No live token: loss and gradient 0. Scores of 0 throughout (-inf): no NaN."""
    logits, ids, dw = case(12, 16, 2, 3)
    got, grad = check(cuda, logits, ids, dw, 2, torch.zeros(12, dtype=torch.uint8))
    assert got[0].item() == 0 and (grad == 0).all() and (got[2] == 0).all()
    logits[3] = -float("inf")
    logits[5, 2:9] = -float("inf")
    logits[6, 1] = float("inf")
    d = lambda t: t.to(cuda)  # noqa: E731
    loss, counts, mean, live = balance.balance_loss(d(logits), d(ids), 1.0)
    grad = balance.router_backward(d(logits), d(ids), counts, live, 1.0, dweights=d(dw))
    assert torch.isfinite(loss) and torch.isfinite(mean).all() and torch.isfinite(grad).all()
    assert (grad[3] == 0).all() and (grad[5, 2:9] == 0).all() and grad[6, 1] == 0
    # a NaN stays in its row's gradient
    logits[8, 4] = float("nan")
    grad = balance.router_backward(d(logits), d(ids), counts, live, 1.0, dweights=d(dw))
    keep = torch.arange(12, device=cuda) != 8
    assert torch.isnan(grad[8]).any() and torch.isfinite(grad[keep]).all()


def test_gradient_against_differences(cuda):
    """The 64-bit gradient against central differences of the 64-bit loss (h = 1e-5: the truncation
    h^2 and the cancellation 1e-16 / h are both under 1e-9 of these values of order 1), and the
    kernel's along it: fp32 losses at a step of 2^-6 have 260 u / 2^-6 of noise and a relative
    truncation of (2^-6)^2."""
    T, E, k = 6, 10, 2
    logits, ids, _ = case(T, E, k, 21)
    x = logits.double().requires_grad_()
    loss = forward64(x, ids, 1.0, 2, None)[0]
    (grad,) = torch.autograd.grad(loss, x)
    h = 1e-5
    for t, e in ((0, 0), (3, 7), (5, 9)):
        step = torch.zeros_like(x)
        step[t, e] = h
        up, down = (forward64(x.detach() + s, ids, 1.0, 2, None)[0].item() for s in (step, -step))
        assert abs((up - down) / (2 * h) - grad[t, e].item()) < 1e-8
    _, counts, _, live = balance.balance_loss(logits.to(cuda), ids.to(cuda), 1.0, segments=2)
    own = balance.router_backward(logits.to(cuda), ids.to(cuda), counts, live, 1.0, segments=2).cpu()
    v, h = own.sign(), 2.0 ** -6
    up, down = (balance.balance_loss((logits + s * h * v).to(cuda), ids.to(cuda), 1.0, segments=2)[0].item()
                for s in (1, -1))
    slope = own.double().abs().sum().item()
    noise = 2 * 260 * U * abs(loss.item()) / (2 * h)
    assert abs((up - down) / (2 * h) - slope) <= noise + 8 * h * h * slope + 1e-6


def test_repeats_its_bits_on_streams_and_in_graphs(cuda):
    logits, ids, dw = (t.to(cuda) for t in case(600, 96, 4, 31))
    mask = (torch.rand(600, generator=torch.Generator().manual_seed(1)) < 0.8).to(cuda)

    def step(x):
        loss, counts, mean, live = balance.balance_loss(x, ids, 0.1, segments=3, mask=mask)
        return loss, counts, mean, balance.router_backward(x, ids, counts, live, 0.1, segments=3,
                                                           mask=mask, dweights=dw)

    want = step(logits)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(logits)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    x, y = logits.clone(), logits.clone()
    graphs = []
    for v in (x, y):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(v)
        graphs.append((g, v, out))
    for n in range(3):
        for i, (g, v, out) in enumerate(graphs):
            v.copy_(logits.roll(7 * n + i, 0))
            g.replay()
        for i, (g, v, out) in enumerate(graphs):
            want = step(logits.roll(7 * n + i, 0))
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_counts_are_the_plans(cuda):
    """The per-expert counts of one segment are k3_moe_route_plan's."""
    import ctypes

    from moonshine_amd._lib import lib
    T, E, k = 700, 40, 6
    logits, ids, _ = case(T, E, k, 41)
    ids[::6, 2] = ids[::6, 1]
    ids[::7, 0] = 40
    ids = ids.to(cuda)
    counts = balance.balance_loss(logits.to(cuda), ids, 1.0)[1]
    n = lib().k3_moe_plan_scratch_bytes(T, E)
    new = lambda m: torch.zeros(m, dtype=torch.int32, device=cuda)  # noqa: E731
    plan, rest = new(E), [new(E + 1), new(E), new(4), new(T * k), new(T * k)]
    scratch = torch.empty(n, dtype=torch.uint8, device=cuda)
    P = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    assert lib().k3_moe_route_plan(P(plan), *map(P, rest), P(ids), T, k, E, P(scratch), n,
                                   ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert torch.equal(counts[0], plan)


def test_refuses(cuda):
    logits, ids, dw = (t.to(cuda) for t in case(12, 16, 2, 1))
    _, counts, _, live = balance.balance_loss(logits, ids, 1.0, segments=3)
    for bad in (lambda: balance.balance_loss(logits, ids, 1.0, segments=5),
                lambda: balance.balance_loss(logits.double(), ids, 1.0),
                lambda: balance.balance_loss(logits, ids.long(), 1.0),
                lambda: balance.balance_loss(logits, ids[:6], 1.0),
                lambda: balance.balance_loss(logits.t(), ids, 1.0),
                lambda: balance.balance_loss(logits, ids, 1.0, mask=ids[:, 0]),
                lambda: balance.router_backward(logits, ids, counts, live, 1.0, segments=2),
                lambda: balance.router_backward(logits, ids, counts, live, 1.0, segments=3, dweights=dw[:, :1]),
                lambda: balance.router_backward(logits, ids, counts, live, 1.0, segments=3, out=dw)):
        with pytest.raises(ValueError):
            bad()


def test_a_training_step_of_the_router(cuda):
    """Router logits, routes, FP8-128 experts, balance loss, gradient and a step of the router's
    weight, as a user runs them: the step's gradient is that of the 64-bit formulas by the weight."""
    import _ops
    import test_gpu_fp8 as F8
    T = 64
    moe, x = F8.layer(cuda, T, seed=90)
    E, k, H = moe.cfg.experts, moe.cfg.top_k, moe.cfg.hidden
    ids = torch.zeros((T, k), dtype=torch.int32, device=cuda)
    w = torch.zeros((T, k), device=cuda)
    y = moe.forward(x, x, ids=ids, weights=w)
    dy = F8.normal((T, H), 91).to(cuda)
    logits = torch.empty((T, E), device=cuda)
    assert _ops.k3_rocm_bf16_gemm_f32(logits, moe.router_weight, x, T, E, H)
    # d(sum dy . out) / d weights[t, r]: the route's own rows, weight 1
    one = torch.ones((T, 1), device=cuda)
    sh = type(moe.shape)(H, E, 1, moe.cfg.ffn, 1.0, moe.cfg.activation, 4.0, 25.0)
    from moonshine_amd import fp8
    rows = [fp8.experts(x, ids[:, r:r + 1].contiguous(), one, moe.store.table, sh) for r in range(k)]
    dw = torch.stack([(dy.float() * v.float()).sum(1) for v in rows], 1)
    loss, counts, mean, live = balance.balance_loss(logits, ids, 0.5)
    grad = balance.router_backward(logits, ids, counts, live, 0.5, dweights=dw,
                                   scaling_factor=moe.cfg.scale)
    total = grad.t() @ x.float()
    # the same in 64 bits from the weight
    W = moe.router_weight.cpu().double().requires_grad_()
    z = x.cpu().double() @ W.t()
    l64, c64, *_, ok, sig = forward64(z, ids.cpu(), 0.5, 1, None)
    (l64 + (weights64(sig, ids.cpu(), ok, moe.cfg.scale) * dw.cpu().double()).sum()).backward()
    assert torch.equal(counts.cpu().double(), c64)
    # logits of 512 fp32 terms (each side's order its own) and the fp32 product above: 2^-12 of the whole
    assert torch.linalg.norm(total.cpu().double() - W.grad) <= 2.0 ** -12 * torch.linalg.norm(W.grad)
    # the weighted rows are the layer's output without its residual's rounding
    back = sum(w[:, r:r + 1] * v.float() for r, v in enumerate(rows)) + x.float()
    assert torch.linalg.norm(back - y.float()) <= 2.0 ** -7 * torch.linalg.norm(y.float())


def test_many_segments(cuda):
    """A segment a block; the last block adds up thousands of partial losses."""
    logits, ids, dw = case(4096, 64, 4, 21)
    check(cuda, logits, ids, dw, 1024, None)
    S, E, k = 65535, 8, 2
    logits, ids, _ = case(S, E, k, 22)
    got = balance.balance_loss(logits.to(cuda), ids.to(cuda), 0.3, segments=S)
    loss, counts, mean, n, *_ = forward64(logits.double(), ids, 0.3, S, None)
    assert torch.equal(got[1].cpu().double(), counts) and torch.equal(got[3].cpu().double(), n)
    assert ((got[2].cpu().double() - mean).abs() <= 230 * U * mean + 1e-38).all()
    # 64 terms a lane, 6 levels and 16 waves behind a term's own 234 u, and 2 more
    assert abs(got[0].item() - loss.item()) <= (234 + 64 + 6 + 16 + 2) * U * loss.item()


def test_gradient_into_the_logits(cuda):
    """The gradient may take the logits' place."""
    for E, T in ((64, 200), (896, 3000)):
        logits, ids, dw = (t.to(cuda) for t in case(T, E, 4, E))
        _, counts, _, live = balance.balance_loss(logits, ids, 0.3)
        want = balance.router_backward(logits, ids, counts, live, 0.3, dweights=dw)
        got = balance.router_backward(logits, ids, counts, live, 0.3, dweights=dw, out=logits)
        assert got is logits and torch.equal(got, want)
