"""RMS norm with the residual's addition, its FP8-128 rows, its gradient and the product of encoded
rows, on the GPU.

Bounds: u = 2^-24. A row's sum of squares is of positive terms, each within the depth of its tree of
additions, under 64, of u: rstd is within 48 u, n = total rstd weight within 64 u. A bf16 output
adds 2^-8 of itself; a code is e4m3 of n times an inverse scale within 70 u: within 2^-4 of its
value, or half of e4m3's least step, 2^-10, of the scale. The gradient's sums over a row are
within 80 u of their terms' magnitudes, the weight's over rows within (rows + 100) u.
"""
import pytest
import torch

import _grouped as R
from moonshine_amd import fp8, norm

pytestmark = pytest.mark.gpu

U, EPS = 2.0 ** -24, 1e-5
SIZES = [(1, 8), (3, 24), (5, 128), (4, 512), (9, 520), (130, 640), (7, 2048), (6, 2056), (61, 7168), (3, 8192), (2, 8200),
         (2, 16384), (1, 32768), (1000, 256), (801, 2176), (5, 4096), (770, 4104), (300, 8200), (3, 16392), (260, 16640)]


def data(rows, cols):
    x, r = R.normal((rows, cols), rows), R.normal((rows, cols), cols)
    if rows > 2:
        x[1], r[1] = 0, 0
        x[2] *= 2.0 ** 40
        r[2] *= 2.0 ** 40
    w = (1 + R.normal((cols,), 3, 0.2).float()).to(torch.bfloat16)
    return x, r, w


def plain(total, w):
    s = total.double()
    rstd = 1 / torch.sqrt(s.pow(2).mean(1) + EPS)
    return rstd, s * rstd[:, None] * w.double()


def close(got, want, size, fp32):
    got = got.cpu().double()
    slack = fp32 * U * size
    bound = slack + 2.0 ** -8 * (want.abs() + slack) + 2.0 ** -133
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("rows,cols", SIZES)
def test_norm(cuda, rows, cols):
    x, r, w = data(rows, cols)
    encode = cols % 128 == 0
    got = norm.residual_norm(x.to(cuda), w.to(cuda), EPS, residual=r.to(cuda), encode=encode)
    total = (x.float() + r.float()).to(torch.bfloat16)
    assert torch.equal(got.total.cpu(), total)
    rstd, n = plain(total, w)
    assert ((got.rstd.cpu().double() - rstd).abs() <= 48 * U * rstd).all()
    close(got.normed, n, n.abs(), 64)
    alone = norm.residual_norm(total.to(cuda), w.to(cuda), EPS)
    assert alone.total.data_ptr() != got.total.data_ptr() and alone.codes is None
    assert torch.equal(alone.normed, got.normed) and torch.equal(alone.rstd, got.rstd)
    if not encode:
        assert got.codes is None and got.scales is None
        return
    a = n.view(rows, -1, 128).abs().amax(2).clamp_min(448 * 2.0 ** -126)
    scale = got.scales.cpu().double()
    assert ((scale - a / 448).abs() <= 70 * U * a / 448).all()
    held = got.codes.cpu().double().view(rows, -1, 128) * scale[:, :, None]
    v = n.view(rows, -1, 128)
    bound = 2.0 ** -4 * v.abs() * (1 + 200 * U) + 200 * U * v.abs() + 2.0 ** -10 * scale[:, :, None]
    assert ((held - v).abs() <= bound).all()
    codes = norm.residual_norm(x.to(cuda), w.to(cuda), EPS, residual=r.to(cuda), encode=True, normed=False)
    assert codes.normed is None and torch.equal(codes.codes.view(torch.uint8), got.codes.view(torch.uint8))


def test_codes_are_the_rows_encoding(cuda):
    """A weight of ones, rows whose norm is exact: the codes are quantize_rows' of the normed rows."""
    x = R.whole((16, 512), 1).to(cuda)
    x = torch.where(x == 0, 1, x).sign().to(torch.bfloat16) * 2  # of norm 2: n is +-1 up to rstd's rounding
    got = norm.residual_norm(x, torch.ones(512, dtype=torch.bfloat16, device=cuda), 0.0, encode=True)
    assert torch.equal(got.normed, x / 2)
    codes, scales = fp8.quantize_rows(got.normed)
    assert torch.equal(got.codes.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(got.scales, scales)


def test_in_place(cuda):
    x, r, w = (t.to(cuda) for t in data(40, 640))
    want = norm.residual_norm(x, w, EPS, residual=r)
    for which in (0, 1):
        a, b = x.clone(), r.clone()
        into = (a, b)[which]
        got = norm.residual_norm(a, w, EPS, residual=b, total=into)
        assert got.total.data_ptr() == into.data_ptr()
        assert torch.equal(into, want.total) and torch.equal(got.normed, want.normed)
    with pytest.raises(RuntimeError):
        room = torch.zeros((80, 640), dtype=torch.bfloat16, device=cuda)
        norm.residual_norm(room[1:41], w, EPS, residual=r, total=room[:40])


def test_non_finite_rows(cuda):
    """A NaN or an infinity is its row's alone; codes of such a row are NaN where its values are."""
    x, r, w = data(4, 256)
    x[0, 5], x[2, 200] = float("nan"), float("inf")
    got = norm.residual_norm(x.to(cuda), w.to(cuda), EPS, residual=r.to(cuda), encode=True)
    rstd, n = plain(got.total.cpu(), w)
    assert torch.equal(got.normed.cpu().isnan(), n.isnan())
    assert got.normed[1].isfinite().all() and got.normed[3].isfinite().all()
    assert got.codes.cpu().float()[n.isnan()].isnan().all()


def backward64(dn, s, w, rstd, dt):
    dn, s, w, r = dn.double(), s.double(), w.double(), rstd.double()[:, None]
    dw, mean = dn * w, (dn * w * s).mean(1, keepdim=True)
    dx = r * (dw - s * r * r * mean)
    size = r.abs() * (dw.abs() + s.abs() * r * r * (dn * w * s).abs().mean(1, keepdim=True))
    if dt is not None:
        dx, size = dx + dt.double(), size + dt.double().abs()
    return dx, size, (dn * s * r).sum(0), (dn * s * r).abs().sum(0)


@pytest.mark.parametrize("rows,cols", SIZES + [(1700, 64), (3500, 520)])
@pytest.mark.parametrize("with_total", [True, False])
def test_backward(cuda, rows, cols, with_total):
    s, _, w = data(rows, cols)
    rstd = plain(s, w)[0].float()
    dn, dt = R.normal((rows, cols), 7, 1e-3), R.normal((rows, cols), 8, 1e-3) if with_total else None
    dx, dw = norm.residual_norm_backward(dn.to(cuda), s.to(cuda), w.to(cuda), rstd.to(cuda),
                                         None if dt is None else dt.to(cuda))
    want, size, wdw, sdw = backward64(dn, s, w, rstd, dt)
    close(dx, want, size, 80)
    assert ((dw.cpu().double() - wdw).abs() <= (rows + 100) * U * sdw + 2.0 ** -140).all()
    for into in ("dn", "s", "dt"):
        a = {"dn": dn.to(cuda), "s": s.to(cuda), "dt": None if dt is None else dt.to(cuda)}
        if a[into] is None:
            continue
        again, dw2 = norm.residual_norm_backward(a["dn"], a["s"], w.to(cuda), rstd.to(cuda), a["dt"], out=a[into])
        assert torch.equal(again, dx) and torch.equal(dw2, dw)


def test_gradient_by_differences(cuda):
    """The formula that the kernel is held to, against central differences of the norm, in 64 bits."""
    g = torch.Generator().manual_seed(1)
    s, dn, w = (torch.randn(sh, generator=g, dtype=torch.float64) for sh in ((3, 16), (3, 16), (16,)))

    def value(s, w):
        return (s / torch.sqrt(s.pow(2).mean(1, keepdim=True) + EPS) * w * dn).sum()

    rstd = 1 / torch.sqrt(s.pow(2).mean(1) + EPS)
    dx, _, dw, _ = backward64(dn, s, w, rstd, None)
    for i, j in ((0, 0), (1, 7), (2, 15)):
        e = torch.zeros_like(s)
        e[i, j] = 1e-6
        assert abs((value(s + e, w) - value(s - e, w)) / 2e-6 - dx[i, j]) < 1e-8
        f = torch.zeros_like(w)
        f[j] = 1e-6
        assert abs((value(s, w + f) - value(s, w - f)) / 2e-6 - dw[j]) < 1e-8


@pytest.mark.parametrize("T", [1, 2, 3, 8, 9, 16, 40, 300, 1000])
@pytest.mark.parametrize("N,K", [(48, 128), (200, 640), (256, 1024), (4100, 896), (512, 4224)])
def test_product_of_encoded_rows_is_the_products(cuda, T, N, K):
    x, w = R.normal((T, K), T).to(cuda), R.normal((N, K), N, 0.02).to(cuda)
    codes, scales = fp8.quantize_weight(w)
    xq, xs = fp8.quantize_rows(x)
    want = fp8.product(x, codes, scales)
    assert torch.equal(fp8.product_encoded(xq, xs, codes, scales), want)
    room = torch.zeros(xs.numel() + 1, device=cuda)  # scales at 4 mod 16 bytes
    at = 1 if room.data_ptr() % 16 == 0 else 0
    room[at:at + xs.numel()] = xs.view(-1)
    odd = room[at:at + xs.numel()].view(xs.shape)
    assert torch.equal(fp8.product_encoded(xq.view(torch.uint8), odd, codes, scales), want)


def test_streams_and_graphs(cuda):
    """A captured forward and backward, replayed between eager work on the same memory."""
    x, r, w = (t.to(cuda) for t in data(70, 896))
    weight = fp8.quantize_weight(R.normal((256, 896), 5, 0.02).to(cuda))
    dn, dt = R.normal((70, 896), 6).to(cuda), R.normal((70, 896), 7).to(cuda)

    def step():
        n = norm.residual_norm(x, w, EPS, residual=r, encode=True)
        return (n.total, n.normed, fp8.product_encoded(n.codes, n.scales, *weight),
                *norm.residual_norm_backward(dn, n.total, w, n.rstd, dt))

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    side = torch.cuda.Stream()
    for turn in range(3):
        x.copy_(R.normal((70, 896), 20 + turn).to(cuda))
        want = [t.clone() for t in step()]
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        with torch.cuda.stream(side):
            again = step()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(again, want))
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_past_32_bits(cuda):
    """Rows past 4 GiB of every tensor have the bits that they have alone."""
    rows, cols = 131200, 16384
    x, r = (torch.zeros((rows, cols), dtype=torch.bfloat16, device=cuda) for _ in range(2))
    w = (1 + R.normal((cols,), 3, 0.2).float()).to(torch.bfloat16).to(cuda)
    x[-3:], r[-3:] = R.normal((3, cols), 1).to(cuda), R.normal((3, cols), 2).to(cuda)
    want = norm.residual_norm(x[-3:].clone(), w, EPS, residual=r[-3:].clone(), encode=True)
    got = norm.residual_norm(x, w, EPS, residual=r, encode=True, total=x)
    for a, b in zip(got, want):
        assert torch.equal(a[-3:].view(torch.uint8), b.view(torch.uint8))
    assert not got.normed[:-3].any()
    dn, dt = R.normal((3, cols), 4).to(cuda), R.normal((3, cols), 5).to(cuda)
    dx, dw = norm.residual_norm_backward(dn, want.total, w, want.rstd, dt)
    r.zero_()
    r[-3:] = dn
    got.normed.zero_()
    got.normed[-3:] = dt
    big, bdw = norm.residual_norm_backward(r, x, w, got.rstd, got.normed, out=r)
    assert torch.equal(big[-3:], dx) and not big[:-3].any()
    # the weight's terms of the other rows are zeros: the three are added in another order
    terms = (dn.double() * want.total.double() * want.rstd.double()[:, None]).abs().sum(0)
    assert ((bdw - dw).double().abs() <= 8 * U * terms).all()
