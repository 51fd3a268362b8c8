"""Plain 64-bit forms of the FP8-128 operators, and the error bounds that the
kernels' arithmetic allows (all on the CPU).

u = 2^-24 is half a step of fp32 (relative). A block's 128 code products are
exact; the matrix unit adds them in an order and with a rounding that are its
own, at most a whole fp32 step (2 u) an addition: 256 u of the sum of their
magnitudes. Scaling by sx sw (u), one fma a block (u each) and, where the
blocks are added in parts, as many additions again: (2 nblk + 4) u. Where sx sw
is under 2^-126 it is a multiple of 2^-149, off by up to 2^-150 and not by u of
itself: 2^-150 of the block's |code products|, at most 2^-150 of all of them.
"""
import numpy as np
import torch

U = 2.0 ** -24
LEAST = np.float32(448.0 * 2.0 ** -126)


def block_scales(a):
    """(scale, inv) as fp32 of block maxima (fp32 numpy)."""
    a = np.maximum(a.astype(np.float32), LEAST)
    return a / np.float32(448), np.float32(448) / a


def encode(v):
    """fp32 numpy within +-448 (1 + 2^-23) -> e4m3 byte, nearest even, written out."""
    v = np.asarray(v, dtype=np.float32)
    mag = np.abs(v).astype(np.float64)
    e = np.maximum(np.floor(np.log2(np.maximum(mag, 2.0 ** -30))), -6.0)
    q = np.rint(mag / 2.0 ** (e - 3)) * 2.0 ** (e - 3)      # a multiple of the step
    e2 = np.maximum(np.floor(np.log2(np.maximum(q, 2.0 ** -30))), -6.0)
    code = np.where(q < 2.0 ** -6, q / 2.0 ** -9, (e2 + 7) * 8 + (q / 2.0 ** e2 - 1) * 8)
    code = np.where(np.isnan(v), 0x7f, code)
    return code.astype(np.uint8) | (np.signbit(v).astype(np.uint8) << 7)


def values(codes):
    """uint8 or float8 codes -> float64 values (torch)."""
    t = torch.from_numpy(codes) if isinstance(codes, np.ndarray) else codes
    return t.cpu().view(torch.float8_e4m3fn).to(torch.float64)


def rows64(v):
    """fp32 numpy [T, K] -> code values, scales [T, K / 128] (torch float64)."""
    b = v.reshape(v.shape[0], -1, 128)
    scale, inv = block_scales(np.abs(b).max(2))
    codes = encode(b * inv[:, :, None]).reshape(v.shape)
    return values(codes), torch.from_numpy(scale).double()


def unpack(q, s, rows_per=1):
    """Code values x scales."""
    full = s.repeat_interleave(rows_per, 0)[: q.shape[0]].repeat_interleave(128, 1)
    return q * full


def product64(q, sx, wq, ws):
    """(sum, bound of the fp32 error) of rows with a weight [N, K], scales [N / 128, K / 128]."""
    x, w = unpack(q, sx), unpack(wq, ws, 128)
    nblk = q.shape[1] // 128
    err = (256 + 2 * nblk + 4) * U * (x.abs() @ w.abs().t())
    if sx.min() * ws.min() < 2.0 ** -126:
        err = err + 2.0 ** -150 * (q.abs() @ wq.abs().t())
    return x @ w.t(), err


def bf16_bound(y, err):
    """Bound of a bf16 output: half a step (2^-8) of the rounded value."""
    return err + 2.0 ** -8 * (y.abs() + err)


def act64(g, u, swiglu, beta, lb):
    s = 1 / (1 + torch.exp(-g))
    if swiglu:
        return g * s * u
    return beta * torch.tanh(g / beta) * s * lb * torch.tanh(u / lb)


def act_bound(g, u, eg, eu, h, swiglu, beta):
    """|d act / dg| <= 1.1 |u| (SwiGLU) or (1 + beta / 4) |u|, |d act / du| <= |g| of both; the
    activation's own error: exp2 and the reciprocal 1 ulp each, the exponent's rounding |g| u, a
    dozen roundings, tanh within 16 u of itself."""
    slope = 1.1 if swiglu else 1 + beta / 4
    return (slope * (u.abs() + eu) * eg + (g.abs() + eg) * eu
            + h.abs() * (64 + 4 * (g.abs() + eg)) * U)


def expert64(x, gate, up, down, swiglu, beta=4.0, lb=25.0):
    """One expert on fp32 numpy rows -> (y64, bound without the bf16 rounding).

    gate, up, down: (code values, scales). The activation's codes are those of h64; where an h
    within its error, or a scale within its own, rounds to another code, the product may be off
    by that much."""
    q, s = rows64(x)
    g, eg = product64(q, s, *gate)
    u, eu = product64(q, s, *up)
    h = act64(g, u, swiglu, beta, lb)
    dh = act_bound(g, u, eg, eu, h, swiglu, beta)
    hf = h.float().numpy()
    hq, hs = rows64(hf)
    held = unpack(hq, hs)
    b = h.abs().view(h.shape[0], -1, 128)
    # relative error of a block's maximum, hence of its scale (and 2 roundings)
    es = ((dh.view(b.shape).amax(2) / b.amax(2).clamp_min(1e-300)).clamp_max(1.0) + 4 * U)
    es = es.repeat_interleave(128, 1)
    scale = hs.repeat_interleave(128, 1)
    lo, hi = ((h + sign * (dh + h.abs() * es + U * h.abs())) / scale for sign in (-1, 1))
    off = torch.zeros_like(h)
    for v in (lo, hi):
        code = values(encode(v.clamp(-448, 448).float().numpy()))
        off = torch.maximum(off, (code * scale - held).abs())
    off = off + held.abs() * es
    w = unpack(*down, 128)
    y, ey = product64(hq, hs, *down)
    return y, ey * 1.01 + off @ w.abs().t()
