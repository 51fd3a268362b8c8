"""Plain 64-bit forms of the products grouped by expert, with the bound of their error.

Values of small whole numbers make every product and every sum exact in fp32 (under 2^24),
so the one rounding left is the output's and results are compared bit for bit. Of other
values, each of the Z additions of a sum may be off by a whole fp32 step (2^-23) of the sum
of the magnitudes, and a bf16 output by half a step more: 2^-8 of the value.
"""
import torch


def routes(T, k, E, seed, skew=0.0):
    """ids int32 [T, k] of different experts."""
    g = torch.Generator().manual_seed(seed)
    score = torch.rand((T, E), generator=g) + skew * torch.rand((1, E), generator=g)
    return score.topk(k, dim=1).indices.to(torch.int32)


def plan(ids, E):
    """offsets, token and route of each row, by a stable sort; an id from E on, and one that its token
    has had, has no row."""
    T, k = ids.shape
    rows = [[] for _ in range(E)]
    for t in range(T):
        seen = set()
        for r in range(k):
            e = int(ids[t, r])
            if 0 <= e < E and e not in seen:
                rows[e].append(t * k + r)
                seen.add(e)
    offsets = [0]
    for r in rows:
        offsets.append(offsets[-1] + len(r))
    route = torch.tensor([r for rs in rows for r in rs], dtype=torch.int32)
    return torch.tensor(offsets, dtype=torch.int32), route // k, route


def whole(shape, seed, most=3):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g).to(torch.bfloat16)


def normal(shape, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(torch.bfloat16)


def picked(rows, index):
    """rows[index] in 64 bits, a row of zeros for an index that is none."""
    rows = rows.double()
    if index is None:
        return rows
    ok = (index >= 0) & (index < rows.shape[0])
    return rows[index.long().clamp(0, rows.shape[0] - 1)] * ok[:, None]


def by_rows(rows, weights, offsets, index, transposed):
    """(output rows in order, sums of magnitudes) of product, or (transposed) of the input gradient."""
    v = picked(rows, index)
    width = weights.shape[2] if transposed else weights.shape[1]
    out, size = torch.zeros((v.shape[0], width), dtype=torch.float64), None
    size = torch.zeros_like(out)
    for e in range(weights.shape[0]):
        a, b = int(offsets[e]), int(offsets[e + 1])
        if a < b:
            w = weights[e].double() if transposed else weights[e].double().t()
            out[a:b] = v[a:b] @ w
            size[a:b] = v[a:b].abs() @ w.abs()
    return out, size


def by_weights(dy, x, offsets, dy_index, x_index):
    d, v = picked(dy, dy_index), picked(x, x_index)
    E = offsets.shape[0] - 1
    out = torch.zeros((E, d.shape[1], v.shape[1]), dtype=torch.float64)
    size = torch.zeros_like(out)
    for e in range(E):
        a, b = int(offsets[e]), int(offsets[e + 1])
        if a < b:
            out[e] = d[a:b].t() @ v[a:b]
            size[e] = d[a:b].abs().t() @ v[a:b].abs()
    return out, size


def bound(out, size, Z, dtype):
    """Of each value: Z additions, and the output's rounding."""
    fp32 = Z * 2.0 ** -23 * size
    return fp32 + (2.0 ** -8 * (out.abs() + fp32) + 2.0 ** -134 if dtype == torch.bfloat16 else 0.0)
