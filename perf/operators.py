"""The 8-bit floating point and router-training operators, as they are timed.

Four kinds of call:

  rows, weight  FP8-128 quantizers: e4m3 codes with a scale for every 128
                values of a token row, or every 128 x 128 values of a weight
  product       bf16 tokens times an FP8-128 weight, tokens quantized on the
                way in: from one token to a prefill chunk
  experts       the routed experts of a layer with FP8-128 weights, on routes
                that the router has given: decode, batched decode, prefill
  balance       a training step's router side: the balance loss, the
                per-expert counts and mean scores, and the gradient of the
                loss and of the route weights by the router's logits

Everything is seeded torch on the GPU. Weights are N(0, 0.02) in FP8-128,
token rows N(0, 1), router logits N(0, 1.7) (what such rows and weights give
at a width of 7168).
"""
import math

import torch

own = False

SITU, SWIGLU = 0, 1
BETA, LINEAR_BETA, SCALE = 4.0, 25.0, 2.5
TOP = 448.0                    # the largest e4m3 value
LEAST = 448.0 * 2.0 ** -126    # the least maximum of a block: its scale is a normal number

# (hidden, ffn, experts, top_k, activation): the benchmark's layer with a store of 128 experts,
# its reduced configuration, and a small generic layer with the engine's activation
SHAPES = {
    "wide": (7168, 2048, 128, 8, SWIGLU),
    "reduced": (2048, 512, 64, 4, SWIGLU),
    "small": (1024, 1024, 40, 6, SITU),
}


def listed():
    return [
        # a weight of a checkpoint, once at load time; the last row block is ragged
        dict(name="weight-4100x7168", kind="weight", rows=4100, cols=7168),
        # the rows of a prefill chunk
        dict(name="rows-8192x7168", kind="rows", rows=8192, cols=7168),
        # one token through one projection: latency
        dict(name="product-1", kind="product", tokens=1, rows=2048, cols=7168),
        # a batched decode step, an odd number of sequences
        dict(name="product-37", kind="product", tokens=37, rows=7168, cols=7168),
        # a short prompt, ragged rows
        dict(name="product-300", kind="product", tokens=300, rows=4100, cols=7168),
        # a prefill chunk
        dict(name="product-4096", kind="product", tokens=4096, rows=7168, cols=7168),
        # one token through a small layer's experts: latency
        dict(name="experts-reduced-1", kind="experts", shape="reduced", tokens=1),
        # one token of decode: eight experts' weights
        dict(name="experts-wide-1", kind="experts", shape="wide", tokens=1),
        # batched decode: nearly every expert, a few rows each
        dict(name="experts-wide-61", kind="experts", shape="wide", tokens=61),
        # a prefill chunk
        dict(name="experts-wide-4096", kind="experts", shape="wide", tokens=4096),
        # a fine-tuning batch of short padded sequences, a loss for each
        dict(name="balance-6x333", kind="balance", segments=6, length=333, experts=64, top_k=4,
             masked=True),
        # a training batch as one, at the benchmark's router
        dict(name="balance-8192", kind="balance", segments=1, length=8192, experts=896, top_k=16,
             masked=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rows", "weight", "product", "product", "product", "experts", "experts",
                       "experts", "balance", "balance"])
    if kind in ("rows", "weight"):
        return dict(kind=kind, rows=_log_int(rng, 1, 8192), cols=128 * _log_int(rng, 1, 56))
    if kind == "product":
        return dict(kind=kind, tokens=_log_int(rng, 1, 4096), rows=_log_int(rng, 16, 7168),
                    cols=128 * _log_int(rng, 1, 56))
    if kind == "experts":
        return dict(kind=kind, shape=rng.choice(sorted(SHAPES)), tokens=_log_int(rng, 1, 4096))
    segments = _log_int(rng, 1, 16)
    experts = _log_int(rng, 8, 1024)
    return dict(kind=kind, segments=segments, length=_log_int(rng, 1, 8192 // segments),
                experts=experts, top_k=rng.randint(1, min(16, experts)), masked=rng.random() < 0.5)


# ---- inputs, made from the seed alone ---------------------------------------------------


def _gen(seed, part):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 64 + part)
    return g


def _normal(shape, std, gen):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(torch.bfloat16)


def _fp8_weight(rows, cols, gen):
    """Codes (float8_e4m3fn) [rows, cols] and scales [ceil(rows / 128), cols / 128]."""
    pad = -rows % 128
    w = _normal((rows, cols), 0.02, gen).float()
    if pad:
        w = torch.cat([w, w.new_zeros((pad, cols))])
    blocks = w.view(-1, 128, cols // 128, 128)
    scale = blocks.abs().amax((1, 3)).clamp_min(LEAST) * (1.0 / TOP)
    codes = (blocks / scale[:, None, :, None]).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
    return codes.view(-1, cols)[:rows].contiguous(), scale


def _fp8_experts(count, rows, cols, gen):
    """The same matrix of every expert: codes [E, rows, cols], scales [E, rows / 128, cols / 128]."""
    codes = torch.empty((count, rows, cols), dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty((count, rows // 128, cols // 128), device="cuda")
    for e in range(count):
        codes[e], scales[e] = _fp8_weight(rows, cols, gen)
    return codes, scales


def _routes(logits, top_k):
    """ids (int32) and weights of the router: the top scores, renormalized and scaled."""
    score, ids = torch.sigmoid(logits).topk(top_k, dim=1)
    weights = score / score.sum(1, keepdim=True) * SCALE
    return ids.to(torch.int32), weights


def prepare(case, seed):
    kind = case["kind"]
    if kind in ("rows", "weight"):
        std = 1.0 if kind == "rows" else 0.02
        return dict(case=case, x=_normal((case["rows"], case["cols"]), std, _gen(seed, 1)))
    if kind == "product":
        codes, scales = _fp8_weight(case["rows"], case["cols"], _gen(seed, 1))
        return dict(case=case, codes=codes, scales=scales,
                    x=_normal((case["tokens"], case["cols"]), 1.0, _gen(seed, 2)))
    if kind == "experts":
        H, F, E, k, _ = SHAPES[case["shape"]]
        g = _gen(seed, 1)
        w = dict(gate=_fp8_experts(E, F, H, g), down=_fp8_experts(E, H, F, g),
                 up=_fp8_experts(E, F, H, g))
        # the device table of a resident store: each expert's six addresses
        at = [t.data_ptr() + t.stride(0) * t.element_size() * torch.arange(E, device="cuda")
              for pair in w.values() for t in pair]
        T = case["tokens"]
        ids, weights = _routes(torch.randn((T, E), generator=_gen(seed, 2), device="cuda") * 1.7, k)
        return dict(case=case, **w, table=torch.stack(at, 1).contiguous(), ids=ids, weights=weights,
                    x=_normal((T, H), 1.0, _gen(seed, 3)),
                    residual=_normal((T, H), 1.0, _gen(seed, 4)))
    S, L, E, k = case["segments"], case["length"], case["experts"], case["top_k"]
    logits = torch.randn((S * L, E), generator=_gen(seed, 1), device="cuda") * 1.7
    ids, _ = _routes(logits, k)
    mask = None
    if case["masked"]:  # sequences of different lengths, padded to the longest
        n = torch.randint(0, L + 1, (S, 1), generator=_gen(seed, 2), device="cuda")
        n[0] = L
        mask = (torch.arange(L, device="cuda")[None] < n).reshape(-1).to(torch.uint8)
    return dict(case=case, logits=logits, ids=ids, mask=mask,
                dweights=torch.randn((S * L, k), generator=_gen(seed, 3), device="cuda") * 1e-3 / (S * L))


# ---- one pass ---------------------------------------------------------------------------

COEF = 0.01


def run(state):
    case = state["case"]
    return _run_own(case["kind"], state) if own else _run_plain(case["kind"], state)


def _run_own(kind, s):
    from moonshine_amd import balance, fp8

    if kind == "rows":
        codes, scales = fp8.quantize_rows(s["x"])
        return codes, scales
    if kind == "weight":
        codes, scales = fp8.quantize_weight(s["x"])
        return codes, scales
    if kind == "product":
        return fp8.product(s["x"], s["codes"], s["scales"])
    if kind == "experts":
        H, F, E, k, act = SHAPES[s["case"]["shape"]]
        shape = fp8.shape(H, E, k, F, SCALE, act, BETA, LINEAR_BETA)
        return fp8.experts(s["x"], s["ids"], s["weights"], s["table"], shape, s["residual"])
    segments = s["case"]["segments"]
    loss, counts, mean, valid = balance.balance_loss(s["logits"], s["ids"], COEF,
                                                     segments=segments, mask=s["mask"])
    grad = balance.router_backward(s["logits"], s["ids"], counts, valid, COEF, segments=segments,
                                   mask=s["mask"], dweights=s["dweights"], scaling_factor=SCALE)
    return loss, counts, mean, grad


def _scales_of(a):
    a = a.clamp_min(LEAST)
    top = torch.full_like(a, TOP)  # tensors: a scalar's division may go by its reciprocal
    return a / top, top / a


def _quantize(x):
    """fp32 [rows, cols] -> e4m3 codes [rows, cols], scales [rows, cols / 128]."""
    v = x.view(x.shape[0], -1, 128)
    scale, inv = _scales_of(v.abs().amax(2))
    return (v * inv[:, :, None]).to(torch.float8_e4m3fn).view(x.shape), scale


def _unpack(codes, scales):
    """codes x scales of a weight (or of many), fp32."""
    rows, cols = codes.shape[-2:]
    full = scales.repeat_interleave(128, -2)[..., :rows, :].repeat_interleave(128, -1)
    return codes.float().mul_(full)


def _times(x, codes, scales):
    """q(x) . W^T in fp32."""
    q, sx = _quantize(x)
    return (q.float() * sx.repeat_interleave(128, 1)) @ _unpack(codes, scales).t()


def _gated(g, u, act):
    if act == SWIGLU:
        return g * torch.sigmoid(g) * u
    return BETA * torch.tanh(g / BETA) * torch.sigmoid(g) * (LINEAR_BETA * torch.tanh(u / LINEAR_BETA))


def _run_plain(kind, s):
    if kind == "rows":
        return _quantize(s["x"].float())
    if kind == "weight":
        rows, cols = s["x"].shape
        w = torch.nn.functional.pad(s["x"].float(), (0, 0, 0, -rows % 128))
        v = w.view(-1, 128, cols // 128, 128)
        scale, inv = _scales_of(v.abs().amax((1, 3)))
        codes = (v * inv[:, None, :, None]).to(torch.float8_e4m3fn)
        return codes.view(-1, cols)[:rows], scale
    if kind == "product":
        return _times(s["x"].float(), s["codes"], s["scales"]).to(torch.bfloat16)
    if kind == "experts":
        act, (T, k) = SHAPES[s["case"]["shape"]][4], s["ids"].shape
        order = s["ids"].reshape(-1).sort(stable=True)
        chosen, counts = order.values.unique_consecutive(return_counts=True)
        y = torch.empty((T * k, s["x"].shape[1]), device="cuda")
        x = s["x"].float()
        for e, routes in zip(chosen.tolist(), order.indices.split(counts.tolist())):
            rows = x[routes // k]
            g = _times(rows, s["gate"][0][e], s["gate"][1][e])
            u = _times(rows, s["up"][0][e], s["up"][1][e])
            y[routes] = _times(_gated(g, u, act), s["down"][0][e], s["down"][1][e])
        y = y.to(torch.bfloat16).float().view(T, k, -1)
        sum_ = (y * s["weights"][:, :, None]).sum(1).to(torch.bfloat16).float()
        return (s["residual"].float() + sum_).to(torch.bfloat16)
    S, L, E, k = (s["case"][n] for n in ("segments", "length", "experts", "top_k"))
    x, ids = s["logits"], s["ids"].long()
    sigma, rest = torch.sigmoid(x), torch.sigmoid(-x)
    z = sigma.sum(1, keepdim=True)
    p = sigma / z
    live = torch.ones(S * L, device="cuda") if s["mask"] is None else s["mask"].float()
    n = live.view(S, L).sum(1)
    chosen = torch.zeros_like(x).scatter_(1, ids, live[:, None].expand(-1, k))
    counts = chosen.view(S, L, E).sum(1)
    mean = (p * live[:, None]).view(S, L, E).sum(1) / n.clamp_min(1)[:, None]
    f = counts * (E / k) / n.clamp_min(1)[:, None]
    loss = (f * mean).sum() * (COEF / S)
    # the gradient by the scores, then by the logits
    ft = f[:, None, :].expand(S, L, E).reshape(S * L, E)
    share = (live.view(S, L) * (COEF / S) / n.clamp_min(1)[:, None]).view(-1, 1)
    grad = (ft - (ft * p).sum(1, keepdim=True)) / z * share
    picked = sigma.gather(1, ids)
    total = picked.sum(1, keepdim=True) + 1e-20
    dw = s["dweights"] * live[:, None]
    grad.scatter_add_(1, ids, (dw - (dw * picked).sum(1, keepdim=True) / total) * SCALE / total)
    return loss, counts.to(torch.int32), mean, grad * sigma * rest


# ---- what a pass cannot do without ------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind in ("rows", "weight"):
        n = case["rows"] * case["cols"]
        scales = n / 128 if kind == "rows" else n / 128 ** 2
        return {"bytes": 3 * n + 4 * scales, "flops": 3 * n}
    if kind == "product":
        T, N, K = case["tokens"], case["rows"], case["cols"]
        return {"bytes": N * K * (1 + 4 / 128 ** 2) + 2 * T * K + 2 * T * N, "flops": 2 * T * N * K}
    if kind == "experts":
        H, F, E, k, _ = SHAPES[case["shape"]]
        T = case["tokens"]
        chosen = E * (1 - (1 - k / E) ** T)  # what uniform routes touch
        return {"bytes": chosen * 3 * H * F * (1 + 4 / 128 ** 2) + 6 * T * H + 8 * T * k,
                "flops": 6 * T * k * H * F}
    S, E, k = case["segments"], case["experts"], case["top_k"]
    T = S * case["length"]
    return {"bytes": 8 * T * E + 8 * T * k + 8 * S * E + (T if case["masked"] else 0),
            "flops": 12 * T * E}


# ---- the definition, in 64 bits ---------------------------------------------------------


def _e4m3(v):
    """Nearest e4m3 values (ties to even) of fp32 values within +-448, in 64 bits."""
    v = v.double()
    _, e = torch.frexp(v)  # |v| = m 2^e, 0.5 <= m < 1
    step = torch.pow(2.0, (e - 4).clamp_min(-9).double())
    return torch.round(v / step) * step


def _held(v, over):
    """(code values, scale) of blocks of fp32 values, the scale over the dimensions `over`."""
    a = v.double().abs().amax(over, keepdim=True).clamp_min(LEAST)
    scale, inv = (a / TOP).float(), (TOP / a).float()
    return _e4m3((v.double() * inv.double()).float()), scale.double()


def _product64(x, codes, scales):
    """sum over blocks of (scales x the block's code products), x fp32 [T, K], one weight."""
    out = torch.zeros((x.shape[0], codes.shape[0]), dtype=torch.float64, device="cuda")
    row_block = torch.arange(codes.shape[0], device="cuda") // 128
    q, sx = _held(x.reshape(x.shape[0], -1, 128), 2)
    step = max(1, (1 << 18) // codes.shape[0])  # blocks of 128 columns at once
    for b in range(0, q.shape[1], step):
        left = (q[:, b:b + step] * sx[:, b:b + step]).flatten(1)
        n = left.shape[1] // 128
        right = codes[:, 128 * b:128 * (b + n)].double().view(-1, n, 128)
        right = right * scales[:, b:b + n].double()[row_block][:, :, None]
        out += left @ right.flatten(1).t()
    return out


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "rows":
        x = s["x"].view(case["rows"], -1, 128)
        codes, scale = _held(x.float(), 2)
        return codes.view(s["x"].shape), scale[:, :, 0]
    if kind == "weight":
        rows, cols = s["x"].shape
        x = torch.zeros((-(-rows // 128) * 128, cols), device="cuda")
        x[:rows] = s["x"]
        codes, scale = _held(x.view(-1, 128, cols // 128, 128), (1, 3))
        return codes.reshape(-1, cols)[:rows], scale[:, 0, :, 0]
    if kind == "product":
        return _product64(s["x"].float(), s["codes"], s["scales"])
    if kind == "experts":
        act = SHAPES[case["shape"]][4]
        out = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
        for e in range(s["gate"][0].shape[0]):
            token, rank = torch.where(s["ids"] == e)
            if not len(token):
                continue
            x = s["x"][token].float()
            g = _product64(x, s["gate"][0][e], s["gate"][1][e])
            u = _product64(x, s["up"][0][e], s["up"][1][e])
            if act == SWIGLU:
                h = g / (1 + torch.exp(-g)) * u
            else:
                h = (BETA * torch.tanh(g / BETA) / (1 + torch.exp(-g))
                     * LINEAR_BETA * torch.tanh(u / LINEAR_BETA))
            y = _product64(h.float(), s["down"][0][e], s["down"][1][e])
            out.index_add_(0, token, y * s["weights"][token, rank].double()[:, None])
        return out + s["residual"].double()
    S, L, E, k = (case[n] for n in ("segments", "length", "experts", "top_k"))
    x = s["logits"].double().requires_grad_()
    live = (torch.ones(S * L, device="cuda") if s["mask"] is None else s["mask"]).double()
    sigma = 1 / (1 + torch.exp(-x))
    p = sigma / sigma.sum(1, keepdim=True)
    loss, means = 0.0, []
    for i in range(S):
        at = slice(i * L, (i + 1) * L)
        n = max(1.0, float(live[at].sum()))
        hits = torch.zeros(E, dtype=torch.float64, device="cuda")
        hits.index_add_(0, s["ids"][at].reshape(-1).long(), live[at].repeat_interleave(k))
        mean = (p[at] * live[at, None]).sum(0) / n
        loss = loss + (hits * E / (k * n) * mean).sum() * COEF / S
        means.append(mean)
    picked = torch.gather(sigma, 1, s["ids"].long())
    weights = SCALE * picked / picked.sum(1, keepdim=True)
    through = (weights * s["dweights"].double() * live[:, None]).sum()
    (grad,) = torch.autograd.grad(loss + through, x)
    return loss.detach(), None, torch.stack(means).detach(), grad
