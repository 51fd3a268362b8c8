"""FP8-128 quantizers, product, routed experts and the native block's FP8-128
projections on the GPU, against plain 64-bit forms (tests/_fp8.py, where the
bounds are derived)."""
import numpy as np
import pytest
import torch

import _fp8 as R
from moonshine_amd import fp8
from moonshine_amd import native as N
from moonshine_amd.synth import ACT_SITU, ACT_SWIGLU, Config

pytestmark = pytest.mark.gpu


def normal(shape, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(torch.bfloat16)


def special_rows(rows, cols, seed):
    """bf16 rows with blocks of zeros, of one value, tiny, huge and far-apart values."""
    x = normal((rows, cols), seed)
    x[0, :128] = 0
    x[-1, -128:] = 0
    x[-1, -1] = -3.0
    if rows > 2:
        x[1] *= 2.0 ** -120
        x[2] *= 2.0 ** 100
        x[2, 5] = 2.0 ** 60
    return x


# ---- quantizers ----------------------------------------------------------------------------


@pytest.mark.parametrize("rows,cols", [(1, 128), (3, 256), (17, 7168), (300, 896), (129, 128)])
def test_quantize_rows_bits(cuda, rows, cols):
    x = special_rows(rows, cols, rows + cols)
    codes, scales = fp8.quantize_rows(x.to(cuda))
    v = x.float().numpy().reshape(rows, -1, 128)
    s, inv = R.block_scales(np.abs(v).max(2))
    np.testing.assert_array_equal(scales.cpu().numpy(), s)
    np.testing.assert_array_equal(codes.view(torch.uint8).cpu().numpy(),
                                  R.encode(v * inv[:, :, None]).reshape(rows, cols))


@pytest.mark.parametrize("rows,cols", [(1, 128), (128, 256), (129, 384), (300, 128), (1000, 1024)])
def test_quantize_weight_bits(cuda, rows, cols):
    w = special_rows(rows, cols, rows * 3 + cols)
    codes, scales = fp8.quantize_weight(w.to(cuda))
    pad = np.zeros((-(-rows // 128) * 128, cols), dtype=np.float32)
    pad[:rows] = w.float().numpy()
    v = pad.reshape(-1, 128, cols // 128, 128)
    s, inv = R.block_scales(np.abs(v).max((1, 3)))
    np.testing.assert_array_equal(scales.cpu().numpy(), s)
    want = R.encode(v * inv[:, None, :, None]).reshape(-1, cols)[:rows]
    np.testing.assert_array_equal(codes.view(torch.uint8).cpu().numpy(), want)


def test_quantize_every_bf16(cuda):
    """Every finite bf16 value, each block led by the power of two that sets its scale."""
    bits = np.arange(1 << 16, dtype=np.uint32)
    v = (bits << 16).view(np.float32)
    v = v[np.isfinite(v)]
    v = np.concatenate([v, np.zeros(-len(v) % 128, dtype=np.float32)])
    x = torch.from_numpy(v.reshape(-1, 128)).to(torch.bfloat16)
    codes, scales = fp8.quantize_rows(x.to(cuda))
    s, inv = R.block_scales(np.abs(v.reshape(-1, 128)).max(1))
    np.testing.assert_array_equal(scales.cpu().numpy()[:, 0], s)
    np.testing.assert_array_equal(codes.view(torch.uint8).cpu().numpy(),
                                  R.encode(v.reshape(-1, 128) * inv[:, None]))


def test_quantize_non_finite(cuda):
    """A NaN has a NaN code; a block with an infinity gives NaN in every product."""
    x = normal((3, 256), 5)
    x[0, 7] = float("nan")
    x[1, 130] = float("inf")
    codes, scales = fp8.quantize_rows(x.to(cuda))
    held = codes.float().cpu()
    assert torch.isnan(held[0, 7]) and torch.isnan(held[0]).sum() == 1
    assert torch.isnan(held[1, 130]) and torch.isinf(scales[1, 1]).item()
    assert torch.isfinite(held[2]).all() and torch.isfinite(scales[2]).all().item()
    w, ws = fp8.quantize_weight(normal((40, 256), 6, 0.02).to(cuda))
    for rows in (x, x[:1], x[1:2], torch.cat([x] * 30)):
        y = fp8.product(rows.to(cuda), w, ws).float().cpu()
        finite = torch.isfinite(rows.float()).all(1)
        assert torch.isnan(y[~finite]).all() and torch.isfinite(y[finite]).all()


# ---- product -------------------------------------------------------------------------------


def check_product(cuda, T, rows, cols, seed, x=None):
    x = special_rows(T, cols, seed) if x is None else x
    if T > 2 and cols > 0:
        x[2] = normal((cols,), seed + 9)  # the huge row would swamp nothing but itself; keep it finite
    w = normal((rows, cols), seed + 1, 0.02)
    wq, ws = fp8.quantize_weight(w.to(cuda))
    out = torch.full((T + 2, rows), -7.0, dtype=torch.bfloat16, device=cuda)
    fp8.product(x.to(cuda), wq, ws, out=out[1:T + 1])
    got = out.cpu()
    assert (got[0] == -7).all() and (got[-1] == -7).all()  # rows before and behind
    q, s = R.rows64(x.float().numpy())
    y, err = R.product64(q, s, R.values(wq), ws.cpu().double())
    off = (got[1:-1].double() - y).abs()
    bound = R.bf16_bound(y, err) + 2.0 ** -133  # a subnormal result's own half step
    assert (off <= bound).all(), (off / bound).max()
    return x, wq, ws, got[1:-1]


# tokens at the edges of 16-, 32-, 64- and 128-row tiles, rows at those of 16, 64, 128 and 256
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 8, 16, 17, 32, 33, 64, 65, 100, 128, 129, 257])
@pytest.mark.parametrize("rows,cols", [(1, 128), (130, 640), (256, 256)])
def test_product_small(cuda, T, rows, cols):
    check_product(cuda, T, rows, cols, 100 * T + rows)


@pytest.mark.parametrize("T,rows,cols", [
    (1, 2048, 7168), (1, 17, 7168), (1, 4100, 128), (2, 576, 2048), (7, 1000, 1536), (16, 2048, 7168),
    (31, 512, 4096), (61, 1100, 2048), (96, 257, 1024), (200, 1030, 896), (300, 4100, 1024),
    (513, 700, 512), (1000, 300, 640), (1029, 2049, 256)])
def test_product_sizes(cuda, T, rows, cols):
    check_product(cuda, T, rows, cols, T + rows + cols)


def test_product_repeats_its_bits(cuda):
    for T in (1, 37, 300):
        x, wq, ws, y = check_product(cuda, T, 700, 1024, T)
        for _ in range(3):
            assert torch.equal(fp8.product(x.to(cuda), wq, ws).cpu().view(torch.int16),
                               y.view(torch.int16))


def test_product_odd_output_alignment(cuda):
    """An output that starts at 2 bytes past a boundary: the same bits."""
    for T in (1, 20, 150):
        x, w = normal((T, 512), T).to(cuda), normal((260, 512), T + 1, 0.02).to(cuda)
        wq, ws = fp8.quantize_weight(w)
        want = fp8.product(x, wq, ws)
        room = torch.zeros(T * 260 + 2, dtype=torch.bfloat16, device=cuda)
        fp8.product(x, wq, ws, out=room[1:T * 260 + 1].view(T, 260))
        assert torch.equal(room[1:-1].view(T, 260), want) and room[0] == 0 and room[-1] == 0


def test_product_large_offsets(cuda):
    """A weight of more than 2^32 bytes: its last rows."""
    rows, cols = 300_000, 16384
    codes = torch.zeros((rows, cols), dtype=torch.uint8, device=cuda)
    scales = torch.ones((-(-rows // 128), cols // 128), device=cuda)
    tail = R.encode(np.random.default_rng(1).uniform(-4, 4, (5, cols)).astype(np.float32))
    codes[-5:] = torch.from_numpy(tail).to(cuda)
    for T in (1, 3, 40, 130):
        x = normal((T, cols), T)
        got = fp8.product(x.to(cuda), codes, scales)[:, -6:].cpu()
        q, s = R.rows64(x.float().numpy())
        y, err = R.product64(q, s, R.values(tail), torch.ones((1, cols // 128), dtype=torch.float64))
        assert (got[:, 0] == 0).all()
        assert ((got[:, 1:].double() - y).abs() <= R.bf16_bound(y, err)).all()


def test_product_refuses(cuda):
    x = normal((4, 256), 1).to(cuda)
    wq, ws = fp8.quantize_weight(normal((64, 256), 2).to(cuda))
    for bad in (lambda: fp8.product(x[:, :128], wq, ws), lambda: fp8.product(x.t(), wq, ws),
                lambda: fp8.product(x.float(), wq, ws), lambda: fp8.product(x, wq, ws[:, :1]),
                lambda: fp8.product(x, wq.t(), ws), lambda: fp8.product(x, wq, ws.double()),
                lambda: fp8.product(x, wq, ws, out=torch.empty_like(x)),
                lambda: fp8.product(x[:0], wq, ws), lambda: fp8.quantize_rows(x[:, :100].contiguous())):
        with pytest.raises((ValueError, RuntimeError)):
            bad()


# ---- experts -------------------------------------------------------------------------------


def make_store(cuda, E, H, F, seed):
    return fp8.Fp8ExpertStore.synthetic(E, H, F, seed, device=cuda)


def reference(store, x, ids, weights, residual, swiglu, E):
    """(output64, bound) of the expert stage, invalid and repeated routes left out."""
    T, k = ids.shape
    total = torch.zeros(x.shape, dtype=torch.float64)
    err = torch.zeros_like(total)
    seen = [[] for _ in range(E)]
    for t in range(T):
        for r in range(k):
            e = int(ids[t, r])
            if 0 <= e < E and e not in ids[t, :r].tolist():
                seen[e].append((t, r))
    rows = x.float().numpy()
    for e, routes in enumerate(seen):
        if not routes:
            continue
        t = [a for a, _ in routes]
        mats = [(R.values(c[e]), s[e].cpu().double()) for c, s in (store.gate, store.up, store.down)]
        y, ey = R.expert64(rows[t], *mats, swiglu)
        ey = R.bf16_bound(y, ey)
        w = torch.tensor([float(weights[a, b]) for a, b in routes], dtype=torch.float64)[:, None]
        for i, a in enumerate(t):
            total[a] += y[i] * w[i]
            # the weighted bf16 row, and 3 roundings of fp32 a route in the sum (k <= 32)
            err[a] += ey[i] * w[i].abs() + 64 * R.U * (y[i].abs() + ey[i]) * w[i].abs()
    err = R.bf16_bound(total, err)
    if residual is not None:
        total = total + residual.double()
        err = R.bf16_bound(total, err)
    return total, err


def check_experts(cuda, store, T, k, act, seed, ids=None, residual=True, weights=None):
    E, H = store.experts, store.hidden
    x = normal((T, H), seed)
    r = normal((T, H), seed + 1) if residual else None
    g = torch.Generator().manual_seed(seed + 2)
    if ids is None:
        ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(torch.int32)
    if weights is None:
        weights = torch.rand((T, k), generator=g) + 0.1
    sh = fp8.shape(H, E, k, store.ffn, 1.0, act)
    out = torch.full((T + 1, H), 9.0, dtype=torch.bfloat16, device=cuda)
    fp8.experts(x.to(cuda), ids.to(cuda), weights.to(cuda), store.table, sh,
                None if r is None else r.to(cuda), out=out[:T])
    got = out.cpu()
    assert (got[T] == 9).all()
    want, bound = reference(store, x, ids, weights, r, act == ACT_SWIGLU, E)
    off = (got[:T].double() - want).abs()
    assert (off <= bound).all(), (off / bound).max()
    # the bound is a worst case: the rows as a whole are far inside it
    assert torch.linalg.norm(off) <= 0.02 * torch.linalg.norm(want) + 1e-30
    return got[:T]


SIZES = [(4, 128, 128, 2), (8, 256, 384, 3), (16, 1024, 512, 4), (5, 384, 256, 5)]


@pytest.mark.parametrize("E,H,F,k", SIZES)
@pytest.mark.parametrize("T", [1, 2, 3, 17, 70])
@pytest.mark.parametrize("act", [ACT_SWIGLU, ACT_SITU])
def test_experts(cuda, E, H, F, k, T, act):
    check_experts(cuda, make_store(cuda, E, H, F, E), T, k, act, 1000 * T + E, residual=T != 17)


@pytest.mark.parametrize("rows", [1, 15, 16, 17, 32, 33, 63, 64, 65, 127, 128, 129, 200, 300])
def test_experts_rows_of_one_expert(cuda, rows):
    """Every token at expert 2, some at expert 0: the edges of every row tile."""
    store = make_store(cuda, 4, 256, 256, 3)
    ids = torch.full((rows, 2), 2, dtype=torch.int32)
    ids[:, 1] = 7                    # no such expert
    ids[: rows // 3, 1] = 0
    check_experts(cuda, store, rows, 2, ACT_SWIGLU, rows, ids=ids)


@pytest.mark.parametrize("T", [1, 5, 40])
def test_experts_invalid_and_repeated_routes(cuda, T):
    store = make_store(cuda, 6, 128, 256, 4)
    ids = torch.randint(0, 6, (T, 4), generator=torch.Generator().manual_seed(T), dtype=torch.int32)
    ids[0] = torch.tensor([3, 3, -1, 3])
    ids[-1, 1:] = ids[-1, :1]
    check_experts(cuda, store, T, 4, ACT_SWIGLU, T, ids=ids)
    ids[:] = 6                       # nothing is routed: the residual alone
    x, r = normal((T, 128), 1), normal((T, 128), 2)
    got = fp8.experts(x.to(cuda), ids.to(cuda), torch.ones((T, 4), device=cuda), store.table,
                      fp8.shape(128, 6, 4, 256, 1.0, ACT_SWIGLU), r.to(cuda))
    assert torch.equal(got.cpu(), r)


def test_experts_one_expert_top_32(cuda):
    check_experts(cuda, make_store(cuda, 1, 256, 128, 5), 33, 1, ACT_SWIGLU, 8)
    check_experts(cuda, make_store(cuda, 40, 128, 128, 6), 9, 32, ACT_SITU, 9)
    check_experts(cuda, make_store(cuda, 40, 128, 128, 6), 1, 32, ACT_SITU, 10)


def test_experts_zero_and_negative_weights(cuda):
    store = make_store(cuda, 8, 256, 256, 7)
    w = torch.tensor([[0.0, -1.5, 2.0]]).repeat(20, 1)
    check_experts(cuda, store, 20, 3, ACT_SWIGLU, 11, weights=w)
    check_experts(cuda, store, 1, 3, ACT_SWIGLU, 12, weights=w[:1])


def test_experts_tokens_do_not_touch_each_other(cuda):
    """A NaN row stays in its row, and every batch of a token set repeats its bits."""
    store = make_store(cuda, 16, 512, 256, 8)
    g = torch.Generator().manual_seed(3)
    T, k = 50, 4
    x = normal((T, 512), 4).to(cuda)
    ids = torch.stack([torch.randperm(16, generator=g)[:k] for _ in range(T)]).to(torch.int32).to(cuda)
    w = torch.rand((T, k), generator=g).to(cuda)
    sh = fp8.shape(512, 16, k, 256, 1.0, ACT_SWIGLU)
    want = fp8.experts(x, ids, w, store.table, sh)
    y = x.clone()
    y[13, 5] = float("nan")
    got = fp8.experts(y, ids, w, store.table, sh)
    keep = torch.arange(T, device=cuda) != 13
    assert torch.isnan(got[13]).all()
    assert torch.equal(got[keep], want[keep])
    for _ in range(3):
        assert torch.equal(fp8.experts(x, ids, w, store.table, sh), want)


def test_experts_refuse(cuda):
    store = make_store(cuda, 4, 128, 128, 2)
    sh = fp8.shape(128, 4, 2, 128, 1.0, ACT_SWIGLU)
    x, ids, w = normal((3, 128), 1).to(cuda), torch.zeros((3, 2), dtype=torch.int32, device=cuda), \
        torch.ones((3, 2), device=cuda)
    ok = dict(hidden=x, ids=ids, weights=w, table=store.table, shape=sh)
    for bad in (dict(ids=ids.long()), dict(ids=ids[:, :1]), dict(weights=w.double()),
                dict(table=store.table[:3]), dict(hidden=x.float()), dict(hidden=x.t()),
                dict(residual=x[:2]), dict(out=x[:1]), dict(weights=w.cpu()),
                dict(shape=fp8.shape(256, 4, 2, 128, 1.0, ACT_SWIGLU))):
        with pytest.raises(ValueError):
            fp8.experts(**{**ok, **bad})


# ---- layer, streams, graphs ----------------------------------------------------------------


def layer(cuda, T, E=32, H=512, F=256, k=4, seed=50):
    cfg = Config("fp8-small", T, H, E, k, F, seed=seed)
    g = torch.Generator().manual_seed(seed)
    rw = (torch.randn((E, H), generator=g) * 0.02).to(torch.bfloat16).to(cuda)
    rb = (torch.randn(E, generator=g) * 0.01).to(cuda)
    return fp8.Fp8RoutedMoE(cfg, rw, rb, make_store(cuda, E, H, F, seed)), normal((T, H), seed + 1).to(cuda)


@pytest.mark.parametrize("T", [1, 6, 100])
def test_layer_is_router_then_experts(cuda, T):
    import _ops
    moe, x = layer(cuda, T)
    E, k = moe.cfg.experts, moe.cfg.top_k
    ids = torch.zeros((T, k), dtype=torch.int32, device=cuda)
    w = torch.zeros((T, k), device=cuda)
    out = moe.forward(x, x, ids=ids, weights=w)
    logits = torch.empty((T, E), device=cuda)
    assert _ops.k3_rocm_bf16_gemm_f32(logits, moe.router_weight, x, T, E, x.shape[1])
    ids2, w2 = torch.zeros_like(ids), torch.zeros_like(w)
    assert _ops.k3_rocm_router_topk_f32_batch(ids2, w2, logits, moe.router_bias, T, E, k, moe.cfg.scale)
    assert torch.equal(ids, ids2) and torch.equal(w, w2)
    assert torch.equal(out, moe.experts_only(x, ids, w, x))
    assert torch.equal(moe.forward(x, x), out)


@pytest.mark.parametrize("T", [1, 5, 90])
def test_layer_on_another_stream_and_in_graphs(cuda, T):
    """Two captured graphs of two layers, replayed in turn with eager calls between."""
    moes = [layer(cuda, T, seed=60), layer(cuda, T, seed=61)]
    want = [m.forward(x, x) for m, x in moes]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [m.forward(x, x) for m, x in moes]
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graphs, outs, inputs = [], [], [x.clone() for _, x in moes]
    for (m, _), x in zip(moes, inputs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(m.forward(x, x))
        graphs.append(g)
    for n in range(3):
        new = [normal(x.shape, 70 + n + i).to(cuda) for i, x in enumerate(inputs)]
        for g, x, v in zip(graphs, inputs, new):
            x.copy_(v)
            g.replay()
        eager = [m.forward(v, v) for (m, _), v in zip(moes, new)]
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T", [1, 20, 150])
def test_product_in_a_graph(cuda, T):
    x = normal((T, 1024), T).to(cuda)
    wq, ws = fp8.quantize_weight(normal((520, 1024), 3, 0.02).to(cuda))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = fp8.product(x, wq, ws)
    for n in range(4):
        v = normal((T, 1024), 30 + n).to(cuda)
        x.copy_(v)
        g.replay()
        want = fp8.product(v, wq, ws)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


# ---- native block --------------------------------------------------------------------------


@pytest.mark.parametrize("T", [1, 5, 100])
@pytest.mark.parametrize("shared_stream", [False, True])
def test_native_block_fp8_statics(cuda, T, shared_stream):
    """The block with FP8-128 projections is its entry points in order, bit for bit."""
    import _ops
    from moonshine_amd.layer import RoutedMoE
    cfg = N.NativeConfig("native-fp8", T, 1024, 512, 64, 4, 256, 768, static_kind=N.STATIC_FP8,
                         seed=2100)
    blk = N.NativeLayer(cfg, device=cuda)
    x, r = normal((T, 1024), T).to(cuda), normal((T, 1024), T + 1).to(cuda)
    ids = torch.zeros((T, 4), dtype=torch.int32, device=cuda)
    w = torch.zeros((T, 4), device=cuda)
    side = torch.cuda.Stream() if shared_stream else None
    out = blk.forward(x, r, ids=ids, weights=w, shared_stream=side.cuda_stream if side else None)
    torch.cuda.synchronize()
    mul = lambda s, v: fp8.product(v, s.data, s.scales)  # noqa: E731
    latent = mul(blk.routed_down, x)
    class Held:                      # RoutedMoE over the block's experts
        table = blk.store.table
    import dataclasses
    from moonshine_amd.synth import Config as C
    moe = RoutedMoE(C("x", T, 512, 64, 4, 256, scale=cfg.scale, activation=cfg.activation,
                      beta=cfg.beta, linear_beta=cfg.linear_beta), x, r, Held)
    routed = moe.experts_only(latent, ids, w)
    normed = torch.empty_like(routed)
    assert _ops.k3_rocm_rms_norm_bf16(normed, routed, blk.norm, T, 512, cfg.eps)
    full = mul(blk.routed_up, normed)
    gate, up = mul(blk.shared_gate, x), mul(blk.shared_up, x)
    act = torch.empty_like(gate)
    assert _ops.k3_rocm_situ_bf16(act, gate, up, act.numel(), cfg.beta, cfg.linear_beta)
    shared = mul(blk.shared_down, act)
    total, want = torch.empty_like(full), torch.empty_like(full)
    assert _ops.k3_rocm_add_bf16(total, full, shared, full.numel())
    assert _ops.k3_rocm_add_bf16(want, r, total, full.numel())
    assert torch.equal(out, want)
    # an unaligned weight is refused, as the product refuses it
    blk.weights.shared_down.data += 8
    with pytest.raises(RuntimeError):
        blk.forward(x, r)
