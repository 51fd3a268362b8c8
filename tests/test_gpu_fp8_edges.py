"""FP8-128 products and experts on the GPU where one kernel hands over to the next:
few tokens in one launch or in tiles, K in one part or several, an expert's rows at
its tiles' heights, a plan in one launch or several, the widest and longest calls.
Bounds as in tests/_fp8.py."""
import pytest
import torch

import _fp8 as R
from moonshine_amd import fp8
from moonshine_amd.synth import ACT_SITU, ACT_SWIGLU
from test_gpu_fp8 import check_experts, check_product, make_store, normal

pytestmark = pytest.mark.gpu


# ---- product -------------------------------------------------------------------------------


@pytest.mark.parametrize("T", [2, 3, 4, 5, 6, 7, 8, 9])
@pytest.mark.parametrize("rows,cols", [(16, 384), (4096, 256), (4100, 896), (33, 8320)])
def test_product_of_few_tokens(cuda, T, rows, cols):
    check_product(cuda, T, rows, cols, 7 * T + rows)


# tokens and rows at the edges of groups of 16 in one launch, and of its bounds
@pytest.mark.parametrize("T,rows,cols", [
    (9, 16, 128), (9, 4096, 128), (15, 17, 4096), (16, 2048, 1152), (17, 31, 2048), (31, 512, 1024), (48, 1365, 384),
    (64, 1024, 4096), (255, 256, 256), (256, 256, 128), (257, 256, 128), (4096, 16, 256), (4097, 16, 256)])
def test_product_by_groups_of_16(cuda, T, rows, cols):
    check_product(cuda, T, rows, cols, T + rows + 5)


# tokens at the edges of 16-, 32-, 64- and 128-row tiles
@pytest.mark.parametrize("T", [9, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 257])
@pytest.mark.parametrize("rows,cols", [(4100, 128), (130, 4224), (4352, 640)])
def test_product_tiles(cuda, T, rows, cols):
    check_product(cuda, T, rows, cols, 11 * T + rows)


@pytest.mark.parametrize("T", [20, 150, 300])
def test_product_tiles_output_alignment(cuda, T):
    """Outputs at 2, 8 and 16 bytes past a boundary, rows of 8 and of 4 columns: the same bits."""
    x = normal((T, 256), T).to(cuda)
    for rows in (4104, 4100, 4101):
        wq, ws = fp8.quantize_weight(normal((rows, 256), T + 1, 0.02).to(cuda))
        want = fp8.product(x, wq, ws)
        for at in (1, 4, 8):
            room = torch.full((T * rows + 16,), 3.0, dtype=torch.bfloat16, device=cuda)
            fp8.product(x, wq, ws, out=room[at:at + T * rows].view(T, rows))
            assert torch.equal(room[at:at + T * rows].view(T, rows), want)
            assert (room[:at] == 3).all() and (room[at + T * rows:] == 3).all()


# K whole and in 2 to 16 parts, the last one shorter; every height of tile
@pytest.mark.parametrize("T,rows,cols", [
    (9, 130, 16384), (20, 257, 7296), (33, 1030, 2176), (37, 4100, 4224), (70, 129, 8192), (97, 2050, 1664),
    (129, 513, 4736), (140, 5000, 640), (260, 300, 6272), (300, 4100, 2176), (515, 1030, 1152),
    (1030, 1300, 2176), (2050, 1030, 384), (65535, 130, 128)])
def test_product_cuts(cuda, T, rows, cols):
    check_product(cuda, T, rows, cols, T + 3 * rows + cols)


def test_product_of_many_parts_in_graphs(cuda):
    """Two graphs whose products cut K, replayed in turn with eager calls between."""
    wq, ws = fp8.quantize_weight(normal((1100, 7168), 3, 0.02).to(cuda))
    xs = [normal((T, 7168), T).to(cuda) for T in (37, 150)]
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(fp8.product(x, wq, ws))
        graphs.append(g)
    for n in range(4):
        new = [normal(x.shape, 40 + n).to(cuda) for x in xs]
        for x, v, g in zip(xs, new, graphs):
            x.copy_(v)
            g.replay()
        want = [fp8.product(v, wq, ws) for v in new]
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_calls_on_two_streams_at_once(cuda):
    store = make_store(cuda, 16, 512, 256, 8)
    sh = fp8.shape(512, 16, 4, 256, 1.0, ACT_SWIGLU)
    wq, ws = fp8.quantize_weight(normal((700, 512), 3, 0.02).to(cuda))
    g = torch.Generator().manual_seed(3)
    sets = []
    for T in (1, 6, 60, 300):
        x = normal((T, 512), T).to(cuda)
        ids = torch.stack([torch.randperm(16, generator=g)[:4] for _ in range(T)]).to(torch.int32).to(cuda)
        sets.append((x, ids, torch.rand((T, 4), generator=g).to(cuda)))

    def run(x, ids, w):
        return fp8.product(x, wq, ws), fp8.experts(x, ids, w, store.table, sh)

    want = [run(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] += [run(*s) for s in sets]
    torch.cuda.synchronize()
    for lane in got:
        for n, pair in enumerate(lane):
            for a, b in zip(pair, want[n % len(sets)]):
                assert torch.equal(a, b)


# ---- experts -------------------------------------------------------------------------------


@pytest.mark.parametrize("T", [255, 256, 257, 300, 1000, 1024, 1025])
@pytest.mark.parametrize("E,k", [(6, 4), (64, 8), (40, 32), (1024, 3)])
def test_experts_plan(cuda, T, E, k):
    """Any ids: valid ones, repeats and ids of no expert."""
    store = make_store(cuda, E, 128, 128, 4)
    ids = torch.randint(-1, E + 1, (T, k), generator=torch.Generator().manual_seed(T + E),
                        dtype=torch.int32)
    ids[3] = E
    check_experts(cuda, store, T, k, ACT_SWIGLU, T, ids=ids)


@pytest.mark.parametrize("rows", [31, 95, 96, 255, 256, 257, 288, 384, 385, 511, 512, 513, 700, 1025])
def test_experts_tile_heights(cuda, rows):
    """`rows` tokens at expert 1, a third and a tenth of them at experts 0 and 3."""
    store = make_store(cuda, 5, 256, 384, 3)
    ids = torch.full((rows, 3), 1, dtype=torch.int32)
    ids[:, 1:] = -5
    ids[: rows // 3, 1] = 0
    ids[rows - rows // 10:, 2] = 3
    check_experts(cuda, store, rows, 3, ACT_SITU, rows, ids=ids)


@pytest.mark.parametrize("H,F", [(8192, 256), (8320, 256), (256, 2048), (256, 2176), (256, 4096), (256, 4224),
                                 (384, 128), (128, 640)])
@pytest.mark.parametrize("T", [1, 3])
def test_experts_widths(cuda, H, F, T):
    check_experts(cuda, make_store(cuda, 3, H, F, 9), T, 2, ACT_SWIGLU, H + F)


@pytest.mark.parametrize("T", [2, 8, 16, 31, 64, 65])
@pytest.mark.parametrize("E,H,F,k", [(8, 256, 128, 8), (3, 2048, 1024, 2), (40, 384, 256, 9)])
def test_experts_one_by_one_or_in_tiles(cuda, E, H, F, k, T):
    """Any ids: valid ones, repeats and ids of no expert."""
    ids = torch.randint(-1, E + 1, (T, k), generator=torch.Generator().manual_seed(T + E),
                        dtype=torch.int32)
    ids[T // 2] = E
    check_experts(cuda, make_store(cuda, E, H, F, 9), T, k, ACT_SITU, H + T, ids=ids)


@pytest.mark.parametrize("H,F", [(512, 256), (1152, 640)])
def test_experts_bits_do_not_depend_on_the_batch(cuda, H, F):
    """A token alone, in a small and in a large batch."""
    E, k, T = 12, 4, 400
    store = make_store(cuda, E, H, F, 8)
    g = torch.Generator().manual_seed(5)
    x, r = normal((T, H), 4).to(cuda), normal((T, H), 5).to(cuda)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(torch.int32).to(cuda)
    w = torch.rand((T, k), generator=g).to(cuda)
    sh = fp8.shape(H, E, k, F, 1.0, ACT_SITU)
    want = fp8.experts(x, ids, w, store.table, sh, r)
    for n in (1, 2, 30, 100, 256, 399):
        got = fp8.experts(x[:n].contiguous(), ids[:n].contiguous(), w[:n].contiguous(), store.table, sh,
                          r[:n].contiguous())
        assert torch.equal(got, want[:n]), n
    for t in (7, 399):
        got = fp8.experts(x[t:t + 1], ids[t:t + 1], w[t:t + 1], store.table, sh, r[t:t + 1])
        assert torch.equal(got[0], want[t])


def test_experts_of_the_most_tokens(cuda):
    """65535 tokens: a sample of them against the same tokens in a small batch."""
    E, H, F, k, T = 8, 128, 128, 2, 65535
    store = make_store(cuda, E, H, F, 8)
    g = torch.Generator().manual_seed(6)
    x = normal((T, H), 4).to(cuda)
    ids = torch.randint(0, E + 1, (T, k), generator=g, dtype=torch.int32).to(cuda)
    w = torch.rand((T, k), generator=g).to(cuda)
    sh = fp8.shape(H, E, k, F, 1.0, ACT_SWIGLU)
    out = fp8.experts(x, ids, w, store.table, sh)
    some = torch.cat([torch.arange(0, T, 331), torch.tensor([T - 2, T - 1])]).to(cuda)
    got = fp8.experts(x[some], ids[some], w[some], store.table, sh)
    assert torch.equal(got, out[some])
    a = some[:40].cpu()
    check_experts(cuda, store, 40, k, ACT_SWIGLU, 7, ids=ids.cpu()[a])


@pytest.mark.parametrize("T", [1, 4, 300])
def test_experts_in_place(cuda, T):
    """The output in the place of the hidden rows, and of the residual's."""
    store = make_store(cuda, 8, 256, 128, 2)
    g = torch.Generator().manual_seed(9)
    ids = torch.stack([torch.randperm(8, generator=g)[:3] for _ in range(T)]).to(torch.int32).to(cuda)
    w = torch.rand((T, 3), generator=g).to(cuda)
    sh = fp8.shape(256, 8, 3, 128, 1.0, ACT_SWIGLU)
    x, r = normal((T, 256), 4).to(cuda), normal((T, 256), 5).to(cuda)
    want, alone = fp8.experts(x, ids, w, store.table, sh, r), fp8.experts(x, ids, w, store.table, sh, x)
    a, b, c = x.clone(), r.clone(), x.clone()
    assert torch.equal(fp8.experts(a, ids, w, store.table, sh, r, out=a), want)
    assert torch.equal(fp8.experts(x, ids, w, store.table, sh, b, out=b), want)
    assert torch.equal(fp8.experts(c, ids, w, store.table, sh, c, out=c), alone)


@pytest.mark.parametrize("T", [1, 5, 280])
def test_experts_weights_of_routes_that_are_none(cuda, T):
    """A route that is left out adds nothing, whatever its weight."""
    store = make_store(cuda, 6, 128, 128, 2)
    ids = torch.tensor([[4, 6, 4, 1]], dtype=torch.int32).repeat(T, 1)
    w = torch.tensor([[0.5, float("nan"), float("inf"), -2.0]]).repeat(T, 1)
    sh = fp8.shape(128, 6, 4, 128, 1.0, ACT_SWIGLU)
    x = normal((T, 128), 4).to(cuda)
    got = fp8.experts(x, ids.to(cuda), w.to(cuda), store.table, sh)
    w[:, 1:3] = 0
    want = fp8.experts(x, ids.to(cuda), w.to(cuda), store.table, sh)
    assert torch.isfinite(got).all() and torch.equal(got, want)


def test_product_refuses_an_output_over_its_input(cuda):
    wq, ws = fp8.quantize_weight(normal((256, 256), 3, 0.02).to(cuda))
    room = normal((12, 256), 4).to(cuda)
    before = room.clone()
    for T in (1, 3, 6):
        for to in (0, T - 1):
            with pytest.raises(RuntimeError):
                fp8.product(room[:T], wq, ws, out=room[to:to + T])
    assert torch.equal(room, before)
    fp8.product(room[:3], wq, ws, out=room[3:6])
    assert torch.equal(room[3:6], fp8.product(before[:3], wq, ws))
