"""Products grouped by expert where they can go wrong: rows that none or all experts have, indices and
offsets out of range, values that must not be read, memory that must stay, graphs and streams."""
import pytest
import torch

import _grouped as R
from moonshine_amd import grouped
from test_gpu_grouped import equal, laid_out

pytestmark = pytest.mark.gpu

NAN = float("nan")


def ints(values, cuda):
    return torch.tensor(values, dtype=torch.int32, device=cuda)


@pytest.mark.parametrize("n", [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 96, 127, 128, 129, 160, 161, 192, 224, 255, 256, 257,
                               288, 320, 512, 513, 1537])
def test_rows_of_an_expert_at_the_edges_of_its_tiles(cuda, n):
    """Between experts of one row; columns of one whole and one part tile, a part of a stage."""
    E, N, K = 3, 328, 104
    counts = [1, n, 1]
    offsets = torch.tensor([0, 1, n + 1, n + 2], dtype=torch.int32)
    w, x, dy = R.whole((E, N, K), n), R.whole((n + 2, K), n + 1), R.whole((n + 2, N), n + 2)
    o, rows = offsets.to(cuda), sum(counts)
    assert rows == n + 2
    equal(grouped.product(x.to(cuda), w.to(cuda), o), R.by_rows(x, w, offsets, None, False)[0])
    equal(grouped.input_gradient(dy.to(cuda), w.to(cuda), o), R.by_rows(dy, w, offsets, None, True)[0])
    equal(grouped.weight_gradient(dy.to(cuda), x.to(cuda), o), R.by_weights(dy, x, offsets, None, None)[0])


@pytest.mark.parametrize("N,K", [(8, 8), (8, 1000), (1000, 8), (64, 56), (120, 136), (136, 120), (248, 264), (264, 248),
                                 (512, 64), (520, 72)])
@pytest.mark.parametrize("n", [3, 200])
def test_widths(cuda, N, K, n):
    E = 2
    offsets = torch.tensor([0, n, 2 * n + 1], dtype=torch.int32)
    w, x, dy = R.whole((E, N, K), 1), R.whole((2 * n + 1, K), 2), R.whole((2 * n + 1, N), 3)
    o = offsets.to(cuda)
    equal(grouped.product(x.to(cuda), w.to(cuda), o), R.by_rows(x, w, offsets, None, False)[0])
    equal(grouped.input_gradient(dy.to(cuda), w.to(cuda), o), R.by_rows(dy, w, offsets, None, True)[0])
    for dtype in (torch.float32, torch.bfloat16):
        equal(grouped.weight_gradient(dy.to(cuda), x.to(cuda), o, dtype=dtype),
              R.by_weights(dy, x, offsets, None, None)[0])


@pytest.mark.parametrize("n", [5, 70, 300])
def test_what_lies_behind_is_neither_read_nor_written(cuda, n):
    """NaN in rows past the last expert's, in rows of the tensors that no index names, and in
    experts without rows; outputs keep what they held there."""
    E, N, K = 4, 72, 136
    offsets = torch.tensor([0, n, n, n + 3, n + 3], dtype=torch.int32)
    used, R_ = n + 3, n + 40
    o = offsets.to(cuda)
    w = R.whole((E, N, K), 1)
    w[1], w[3] = NAN, NAN
    x, dy = R.whole((R_, K), 2), R.whole((R_, N), 3)
    x[used:], dy[used:] = NAN, NAN
    out = torch.full((R_, N), 7.0, dtype=torch.bfloat16, device=cuda)
    grouped.product(x.to(cuda), w.to(cuda), o, out=out)
    equal(out[:used], R.by_rows(x[:used], w, offsets, None, False)[0].nan_to_num())
    assert (out[used:] == 7).all()
    dx = torch.full((R_, K), 7.0, dtype=torch.bfloat16, device=cuda)
    grouped.input_gradient(dy.to(cuda), w.to(cuda), o, out=dx)
    equal(dx[:used], R.by_rows(dy[:used], w, offsets, None, True)[0])
    assert (dx[used:] == 7).all()
    want = R.by_weights(dy[:used], x[:used], offsets, None, None)[0]
    equal(grouped.weight_gradient(dy.to(cuda), x.to(cuda), o), want)
    assert not want[1].any() and not want[3].any()
    # picked from a larger tensor, whose other rows are NaN
    big = torch.full((2 * R_, K), NAN, dtype=torch.bfloat16)
    big[1::2] = x
    index = (2 * torch.arange(R_, dtype=torch.int32) + 1).to(cuda)
    equal(grouped.product(big.to(cuda), w.to(cuda), o, index=index)[:used],
          R.by_rows(x[:used], w, offsets, None, False)[0])
    equal(grouped.weight_gradient(dy.to(cuda), big.to(cuda), o, x_index=index), want)


@pytest.mark.parametrize("n", [6, 150, 400])
def test_indices_out_of_range(cuda, n):
    """A row picked from nowhere is zeros, one sent nowhere is not written."""
    E, N, K = 2, 80, 72
    offsets = torch.tensor([0, n // 3, n], dtype=torch.int32)
    w, x, dy = R.whole((E, N, K), 1), R.whole((9, K), 2), R.whole((n, N), 3)
    index = torch.arange(n, dtype=torch.int32) % 9
    index[::4], index[1], index[2] = 9, -1, 1 << 24
    o = offsets.to(cuda)
    equal(grouped.product(x.to(cuda), w.to(cuda), o, index=index.to(cuda)), R.by_rows(x, w, offsets, index, False)[0])
    equal(grouped.weight_gradient(dy.to(cuda), x.to(cuda), o, x_index=index.to(cuda)),
          R.by_weights(dy, x, offsets, None, index)[0])
    d = R.whole((9, N), 4)
    equal(grouped.input_gradient(d.to(cuda), w.to(cuda), o, index=index.to(cuda)),
          R.by_rows(d, w, offsets, index, True)[0])
    equal(grouped.weight_gradient(d.to(cuda), R.whole((n, K), 5).to(cuda), o, dy_index=index.to(cuda)),
          R.by_weights(d, R.whole((n, K), 5), offsets, index, None)[0])
    to = torch.arange(n, dtype=torch.int32).flip(0)
    to[0], to[3] = n, -1
    out = torch.full((n, K), 7.0, dtype=torch.bfloat16, device=cuda)
    grouped.input_gradient(dy.to(cuda), w.to(cuda), o, to=to.to(cuda), out=out)
    want = torch.full((n, K), 7.0, dtype=torch.float64)
    rows = R.by_rows(dy, w, offsets, None, True)[0]
    ok = (to >= 0) & (to < n)
    want[to[ok].long()] = rows[ok]
    equal(out, want)


@pytest.mark.parametrize("values", [[0, 900, 5, 40], [0, 10, 1 << 30, 1 << 30], [-5, 3, 9, 12], [40, 40, 40, 40]])
def test_offsets_out_of_range_stay_in_memory(cuda, values):
    """Offsets that no plan makes: no row outside is read or written."""
    E, N, K, rows = 3, 72, 64, 40
    w, x, dy = R.whole((E, N, K), 1).to(cuda), R.whole((rows, K), 2).to(cuda), R.whole((rows, N), 3).to(cuda)
    o = ints(values, cuda)
    room = torch.full((3 * rows, N), 7.0, dtype=torch.bfloat16, device=cuda)
    grouped.product(x, w, o, out=room[rows:2 * rows])
    assert (room[:rows] == 7).all() and (room[2 * rows:] == 7).all()
    assert grouped.input_gradient(dy, w, o).shape == (rows, K)
    assert grouped.weight_gradient(dy, x, o).shape == (E, N, K)
    torch.cuda.synchronize()


@pytest.mark.parametrize("E,N,K", [(3, 72, 136), (2, 300 // 4 * 4 + 4, 520)])
def test_accumulates_in_fp32(cuda, E, N, K):
    n = 90
    offsets = torch.tensor([0, n, n] + [2 * n] * (E - 2), dtype=torch.int32)
    dy, x = R.whole((2 * n, N), 1), R.whole((2 * n, K), 2)
    start = torch.randint(-9, 9, (E, N, K), generator=torch.Generator().manual_seed(3)).float()
    out = start.to(cuda)
    got = grouped.weight_gradient(dy.to(cuda), x.to(cuda), offsets.to(cuda), out=out, accumulate=True)
    assert got.data_ptr() == out.data_ptr()
    equal(got, start.double() + R.by_weights(dy, x, offsets, None, None)[0])


def test_past_32_bits(cuda):
    """An expert's weights, and their gradient, past 4 GiB of the tensor; rows past 4 GiB."""
    E, N, K = 9, 16384, 16384
    w = torch.zeros((E, N, K), dtype=torch.bfloat16, device=cuda)
    w[8] = R.whole((N, K), 1).to(cuda)
    offsets = ints([0] + [1] * 8 + [4], cuda)
    x = R.whole((4, K), 2).to(cuda)
    x[0] = 0
    want = torch.zeros((4, N), dtype=torch.float64, device=cuda)
    want[1:] = x[1:].double() @ w[8].double().t()
    equal(grouped.product(x, w, offsets), want.cpu())
    dy = R.whole((4, N), 3).to(cuda)
    want[:, :] = 0
    want[1:] = dy[1:].double() @ w[8].double()
    equal(grouped.input_gradient(dy, w, offsets), want.cpu())
    del w
    g = grouped.weight_gradient(dy, x, offsets, dtype=torch.bfloat16)
    assert torch.equal(g[8].double(), (dy[1:].double().t() @ x[1:].double()).to(torch.bfloat16).double())
    assert not g[:8].any()
    del g
    rows = 140000  # x 16384 x 2 bytes
    x = torch.zeros((rows, K), dtype=torch.bfloat16, device=cuda)
    x[-2:] = R.whole((2, K), 4).to(cuda)
    w = R.whole((2, 40, K), 5).to(cuda)
    got = grouped.product(x, w, ints([0, rows - 1, rows], cuda))
    assert torch.equal(got[-1].double(), (x[-1].double() @ w[1].double().t()).to(torch.bfloat16).double())
    assert torch.equal(got[-2].double(), (x[-2].double() @ w[0].double().t()).to(torch.bfloat16).double())
    assert not got[:-2].any()
    dy = R.whole((rows, 8), 6).to(cuda)
    g = grouped.weight_gradient(dy, x, ints([0, rows - 1, rows], cuda))
    assert torch.equal(g[1].double(), dy[-1].double()[:, None] * x[-1].double()[None])
    assert torch.equal(g[0].double(), dy[-2].double()[:, None] * x[-2].double()[None])


def test_the_same_bits_again_on_streams_and_in_graphs(cuda):
    """Two graphs and a stream at once, replayed between the program's own work, on new inputs."""
    T, k, E, N, K = 300, 2, 5, 264, 328
    made = []
    for seed in (1, 2):
        ids, p, _ = laid_out(T, k, E, 1.0, seed, cuda)
        x, w = R.normal((T, K), seed).to(cuda), R.normal((E, N, K), seed + 5).to(cuda)
        dy = R.normal((T * k, N), seed + 9).to(cuda)

        def step(x=x, w=w, dy=dy, p=p):
            return (grouped.product(x, w, p.offsets, index=p.token_index), grouped.input_gradient(dy, w, p.offsets),
                    grouped.weight_gradient(dy, x, p.offsets, x_index=p.token_index))

        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        made.append((g, step, out, x))
    side = torch.cuda.Stream()
    for turn in range(3):
        for i, (g, step, out, x) in enumerate(made):
            x.copy_(R.normal(tuple(x.shape), 50 + 2 * turn + i).to(cuda))
        want = [[t.clone() for t in step()] for _, step, _, _ in made]
        torch.cuda.synchronize()
        for g, _, _, _ in made:
            g.replay()
        with torch.cuda.stream(side):
            again = made[0][1]()
        torch.cuda.synchronize()
        for (g, _, out, _), w in zip(made, want):
            assert all(torch.equal(a, b) for a, b in zip(out, w))
        assert all(torch.equal(a, b) for a, b in zip(again, want[0]))


def test_refused_over_its_operands(cuda):
    room = R.whole((160, 64), 1).to(cuda)
    before = room.clone()
    o = ints([0, 8], cuda)
    rows, w = room[:8], room[16:80].view(1, 64, 64)
    for out in (room[4:12], room[:8], room[40:48], room[79:87]):
        for fn in (grouped.product, grouped.input_gradient):
            with pytest.raises(RuntimeError):
                fn(rows, w, o, out=out)
    big = room[4:132].view(-1).view(torch.float32).view(1, 64, 64)
    with pytest.raises(RuntimeError):
        grouped.weight_gradient(rows, rows, o, out=big)
    assert torch.equal(room, before)
    got = grouped.product(rows, w, o, out=room[8:16])  # between them
    equal(got, R.by_rows(rows.cpu(), w.cpu(), o.cpu(), None, False)[0])


def test_both_operands_picked(cuda):
    """A weight gradient whose rows both come by indices, some more than once; more tiles than a turn of the
    XCDs, of part tiles and of experts with no row, one, and more than a stage."""
    counts = [1, 0, 31, 33, 200, 64, 97]
    E, N, K, have = len(counts), 520, 1416, 50
    offsets = torch.tensor([0] + counts, dtype=torch.int32).cumsum(0).to(torch.int32)
    g = torch.Generator().manual_seed(1)
    i, j = (torch.randint(0, have, (sum(counts),), generator=g).to(torch.int32) for _ in range(2))
    j[3], i[100] = -1, have
    dy, x = R.whole((have, N), 2), R.whole((have, K), 3)
    want = R.by_weights(dy, x, offsets, i, j)[0]
    o, i, j = offsets.to(cuda), i.to(cuda), j.to(cuda)
    for dtype in (torch.float32, torch.bfloat16):
        equal(grouped.weight_gradient(dy.to(cuda), x.to(cuda), o, dy_index=i, x_index=j, dtype=dtype), want)
    out = torch.ones((E, N, K), device=cuda)
    equal(grouped.weight_gradient(dy.to(cuda), x.to(cuda), o, dy_index=i, x_index=j, out=out, accumulate=True), want + 1)


@pytest.mark.parametrize("K", [2040, 2048, 2056, 4104, 8200])
@pytest.mark.parametrize("n", [1, 16, 17])
def test_few_rows_of_long_reductions(cuda, n, K):
    E, N = 3, 40
    offsets = torch.tensor([0, n, n, n + 1], dtype=torch.int32)
    w, x = R.whole((E, N, K), 1), R.whole((n + 1, K), 2)
    equal(grouped.product(x.to(cuda), w.to(cuda), offsets.to(cuda)), R.by_rows(x, w, offsets, None, False)[0])


@pytest.mark.parametrize("E,rows", [(15, 15), (16, 16), (16, 32), (32, 4096), (32, 4097), (33, 4096)])
def test_where_one_kind_of_tile_takes_over_from_another(cuda, E, rows):
    """1024 columns: up to 1024 blocks of 16 x 16, up to 128 tiles of 256 columns and rows for one row tile
    an expert, and more; all rows of one expert, and spread."""
    wide, inner = 1024, 72
    spread = [rows * e // E for e in range(E + 1)]
    for values in (spread, [0] * (E - 1) + [0, rows]):
        offsets = torch.tensor(values, dtype=torch.int32)
        x = R.whole((rows, inner), 1)
        w = R.whole((E, wide, inner), 2)
        equal(grouped.product(x.to(cuda), w.to(cuda), offsets.to(cuda)), R.by_rows(x, w, offsets, None, False)[0])
        w = w.transpose(1, 2).contiguous()
        equal(grouped.input_gradient(x.to(cuda), w.to(cuda), offsets.to(cuda)), R.by_rows(x, w, offsets, None, True)[0])


@pytest.mark.parametrize("n", [4, 40])
def test_the_largest_tensor_that_an_index_picks_from(cuda, n):
    """65535 rows of 32768 values, just under 4 GiB: its last row, and the first that it has not."""
    rows, wide, inner = 65535, 32768, 8
    big = torch.zeros((rows, wide), dtype=torch.bfloat16, device=cuda)
    ends = R.whole((2, wide), 1)
    big[0], big[-1] = ends[0].to(cuda), ends[1].to(cuda)
    index = torch.tensor(([65534, 65535, 0, -1] * n)[:n], dtype=torch.int32)
    at = torch.tensor(([1, 2, 0, -1] * n)[:n], dtype=torch.int32)  # the same of `ends`
    offsets = torch.tensor([0, n], dtype=torch.int32)
    o, i = offsets.to(cuda), index.to(cuda)
    w, d = R.whole((1, inner, wide), 2), R.whole((n, inner), 3)
    equal(grouped.product(big, w.to(cuda), o, index=i), R.by_rows(ends, w, offsets, at, False)[0])
    equal(grouped.weight_gradient(d.to(cuda), big, o, x_index=i), R.by_weights(d, ends, offsets, None, at)[0])
    equal(grouped.weight_gradient(big, d.to(cuda), o, dy_index=i), R.by_weights(ends, d, offsets, at, None)[0])
    w = w.transpose(1, 2).contiguous()
    equal(grouped.input_gradient(big, w.to(cuda), o, index=i), R.by_rows(ends, w, offsets, at, True)[0])
