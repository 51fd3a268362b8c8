"""The grouped products' row tiles where they can go wrong: of 256 columns ("wide") and of 128 ("narrow"), on
sizes past what goes 16 rows x 16 columns a block ("few"). kind() restates how a call is cut, and each test
asserts which kernel its sizes reach. Whole numbers, bit for bit (tests/_grouped.py)."""
import pytest
import torch

import _grouped as R
from moonshine_amd import grouped
from test_gpu_grouped import equal, laid_out

pytestmark = pytest.mark.gpu

NAN = float("nan")


def kind(direction, rows, experts, columns):
    used = min(rows, experts)
    if direction == "product" and (rows // 16 + used) * -(-columns // 16) <= 1024:
        return "few"
    return "narrow" if used * -(-columns // 256) <= 128 and rows <= 128 * used else "wide"


def ints(values, cuda):
    return torch.tensor(values, dtype=torch.int32, device=cuda)


def weights(direction, E, columns, z, seed):
    """[E, columns, z] for a product, [E, z, columns] for an input gradient."""
    return R.whole((E, columns, z) if direction == "product" else (E, z, columns), seed)


def call(direction, *args, **kwargs):
    return (grouped.product if direction == "product" else grouped.input_gradient)(*args, **kwargs)


def want(direction, rows, w, offsets, index=None):
    return R.by_rows(rows, w, offsets, index, direction == "input")[0]


@pytest.mark.parametrize("direction", ["product", "input"])
@pytest.mark.parametrize("columns,z,tile", [(5480, 104, "narrow"), (10760, 104, "wide"), (10888, 64, "wide")])
@pytest.mark.parametrize("n", [1, 16, 31, 32, 33, 63, 64, 65, 96, 127, 128, 129, 160, 161, 224, 255, 256, 257, 320, 512,
                               513, 1537])
def test_rows_of_an_expert_at_the_edges_of_its_tiles(cuda, direction, columns, z, tile, n):
    E, rows = 3, n + 2
    offsets = torch.tensor([0, 1, n + 1, n + 2], dtype=torch.int32)
    assert kind(direction, rows, E, columns) == (tile if n <= 382 else "wide")
    w, x = weights(direction, E, columns, z, n), R.whole((rows, z), n + 1)
    equal(call(direction, x.to(cuda), w.to(cuda), offsets.to(cuda)), want(direction, x, w, offsets))


@pytest.mark.parametrize("direction", ["product", "input"])
@pytest.mark.parametrize("columns,tile", [(5480, "narrow"), (10760, "wide")])
@pytest.mark.parametrize("z", [8, 40, 56, 72, 120, 136])
@pytest.mark.parametrize("n", [5, 60, 100, 126])
def test_nan_behind_the_end_of_the_reduction(cuda, direction, columns, tile, z, n):
    """Every other row of both operands is NaN: what is read past the end of a row of z % 64 values is the
    start of such a row, and NaN times the other operand's zeros would show."""
    E, rows = 3, n + 6
    offsets = torch.tensor([0, 2, n + 2, rows], dtype=torch.int32)
    assert kind(direction, rows, E, columns) == tile
    w, x = weights(direction, E, columns, z, 1), R.whole((rows, z), 2)
    exact = want(direction, x, w, offsets)
    x[1::2] = NAN
    if direction == "product":
        w[:, 1::2] = NAN
        exact[:, 1::2] = NAN
    exact[1::2] = NAN
    got = call(direction, x.to(cuda), w.to(cuda), offsets.to(cuda)).cpu().double()
    assert torch.equal(got.isnan(), exact.isnan())
    equal(got.nan_to_num(), exact.to(torch.bfloat16).double().nan_to_num())


@pytest.mark.parametrize("direction", ["product", "input"])
@pytest.mark.parametrize("columns,tile", [(5480, "narrow"), (10760, "wide")])
@pytest.mark.parametrize("n", [5, 70, 300])
def test_what_lies_behind_is_neither_read_nor_written(cuda, direction, columns, tile, n):
    E, z, used = 4, 72, n + 3
    rows = used + 40
    offsets = torch.tensor([0, n, n, used, used], dtype=torch.int32)
    assert kind(direction, rows, E, columns) == tile
    w, x = weights(direction, E, columns, z, 1), R.whole((rows, z), 2)
    exact = want(direction, x[:used], w, offsets)
    w[1], w[3], x[used:] = NAN, NAN, NAN  # experts without rows; rows of none
    out = torch.full((rows, columns), 7.0, dtype=torch.bfloat16, device=cuda)
    call(direction, x.to(cuda), w.to(cuda), offsets.to(cuda), out=out)
    equal(out[:used], exact)
    assert (out[used:] == 7).all()
    big = torch.full((2 * rows, z), NAN, dtype=torch.bfloat16)
    big[1::2] = x  # picked from a larger tensor, whose other rows are NaN
    index = (2 * torch.arange(rows, dtype=torch.int32) + 1).to(cuda)
    equal(call(direction, big.to(cuda), w.to(cuda), offsets.to(cuda), index=index)[:used], exact)


@pytest.mark.parametrize("index_of", ["none", "dy", "x", "both"])
@pytest.mark.parametrize("n", [1, 31, 33, 100])
def test_a_weight_gradient_reads_no_other_experts_rows(cuda, index_of, n):
    """The rows of the experts on either side are NaN: so are their gradients, and no others."""
    counts = [7, n, 40, n, 5]
    E, N, K, total = 5, 264, 136, sum(counts)
    offsets = torch.tensor([0] + counts, dtype=torch.int32).cumsum(0).to(torch.int32)
    dy, x = R.whole((total, N), 1), R.whole((total, K), 2)
    exact = R.by_weights(dy, x, offsets, None, None)[0]
    for e in (0, 2, 4):
        dy[offsets[e]:offsets[e + 1]], x[offsets[e]:offsets[e + 1]] = NAN, NAN
    order = torch.randperm(total, generator=torch.Generator().manual_seed(n))
    place = order.argsort().to(torch.int32).to(cuda)
    kwargs = {}
    if index_of in ("dy", "both"):
        dy, kwargs["dy_index"] = dy[order], place
    if index_of in ("x", "both"):
        x, kwargs["x_index"] = x[order], place
    for dtype in (torch.float32, torch.bfloat16):
        got = grouped.weight_gradient(dy.to(cuda), x.to(cuda), offsets.to(cuda), dtype=dtype, **kwargs)
        equal(got[1::2], exact[1::2])
        assert got[::2].isnan().all()


@pytest.mark.parametrize("direction", ["product", "input"])
@pytest.mark.parametrize("columns,tile", [(8200, "narrow"), (16400, "wide")])
@pytest.mark.parametrize("n", [6, 150, 400])
def test_indices_out_of_range(cuda, direction, columns, tile, n):
    E, z = 2, 72
    offsets = torch.tensor([0, n // 3, n], dtype=torch.int32)
    assert kind(direction, n, E, columns) == (tile if n < 300 else "wide")
    w, x = weights(direction, E, columns, z, 1), R.whole((9, z), 2)
    index = torch.arange(n, dtype=torch.int32) % 9
    index[::4], index[1], index[2] = 9, -1, 1 << 24
    to = torch.arange(n, dtype=torch.int32).flip(0)
    to[0], to[3] = n, -1
    out = torch.full((n, columns), 7.0, dtype=torch.bfloat16, device=cuda)
    call(direction, x.to(cuda), w.to(cuda), offsets.to(cuda), index=index.to(cuda), to=to.to(cuda), out=out)
    exact = torch.full((n, columns), 7.0, dtype=torch.float64)
    ok = (to >= 0) & (to < n)
    exact[to[ok].long()] = want(direction, x, w, offsets, index)[ok]
    equal(out, exact)


def cut(values, rows):
    """First and last rows of each expert by offsets that no plan makes: unsigned, and at most `rows`."""
    ends = [min(v % (1 << 32), rows) for v in values]
    return [(a, max(a, b)) for a, b in zip(ends, ends[1:])]


@pytest.mark.parametrize("values", [[0, 900, 5, 40], [0, 10, 1 << 30, 1 << 30], [-5, 3, 9, 12], [40, 40, 40, 40]])
@pytest.mark.parametrize("wide", [72, 5480, 10760])
def test_offsets_out_of_range(cuda, values, wide):
    """Outputs between guards; rows of one expert alone by the formula (where the experts have no more rows
    than there are, for which a launch has blocks), rows of none as they were."""
    E, narrow, rows = 3, 64, 40
    kinds = {72: ("few", "narrow"), 5480: ("narrow", "narrow"), 10760: ("wide", "wide")}[wide]
    assert kinds == (kind("product", rows, E, wide), kind("input", rows, E, wide))
    enough = sum(b - a for a, b in cut(values, rows)) <= rows
    owner = [[e for e, (a, b) in enumerate(cut(values, rows)) if a <= r < b] for r in range(rows)]
    o = ints(values, cuda)
    for direction in ("product", "input"):
        w, x = weights(direction, E, wide, narrow, 1), R.whole((rows, narrow), 2)
        room = torch.full((3 * rows, wide), 7.0, dtype=torch.bfloat16, device=cuda)
        call(direction, x.to(cuda), w.to(cuda), o, out=room[rows:2 * rows])
        got = room.cpu().double()
        assert (got[:rows] == 7).all() and (got[2 * rows:] == 7).all()
        for r in range(rows):
            if not owner[r]:
                assert (got[rows + r] == 7).all()
            elif enough:
                m = w[owner[r][0]].double()
                exact = m @ x[r].double() if direction == "product" else x[r].double() @ m
                assert torch.equal(got[rows + r], exact.to(torch.bfloat16).double())
    dy, x = R.whole((rows, wide), 3), R.whole((rows, narrow), 4)
    room = torch.full((3 * E, wide, narrow), 7.0, device=cuda)
    grouped.weight_gradient(dy.to(cuda), x.to(cuda), o, out=room[E:2 * E])
    assert (room[:E] == 7).all() and (room[2 * E:] == 7).all()
    for e, (a, b) in enumerate(cut(values, rows)):
        equal(room[E + e], dy[a:b].double().t() @ x[a:b].double())


@pytest.mark.parametrize("T,tile", [(300, "narrow"), (700, "wide")])
def test_the_same_bits_again_on_streams_and_in_graphs(cuda, T, tile):
    k, E, N, K = 2, 5, 400, 328
    assert kind("product", T * k, E, N) == tile == kind("input", T * k, E, K)
    made = []
    for seed in (1, 2):
        _, p, _ = laid_out(T, k, E, 1.0, seed, cuda)
        x, w, dy = (R.normal(s, seed + i).to(cuda) for i, s in enumerate([(T, K), (E, N, K), (T * k, N)]))

        def step(x=x, w=w, dy=dy, p=p):
            return grouped.product(x, w, p.offsets, index=p.token_index), grouped.input_gradient(dy, w, p.offsets)

        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        made.append((g, step, out, x))
    side = torch.cuda.Stream()
    for turn in range(3):
        for i, (_, _, _, x) in enumerate(made):
            x.copy_(R.normal((T, K), 50 + 2 * turn + i).to(cuda))
        eager = [[t.clone() for t in step()] for _, step, _, _ in made]
        torch.cuda.synchronize()
        for g, _, _, _ in made:
            g.replay()
        with torch.cuda.stream(side):
            again = made[0][1]()
        torch.cuda.synchronize()
        for (_, _, out, _), e in zip(made, eager):
            assert all(torch.equal(a, b) for a, b in zip(out, e))
        assert all(torch.equal(a, b) for a, b in zip(again, eager[0]))


@pytest.mark.parametrize("n,columns,tile", [(40, 5464, "narrow"), (130, 1824, "wide")])
def test_the_largest_tensor_that_an_index_picks_from(cuda, n, columns, tile):
    """65535 rows of 32768 values, just under 4 GiB: its last row, and the first that it has not."""
    rows, z = 65535, 32768
    assert kind("product", n, 1, columns) == tile
    big = torch.zeros((rows, z), dtype=torch.bfloat16, device=cuda)
    ends = R.whole((2, z), 1).to(cuda)
    big[0], big[-1] = ends[0], ends[1]
    index = ints(([65534, 65535, 0, -1] * n)[:n], cuda)
    w = torch.randint(-3, 4, (1, columns, z), device=cuda, dtype=torch.int8).to(torch.bfloat16)
    exact = torch.zeros((n, columns), dtype=torch.float64, device=cuda)
    exact[0::4], exact[2::4] = w[0].double() @ ends[1].double(), w[0].double() @ ends[0].double()
    equal(grouped.product(big, w, ints([0, n], cuda), index=index), exact.cpu())
