"""The experts' forward and backward of padded batches, of two layers at once, in graphs: tokens of no expert hold
NaN, which reaches nothing, and the others have the bits of the batch without them."""
import pytest
import torch

import _grouped as R
from moonshine_amd import experts
from moonshine_amd.synth import ACT_SITU, ACT_SWIGLU
from test_gpu_experts_training import problem

pytestmark = pytest.mark.gpu

NAN = float("nan")


@pytest.mark.parametrize("act", [ACT_SITU, ACT_SWIGLU])
@pytest.mark.parametrize("T,k,E,H,F", [(1, 2, 4, 64, 32), (90, 3, 6, 264, 136), (700, 4, 8, 512, 256)])
def test_padding_reaches_nothing(cuda, act, T, k, E, H, F):
    x, res, gu, down, ids, w, d = (t.to(cuda) for t in problem(T, k, E, H, F, T))
    out, saved = experts.forward(x, ids, w, gu, down, act, residual=res)
    want = experts.backward(d, saved, gu, down)
    live = torch.arange(T, device=cuda) * 2 + 1  # each token behind one of padding
    pad = lambda t, value: torch.full((2 * T + 3,) + t.shape[1:], value, dtype=t.dtype, device=cuda)  # noqa: E731
    xp, rp, ip, wp, dp = pad(x, NAN), pad(res, 3.0), pad(ids, -1), pad(w, NAN), pad(d, NAN)
    ip[::4] = E
    for to, t in ((xp, x), (rp, res), (ip, ids), (wp, w), (dp, d)):
        to[live] = t
    dead = torch.ones(2 * T + 3, dtype=torch.bool, device=cuda)
    dead[live] = False
    got, saved = experts.forward(xp, ip, wp, gu, down, act, residual=rp)
    # bits: an expert's rows are as many, in the same order, and both batches' products go by one kernel
    assert torch.equal(got[live], out) and (got[dead] == 3).all()
    dx, dw, dgu, ddown = experts.backward(dp, saved, gu, down)
    assert torch.equal(dx[live], want[0]) and not dx[dead].any()
    assert torch.equal(dw[live], want[1]) and not dw[dead].any()
    assert torch.equal(dgu, want[2]) and torch.equal(ddown, want[3])


def test_two_layers_at_once_and_replayed(cuda):
    """Forward and backward, added to f32 gradients, of two layers on two streams and in two graphs, with the
    program's own calls between the replays."""
    T, k, E, H, F = 150, 2, 6, 264, 136
    made = []
    for seed, act in ((1, ACT_SITU), (2, ACT_SWIGLU)):
        x, res, gu, down, ids, w, d = (t.to(cuda) for t in problem(T, k, E, H, F, seed))
        sums = torch.zeros(gu.shape, device=cuda), torch.zeros(down.shape, device=cuda)

        def step(x=x, res=res, gu=gu, down=down, ids=ids, w=w, d=d, act=act, sums=sums):
            out, saved = experts.forward(x, ids, w, gu, down, act, residual=res)
            return (out, *experts.backward(d, saved, gu, down, *sums)[:2])

        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held = step()
        made.append((g, step, held, sums, x))
    streams = [torch.cuda.Stream() for _ in made]
    for turn in range(3):
        want = []
        for i, (_, step, _, sums, x) in enumerate(made):
            x.copy_(R.normal((T, H), 90 + 2 * turn + i).to(cuda))
            for s in sums:
                s.zero_()
            outs = [t.clone() for t in step()]
            want.append((outs, [s.clone() for s in sums]))
        torch.cuda.synchronize()
        for g, _, _, _, _ in made:  # one after the other, and then at once by streams
            g.replay()
        torch.cuda.synchronize()
        for (_, _, held, sums, _), (outs, once) in zip(made, want):
            assert all(torch.equal(a, b) for a, b in zip(held, outs))
            assert all(torch.equal(a, 2 * b) for a, b in zip(sums, once))
        again = []
        for s, (_, step, _, _, _) in zip(streams, made):
            with torch.cuda.stream(s):
                again.append(step())
        torch.cuda.synchronize()
        for a, (outs, once), (_, _, _, sums, _) in zip(again, want, made):
            assert all(torch.equal(p, q) for p, q in zip(a, outs))
            assert all(torch.equal(p, 2 * q + q) for p, q in zip(sums, once))
