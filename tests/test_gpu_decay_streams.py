"""GPU: decay attention's gradients and cut packed calls on two streams at once give the bits of calls alone: every region of
their workspaces is a call's own."""

import pytest
import torch

import triune_amd.decay as M
from triune_amd import decay_attn, decay_attn_varlen
from triune_amd._lib import plan_on

pytestmark = pytest.mark.gpu


def at_once(calls, repeats=4):
    """Each call's results, alone and `repeats` times beside the other on a stream of its own."""
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in calls], [[] for _ in calls]
    for _ in range(repeats):
        for c, s, r in zip(calls, streams, got):
            with torch.cuda.stream(s):
                r.append(c())
    torch.cuda.synchronize()
    for w, r in zip(want, got):
        for x in r:
            assert all(torch.equal(a, b) for a, b in zip(x, w))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients(dev, dtype):
    """Segments, shared heads and a constant gate: end states, states of every chunk, and both kinds of sums."""
    def call(seed):
        gen = torch.Generator().manual_seed(seed)
        rn = lambda *s: torch.randn(*s, generator=gen).to(dev)  # noqa: E731
        leaves = [x.requires_grad_() for x in (rn(1, 3000, 2, 64).to(dtype), rn(1, 3000, 2, 64).to(dtype),
                                               rn(1, 3000, 6, 48).to(dtype), -0.1 * rn(6).abs(), rn(1, 6, 64, 48))]
        do, dfin = rn(1, 3000, 6, 48).to(dtype), rn(1, 6, 64, 48)
        assert plan_on(leaves[0], "triune_hip_decay_attn_workspace_size", 1, 3000, 6, 2, 64, 48, 0) > 0

        def run():
            o, fin = decay_attn(*leaves[:4], initial_state=leaves[4], scale=0.125)
            return (o.detach(), fin.detach(), *torch.autograd.grad((o, fin), leaves, (do, dfin)))

        return run

    at_once([call(s) for s in range(2)])


@torch.no_grad()
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_packed_over_pools(dev, dtype):
    lens = [2000, 100, 3000, 1, 700]

    def call(seed):
        gen = torch.Generator().manual_seed(seed)
        rn = lambda *s: torch.randn(*s, generator=gen).to(dev)  # noqa: E731
        N = sum(lens)
        args = (rn(N, 2, 64).to(dtype), rn(N, 2, 64).to(dtype), rn(N, 4, 64).to(dtype), -0.01 * rn(N, 4).abs())
        cu = torch.tensor([0, *lens]).cumsum(0).to(torch.int32).to(dev)
        start, slots = rn(6, 4, 64, 64), torch.tensor([5, 0, 3, 1, 2], dtype=torch.int32, device=dev)
        assert plan_on(args[0], "triune_hip_decay_attn_varlen_workspace_size", 5, N, 4, 2, 64, 64, 0) > 0
        return lambda: decay_attn_varlen(*args, cu, scale=0.125, state_pool=start.clone(), slots=slots)

    at_once([call(s) for s in range(2)])


def test_two_calls_of_a_graph(dev):
    """Two calls of one graph share its memory pool, one behind the other; replays give the bits of eager calls."""
    gen = torch.Generator().manual_seed(0)
    rn = lambda *s: torch.randn(*s, generator=gen).to(dev)  # noqa: E731
    calls = [[*(rn(1, 1500, n, 64).to(torch.bfloat16) for n in (2, 2, 4, 4)), -0.1 * rn(1, 1500, 4).abs(), rn(1, 4, 64, 64)]
             for _ in range(2)]

    def one(q, k, v, do, g, s0):
        o, fin, kept = M._attn(q, k, v, g, 0.125, s0, None)
        assert kept is not None
        return (o, fin, *M._attn_bwd(q, k, v, g, 0.125, s0, do, fin, True, 0, kept))

    want = [one(*c) for c in calls]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [one(*c) for c in calls]
    for _ in range(4):
        for r in got:
            for x in r:
                x.fill_(float("nan"))
        graph.replay()
        one(*calls[0])  # eager work between the replays
        torch.cuda.synchronize()
        for w, r in zip(want, got):
            assert all(torch.equal(a, b) for a, b in zip(w, r))
