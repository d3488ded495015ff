"""GPU: decay attention over so many sequences and heads that the states add up to more than 2^31 values, and gradients of
shared heads over more values than one grid of their sum takes: the same bits as with fewer sequences at a time."""

import pytest
import torch
import decay_ref as R

import triune_amd.decay as M
from triune_amd import decay_attn, decay_attn_varlen

pytestmark = pytest.mark.gpu

B, H, D, T = 2050, 64, 128, 3  # 2050 x 64 states of 128 x 128: 2.15e9 values, 8.6 GB


@pytest.fixture(scope="module")
def many(dev):
    gen = torch.Generator(device=dev).manual_seed(0)
    rn = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    x = [rn(B, T, n, D).to(torch.bfloat16) for n in (2, 2, H)]
    assert B * H * D * D > 1 << 31
    yield (*x, -rn(B, T, H).abs(), rn(B, H, D, D))
    torch.cuda.empty_cache()


@torch.no_grad()
def test_packed_over_a_pool(dev, many):
    *x, s0 = many
    flat = [t.flatten(0, 1) for t in x]
    pool, slots = s0.clone(), torch.arange(B, dtype=torch.int32, device=dev).flip(0)
    cu = torch.arange(B + 1, dtype=torch.int32, device=dev) * T
    o, _ = decay_attn_varlen(*flat, cu, state_pool=pool, slots=slots)
    half = B // 2
    for a, b in ((0, half), (half, B)):
        rows = slots[a:b].long()
        want, s = decay_attn_varlen(*(t[a * T:b * T] for t in flat), cu[:b - a + 1], s0[rows])
        assert torch.equal(o[a * T:b * T], want) and torch.equal(pool[rows], s)


def test_dense_with_gradients(dev, many):
    *x, s0 = many
    do = torch.randn(B, T, H, D, generator=torch.Generator(device=dev).manual_seed(1), device=dev).to(torch.bfloat16)
    dfin = s0.flip(0)

    def call(a, b):
        leaves = [t[a:b].detach().requires_grad_() for t in (*x, s0)]
        o, fin = decay_attn(*leaves[:4], initial_state=leaves[4])
        return (o.detach(), fin.detach(), *torch.autograd.grad((o, fin), leaves, (do[a:b], dfin[a:b])))

    got = call(0, B)
    half = B // 2
    for a, b in ((0, half), (half, B)):
        for y, z in zip(got, call(a, b)):
            assert torch.equal(y[a:b], z)


@torch.no_grad()
def test_packed_sequences_past_the_grid_of_a_join(dev):
    """70000 sequences of 64 heads, one of them long enough to be cut among fewer."""
    gen = torch.Generator(device=dev).manual_seed(3)
    rn = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    n, long = 70000, 700
    q, k, v, g = rn(n + long, 1, 65), rn(n + long, 1, 65), rn(n + long, 64, 1), -rn(n + long, 64).abs()
    s0 = rn(n, 64, 65, 1)
    cu = torch.arange(n + 1, device=dev, dtype=torch.int32)
    cu[n // 2 + 1:] += long
    o, fin = decay_attn_varlen(q, k, v, g, cu, s0)
    for a, b in ((0, 30000), (30000, n // 2), (n // 2 + 1, n)):
        t0, t1 = int(cu[a]), int(cu[b])
        want, s = decay_attn_varlen(*(t[t0:t1] for t in (q, k, v, g)), cu[a:b + 1] - cu[a], s0[a:b])
        assert torch.equal(o[t0:t1], want) and torch.equal(fin[a:b], s)
    a = n // 2
    part = [t[a:a + long + 1] for t in (q, k, v, g)]
    want, bound = (R.attn(*part, 1.0, s0[a], bound=e) for e in (None, R.ends(65, 1)))
    R.near(o[a:a + long + 1], want[0], R.U * bound[0], torch.float32, "o")
    R.near(fin[a], want[1], R.U * bound[1], torch.float32, "final")


def test_gradients_of_many_shared_values(dev):
    """3 x 44000 tokens of one head of 128 key dims: 16.9 million values, past the 2^24 threads of the sum over heads."""
    gen = torch.Generator(device=dev).manual_seed(2)
    rn = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    q, k, v, do = (rn(3, 44000, n, d).to(torch.bfloat16) for n, d in ((1, D), (1, D), (2, 8), (2, 8)))
    g = -rn(3, 44000, 2).abs()
    flags = 200 << 8  # the same segments for any batch
    got = M._attn_bwd(q, k, v, g, 1.0, None, do, None, True, flags)
    for b in range(3):
        want = M._attn_bwd(*(t[b:b + 1] for t in (q, k, v, g)), 1.0, None, do[b:b + 1], None, True, flags)
        for y, z in zip(got, want):
            assert torch.equal(y[b:b + 1], z)
