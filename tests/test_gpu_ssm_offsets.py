"""GPU: the state space layer's operators where element offsets pass 31 and 32 bits (far batch rows, far rows of a
pool): the same bits as from tensors of their own."""

import pytest
import torch

from triune_amd import (layer_norm, short_conv, short_conv_decode_step, short_conv_varlen, ssm_decode_step, ssm_scan,
                        ssm_scan_varlen)

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
FAR = 4_400_000_000  # elements between two batch rows: past 32 bits, in bf16 8.8 GB


@pytest.fixture(scope="module")
def space(dev):
    buf = torch.empty(FAR + (1 << 20), device=dev, dtype=BF)
    yield buf
    del buf
    torch.cuda.empty_cache()


def far(space, x, offset):
    """x, its two batch rows FAR apart in `space`."""
    v = space.as_strided(x.shape, (FAR, *x[0].contiguous().stride()), offset)
    v.copy_(x)
    return v


def rn(dev, *shape, dtype=BF, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev)


def test_scan(dev, space):
    B, T, D, N = 2, 96, 128, 16
    u, delta, z, dy = (rn(dev, B, T, D, seed=s) for s in range(4))
    Bm, Cm = rn(dev, B, T, N, seed=5), rn(dev, B, T, N, seed=6)
    A = -torch.exp(rn(dev, D, N, dtype=torch.float32, seed=7))

    def run(u, delta, z, Bm, Cm, dy):
        leaves = [t.requires_grad_() for t in (u.detach(), delta.detach(), z.detach(), Bm.detach(), Cm.detach())]
        y, s = ssm_scan(leaves[0], leaves[1], A, leaves[3], leaves[4], z=leaves[2])
        return (y, s, *torch.autograd.grad(y, leaves, dy))

    want = run(u, delta, z, Bm, Cm, dy)
    step = 1 << 15
    got = run(*(far(space, t, i * step) for i, t in enumerate((u, delta, z, Bm, Cm, dy))))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    with torch.no_grad():
        out = space.as_strided((B, T, D), (FAR, D, 1), 8 * step)
        ssm_scan(u, delta, A, Bm, Cm, z=z, out=out)
        assert torch.equal(out, want[0])


def test_conv_and_norm(dev, space):
    x, dy = rn(dev, 2, 70, 256), rn(dev, 2, 70, 256, seed=1)
    w, b = rn(dev, 256, 4, seed=2).requires_grad_(), rn(dev, 256, seed=3).requires_grad_()

    def conv(x, dy):
        x = x.detach().requires_grad_()
        y, s = short_conv(x, w, b)
        return (y, s, *torch.autograd.grad(y, (x, w, b), dy))

    for a, c in zip(conv(far(space, x, 0), far(space, dy, 1 << 17)), conv(x, dy)):
        assert torch.equal(a, c)

    def norm(x, dy):
        x = x.detach().requires_grad_()
        y = layer_norm(x, b)
        return (y, *torch.autograd.grad(y, (x, b), dy))

    for a, c in zip(norm(far(space, x[:, 0], 0), far(space, dy[:, 0], 1 << 17)), norm(x[:, 0], dy[:, 0])):
        assert torch.equal(a, c)


def test_pools(dev):
    D, N, rows = 1536, 16, 90_000  # 2.2e9 states
    A = -torch.exp(rn(dev, D, N, dtype=torch.float32, seed=7))
    pool = torch.empty(rows, D, N, device=dev)
    slots = torch.tensor([rows - 1, 2], device=dev, dtype=torch.int32)
    s0 = rn(dev, 2, D, N, dtype=torch.float32, seed=1)
    cu = torch.tensor([0, 40, 70], device=dev, dtype=torch.int32)
    u, delta = rn(dev, 70, D), rn(dev, 70, D, seed=2)
    Bm, Cm = rn(dev, 70, N, seed=3), rn(dev, 70, N, seed=4)
    pool[slots.long()] = s0
    y, _ = ssm_scan_varlen(u, delta, A, Bm, Cm, cu, state_pool=pool, slots=slots)
    yw, s = ssm_scan_varlen(u, delta, A, Bm, Cm, cu, initial_state=s0)
    assert torch.equal(y, yw) and torch.equal(pool[slots.long()], s)
    y, _ = ssm_decode_step(u[:2], delta[:2], A, Bm[:2], Cm[:2], pool, inplace=True, slots=slots)
    yw, s = ssm_decode_step(u[:2], delta[:2], A, Bm[:2], Cm[:2], s)
    assert torch.equal(y, yw) and torch.equal(pool[slots.long()], s)
    del pool
    rows = 960_000  # 4.4e9 values
    pool = torch.empty(rows, 3, D, device=dev, dtype=BF)
    slots = torch.tensor([rows - 1, 2], device=dev, dtype=torch.int32)
    w, s0 = rn(dev, D, 4, seed=5), rn(dev, 2, 3, D, seed=6)
    pool[slots.long()] = s0
    y, _ = short_conv_varlen(u, w, cu, state_pool=pool, slots=slots)
    yw, s = short_conv_varlen(u, w, cu, initial_state=s0)
    assert torch.equal(y, yw) and torch.equal(pool[slots.long()], s)
    y, _ = short_conv_decode_step(u[:2], w, pool, inplace=True, slots=slots)
    yw, s = short_conv_decode_step(u[:2], w, s)
    assert torch.equal(y, yw) and torch.equal(pool[slots.long()], s)
    del pool
    torch.cuda.empty_cache()
