"""GPU: the decay attention layer's operators where element offsets pass 31 and 32 bits (far batch rows, far tokens, far rows
of a pool): the same bits as from tensors of their own."""

import pytest
import torch

from triune_amd import add_rms_norm, decay_attn, decay_attn_decode_step, decay_attn_varlen, gated_rms_norm, rms_norm

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
FAR = 4_400_000_000  # elements between two batch rows: past 32 bits, in bf16 8.8 GB
PLACE = 1 << 16  # elements between the tensors that share the space


@pytest.fixture(scope="module")
def space(dev):
    buf = torch.empty(FAR + (1 << 21), device=dev, dtype=BF)
    yield buf
    del buf
    torch.cuda.empty_cache()


def far(space, x, i):
    """x, its two batch rows FAR apart in `space`, at the i-th place."""
    assert x[0].numel() <= PLACE and x.shape[0] == 2
    v = space.as_strided(x.shape, (FAR, *x[0].contiguous().stride()), i * PLACE)
    v.copy_(x)
    return v


def apart(space, x, i):
    """x [T, ...], its tokens an equal distance apart over all of `space`, from the i-th place."""
    step = FAR // (x.shape[0] - 1) // 8 * 8
    v = space.as_strided(x.shape, (step, *x[0].contiguous().stride()), i * PLACE)
    v.copy_(x)
    return v


def rn(dev, *shape, dtype=BF, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev)


def attention(q, k, v, g, do):
    leaves = [t.detach().requires_grad_() for t in (q, k, v, g)]
    o, s = decay_attn(*leaves)
    return (o, s, *torch.autograd.grad(o, leaves, do))


def test_far_batch_rows(dev, space):
    x = (rn(dev, 2, 200, 2, 64), rn(dev, 2, 200, 2, 64, seed=1), rn(dev, 2, 200, 4, 64, seed=2),
         -rn(dev, 2, 200, 4, seed=3).abs(), rn(dev, 2, 200, 4, 64, seed=4))
    want = attention(*x)
    for a, b in zip(attention(*(far(space, t, i) for i, t in enumerate(x))), want):
        assert torch.equal(a, b)
    with torch.no_grad():
        out = space.as_strided(x[2].shape, (FAR, 256, 64, 1), 8 * PLACE)
        decay_attn(*x[:4], out=out)
        assert torch.equal(out, want[0])


def test_far_tokens(dev, space):
    """33 tokens of 137 million elements each: strides that no buffer resource spans."""
    x = (rn(dev, 33, 2, 64), rn(dev, 33, 2, 64, seed=1), rn(dev, 33, 2, 64, seed=2), -rn(dev, 33, 2, seed=3).abs(),
         rn(dev, 33, 2, 64, seed=4))
    wide = [apart(space, t, i) for i, t in enumerate(x)]
    # far rows are loaded element by element, with the products in the same order
    for a, b in zip(attention(*(t[None] for t in wide)), attention(*(t[None] for t in x))):
        assert torch.equal(a, b)
    with torch.no_grad():
        cu = torch.tensor([0, 32, 33], device=dev, dtype=torch.int32)
        for a, b in zip(decay_attn_varlen(*wide[:4], cu), decay_attn_varlen(*x[:4], cu)):
            assert torch.equal(a, b)
        s0 = rn(dev, 33, 2, 64, 64, dtype=F32)
        for a, b in zip(decay_attn_decode_step(*wide[:4], s0), decay_attn_decode_step(*x[:4], s0)):
            assert torch.equal(a, b)


@torch.no_grad()
def test_far_pool_rows(dev):
    rows = 540_000  # of 2 x 64 x 64: 4.4e9 states
    pool = torch.empty(rows, 2, 64, 64, device=dev)
    slots = torch.tensor([rows - 1, 2], device=dev, dtype=torch.int32)
    s0 = rn(dev, 2, 2, 64, 64, dtype=F32, seed=1)
    cu = torch.tensor([0, 340, 400], device=dev, dtype=torch.int32)
    q, k, v, g = rn(dev, 400, 2, 64), rn(dev, 400, 2, 64, seed=2), rn(dev, 400, 2, 64, seed=3), -rn(dev, 400, 2, seed=4).abs()
    pool[slots.long()] = s0
    o, _ = decay_attn_varlen(q, k, v, g, cu, state_pool=pool, slots=slots)
    want, s = decay_attn_varlen(q, k, v, g, cu, initial_state=s0)
    assert torch.equal(o, want) and torch.equal(pool[slots.long()], s)
    x = [t[:2] for t in (q, k, v, g)]
    o, _ = decay_attn_decode_step(*x, pool, inplace=True, slots=slots)
    want, s = decay_attn_decode_step(*x, s)
    assert torch.equal(o, want) and torch.equal(pool[slots.long()], s)
    del pool
    torch.cuda.empty_cache()


def test_norms(dev, space):
    x, r, dy, dh = (rn(dev, 2, 70, 256, seed=s) for s in range(4))
    w, s = rn(dev, 256, seed=5).requires_grad_(), rn(dev, 256, seed=6).requires_grad_()

    def add(x, r, dy, dh):
        x, r = (t.detach().requires_grad_() for t in (x, r))
        y, h = add_rms_norm(x, r, w, s)
        return (y, h, *torch.autograd.grad((y, h), (x, r, w, s), (dy, dh)))

    def plain(x, r, dy, dh):
        x = x.detach().requires_grad_()
        y = rms_norm(x, w)
        return (y, *torch.autograd.grad(y, (x, w), dy))

    def gated(x, r, dy, dh):
        x, r = (t.detach().requires_grad_() for t in (x, r))
        y = gated_rms_norm(x, r, w)
        return (y, *torch.autograd.grad(y, (x, r, w), dy))

    wide = [far(space, t, i) for i, t in enumerate((x, r, dy, dh))]
    for f in (add, plain, gated):
        for a, b in zip(f(*wide), f(x, r, dy, dh)):
            assert torch.equal(a, b), f.__name__
