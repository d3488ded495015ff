"""GPU: the short causal convolution against its 64-bit definition: prompts, packed prompts, single
tokens, gradients, refusals."""

import pytest
import torch
import ssm_ref as R

from triune_amd import short_conv, short_conv_decode_step, short_conv_varlen

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def inputs(dev, B, T, D, W, dtype=F32, wdt=None, bias=True, s0=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    wdt = wdt or dtype
    return (rn(B, T, D).to(dtype).to(dev), rn(D, W).to(wdt).to(dev), rn(D).to(wdt).to(dev) if bias else None,
            rn(B, W - 1, D).to(dtype).to(dev) if s0 else None)


def check(got, x, w, b, s0, act, dtype):
    y, fin, bound, _ = R.conv(x, w, b, s0, act == "silu")
    R.near(got[0], y, bound, dtype)
    assert torch.equal(R.d64(got[1]), fin)


SHAPES = [(1, 1, 1), (2, 2, 7), (1, 3, 8), (2, 16, 9), (3, 17, 70), (1, 33, 130), (2, 100, 64), (1, 65, 520)]


@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("shape", SHAPES)
def test_conv(dev, shape, W, dtype):
    for bias, s0, act in ((True, True, "silu"), (False, False, None)):
        x, w, b, s = inputs(dev, *shape, W, dtype, bias=bias, s0=s0, seed=W)
        check(short_conv(x, w, b, s, act), x, w, b, s, act, dtype)


def test_fp32_weights_and_strides(dev):
    x, w, b, s = inputs(dev, 2, 50, 66, 4, BF, wdt=F32)
    wide = torch.zeros(50, 2, 140, device=dev, dtype=BF)
    wide[..., 3:69] = x.transpose(0, 1)
    buf = torch.full((2, 50, 70), 7.0, device=dev, dtype=BF)
    y, fin = short_conv(wide.transpose(0, 1)[..., 3:69], w.t().contiguous().t(), b, s, out=buf[..., 1:67])
    assert y.data_ptr() == buf[..., 1:67].data_ptr()
    check((y, fin), x, w, b, s, "silu", BF)
    assert bool((buf[..., :1] == 7).all()) and bool((buf[..., 67:] == 7).all())
    e = x[:1, :1].expand(2, 50, -1)
    check(short_conv(e, w, b, s), e, w, b, s, "silu", BF)


def test_values_outside_the_taps_do_not_matter(dev):
    """NaN in one row and channel reaches W tokens of that channel and nothing else; infinities stay."""
    x, w, b, s = inputs(dev, 2, 40, 70, 3)
    ref = short_conv(x, w, b, s, None)[0].clone()
    x[1, 15, 9] = float("nan")
    y = short_conv(x, w, b, s, None)[0]
    assert bool(y[1, 15:18, 9].isnan().all())
    y[1, 15:18, 9] = ref[1, 15:18, 9]
    assert torch.equal(y, ref)


def test_prompt_in_pieces(dev):
    x, w, b, s = inputs(dev, 2, 61, 24, 4, BF)
    whole = short_conv(x, w, b, s)
    st, ys = s, []
    for lo, hi in ((0, 1), (1, 3), (3, 40), (40, 60)):
        y, st = short_conv(x[:, lo:hi], w, b, st)
        ys.append(y)
    y, st = short_conv_decode_step(x[:, 60:], w, st, b, inplace=True)
    assert torch.equal(torch.cat([*ys, y], 1), whole[0]) and torch.equal(st, whole[1])


@pytest.mark.parametrize("W", [2, 4])
@pytest.mark.parametrize("lens", [[1], [5, 0, 33, 1, 2, 100], [0, 0], [300, 2], [1, 1, 1, 1, 1, 1, 1], [3] * 70])
def test_varlen(dev, lens, W):
    D, n, total = 70, len(lens), sum(lens) + 9
    x, w, b, _ = inputs(dev, 1, total, D, W, seed=n)
    s0 = torch.randn(n, W - 1, D, generator=torch.Generator().manual_seed(1)).to(dev)
    cu = torch.tensor([4] + lens).cumsum(0).to(torch.int32)
    out = torch.full((1, total, D), 7.0, device=dev)
    y, fin = short_conv_varlen(x, w, cu, b, s0, out=out)
    assert y.data_ptr() == out.data_ptr()
    assert bool((y[0, :4] == 7).all()) and bool((y[0, int(cu[-1]):] == 7).all())
    pool, slots = torch.randn(n + 2, W - 1, D, device=dev), torch.randperm(n + 2)[:n]
    pool[slots.to(dev)] = s0
    before = pool.clone()
    yp, p = short_conv_varlen(x[0], w, cu, b, state_pool=pool, slots=slots)
    assert p is pool and torch.equal(yp[4:int(cu[-1])], y[0, 4:int(cu[-1])])
    for i, ln in enumerate(lens):
        c = slice(int(cu[i]), int(cu[i]) + ln)
        check((y[:, c], fin[i:i + 1]), x[:, c], w, b, s0[i:i + 1], "silu", F32)
        assert torch.equal(pool[slots[i]], fin[i])
    for r in set(range(n + 2)) - set(slots.tolist()):
        assert torch.equal(pool[r], before[r])


def test_decode_slots(dev):
    x, w, b, _ = inputs(dev, 4, 1, 70, 4, BF)
    pool = torch.randn(6, 3, 70, device=dev).to(BF)
    before = pool.clone()
    slots = torch.tensor([5, -1, 0, 6], device=dev)
    y, p = short_conv_decode_step(x, w, pool, b, inplace=True, slots=slots)
    for i, sl in ((0, 5), (2, 0)):
        check((y[i:i + 1], p[sl:sl + 1]), x[i:i + 1], w, b, before[sl:sl + 1], "silu", BF)
    assert bool((y[1] == 0).all()) and bool((y[3] == 0).all()) and torch.equal(p[1:5], before[1:5])
    y2, p2 = short_conv_decode_step(x[:, 0], w, before, b, slots=slots)
    assert torch.equal(y2, y[:, 0]) and torch.equal(p2, p) and p2 is not before


@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("shape", SHAPES + [(2, 600, 33)])
def test_gradients(dev, shape, W, dtype):
    """Each gradient of x carries at most 2 W + 30 units of its terms (W products and the upstream
    through silu'), dw and dbias also their sums' (a run's 32 and at most 64 runs and parts)."""
    for bias, s0, act, wdt in ((True, True, "silu", None), (False, False, None, F32), (True, True, None, None)):
        x, w, b, s = inputs(dev, *shape, W, dtype, wdt=wdt, bias=bias, s0=s0, seed=W)
        g = torch.Generator().manual_seed(2)
        dy = torch.randn(x.shape, generator=g).to(dtype).to(dev)
        ds = torch.randn(shape[0], W - 1, shape[2], generator=g).to(dtype).to(dev)
        leaves = [t.requires_grad_() for t in (x, w, b, s) if t is not None]
        y, fin = short_conv(x, w, b, s, act)
        got = dict(zip(map(id, leaves), torch.autograd.grad((y, fin), leaves, (dy, ds))))
        form = (x, w, b, s, act == "silu", dy, ds)
        ref, env = R.conv_grads(*form), R.conv_grads(*form, absolute=True)
        # silu' = s (1 + p (1 - s)) may cancel: its units are of s (1 + |p|), and p carries W + 2 of
        # its own terms, so the scale of the roundings takes silu' at 2 with p's terms beside it
        _, _, pe, (_, p) = R.conv(x, w, b, s, act == "silu")
        if act == "silu":
            flat = (x, w, b, s, False, (dy.cpu().double() * (1 + p.abs() + pe / R.U)).to(torch.float64), ds)
            env = R.conv_grads(*flat, absolute=True)
        for t, r, e in zip((x, w, b, s), ref, env):
            if t is None:
                continue
            R.near(got[id(t)], r, (2 * W + 30 + (96 if t is w or t is b else 0)) * R.U * e, t.dtype)


def test_gradients_of_one_output_and_determinism(dev):
    x, w, b, s = inputs(dev, 2, 300, 70, 4)
    for t in (x, w, b, s):
        t.requires_grad_()
    y, fin = short_conv(x, w, b, s)
    a = torch.autograd.grad(y.sum(), (x, w, b, s), retain_graph=True)
    for p, q in zip(a, torch.autograd.grad(y.sum(), (x, w, b, s))):
        assert torch.equal(p, q)
    y, fin = short_conv(x, w, b, s)
    dx, ds = torch.autograd.grad(fin.sum(), (x, s))
    assert bool((dx[:, -3:] == 1).all()) and bool((dx[:, :-3] == 0).all()) and bool((ds == 0).all())


def test_graph_replays(dev):
    x, w, b, s = inputs(dev, 2, 100, 70, 4, BF)
    pool = s.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, fin = short_conv(x, w, b, s)
        ys, _ = short_conv_decode_step(x[:, 0], w, pool, b, inplace=True)
    eager = s.clone()
    pool.copy_(s)
    for n in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(n)))
        g.replay()
        e = short_conv(x, w, b, s)
        es, _ = short_conv_decode_step(x[:, 0], w, eager, b, inplace=True)
        torch.cuda.synchronize()
        assert torch.equal(y, e[0]) and torch.equal(fin, e[1]) and torch.equal(ys, es) and torch.equal(pool, eager)


def test_empty_and_refusals(dev):
    x, w, b, s = inputs(dev, 2, 5, 8, 4)
    y, fin = short_conv(x[:, :0], w, b, s)
    assert y.shape == (2, 0, 8) and torch.equal(fin, s)
    leaves = [t.clone().requires_grad_() for t in (x[:, :0], w, b, s)]
    y, fin = short_conv(*leaves)
    for t, g in zip(leaves, torch.autograd.grad((y.sum(), fin.sum()), leaves)):
        assert g.shape == t.shape and bool((g == (1 if t is leaves[3] else 0)).all())
    for a in ((x[0], w), (x, w[:4]), (x, w[:, :1]), (x, w, b[:4]), (x, w, b, s[:1]), (x, w, b, s, "gelu")):
        with pytest.raises(ValueError):
            short_conv(*a)
    with pytest.raises(TypeError):
        short_conv(x.half(), w.bfloat16())
    with pytest.raises(ValueError):
        short_conv(x, w, b.half())
    with pytest.raises(ValueError, match="gradient"):
        short_conv_decode_step(x[:, :1], w.clone().requires_grad_(), s)
    with pytest.raises(ValueError):
        short_conv_decode_step(x, w, s)
    with pytest.raises(ValueError):
        short_conv_decode_step(x[:, 0], w, s.half(), inplace=True)
    cu = torch.tensor([0, 5], device=dev, dtype=torch.int32)
    with pytest.raises(ValueError):
        short_conv_varlen(x, w, cu)
    with pytest.raises(ValueError):
        short_conv_varlen(x[:1], w, cu, state_pool=s)
    with pytest.raises(ValueError, match="gradient"):
        short_conv_varlen(x[:1], w.clone().requires_grad_(), cu)


def test_pools_that_want_gradients_are_refused(dev):
    x, w = torch.zeros(8, 6, device=dev), torch.zeros(6, 4, device=dev)
    cu, slots = torch.tensor([0, 8], dtype=torch.int32, device=dev), torch.tensor([0], dtype=torch.int32, device=dev)
    pool = torch.zeros(2, 3, 6, device=dev, requires_grad=True)
    with pytest.raises(ValueError):
        short_conv_varlen(x, w, cu, state_pool=pool, slots=slots)


def test_runs_of_large_calls(dev):
    """Calls that fill the chip take longer runs: the same bits as short pieces, dense and packed; dw and dbias
    against 64 bits (32 tokens of a run, four runs of a block, 65 blocks' parts: within the 96 of test_gradients)."""
    T, D, W = 8209, 2060, 4
    x, w, b, s = inputs(dev, 1, T, D, W, BF)
    cu = torch.tensor([0, 5, 5, 1003, 8209], dtype=torch.int32, device=dev)
    y, fin = short_conv(x, w, b, s)
    at, parts, state = 0, [], s
    while at < T:
        p, state = short_conv(x[:, at:at + 1021], w, b, state)
        parts.append(p)
        at += 1021
    assert torch.equal(torch.cat(parts, 1), y) and torch.equal(state, fin)
    yp, fp = short_conv_varlen(x[0], w, cu, b)
    for i, (lo, hi) in enumerate(zip(cu.tolist(), cu.tolist()[1:])):
        e = short_conv(x[:, lo:hi], w, b)
        assert torch.equal(yp[lo:hi], e[0][0]) and torch.equal(fp[i], e[1][0])
    dy = torch.randn(1, T, D, generator=torch.Generator().manual_seed(2)).to(BF).to(dev)
    ds = torch.zeros_like(s)
    leaves = [t.requires_grad_() for t in (x, w, b, s)]
    got = torch.autograd.grad(short_conv(*leaves, activation=None), leaves, (dy, ds))
    form = (x, w, b, s, False, dy, ds)
    for t, g, r, e in zip(leaves, got, R.conv_grads(*form), R.conv_grads(*form, absolute=True)):
        R.near(g, r, (2 * W + 30 + (96 if t is w or t is b else 0)) * R.U * e, BF)
