"""GPU: layer norm against its 64-bit definition, forward and backward, and refusals."""

import pytest
import torch
import ssm_ref as R

from triune_amd import layer_norm

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def inputs(dev, R_, D, dtype=F32, wdt=None, offset=0.5, seed=0):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    wdt = wdt or dtype
    return (rn(R_, D) + offset).to(dtype).to(dev), (1 + rn(D) / 4).to(wdt).to(dev), rn(D).to(wdt).to(dev)


def fwd_bound(x, w, b, eps):
    """The mean's error is at most 14 units of mean |x| (a tree over the lanes on 8 K <= 32 values in a
    row), the centred value's that and one rounding, the variance's 34 units and twice the mean's; rstd 4."""
    y, xh, r = R.norm(x, w, b, eps)
    x = R.d64(x)
    m = 50 * x.abs().mean(-1, keepdim=True) * r
    e = m + (24 + m / 2) * xh.abs() + m * xh.abs()
    if w is not None:
        e = e * R.d64(w).abs()
    return y, R.U * (e + 2 * y.abs() + (0 if b is None else R.d64(b).abs()))


SHAPES = [(1, 1), (3, 2), (5, 7), (1, 8), (4, 64), (7, 384), (9, 511), (2, 513), (3, 1001), (5, 1536), (2, 2048),
          (3, 2050), (2, 4096), (1, 5001), (2, 8192), (2, 8195), (1, 16384)]


@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("shape", SHAPES)
def test_norm(dev, shape, dtype):
    for wdt in (dtype, F32):
        x, w, b = inputs(dev, *shape, dtype, wdt)
        y, bound = fwd_bound(x, w, b, 1e-5)
        R.near(layer_norm(x, w, b), y, bound, dtype)
    for w_, b_ in ((None, None), (w, None), (None, b)):
        y, bound = fwd_bound(x, w_, b_, 1e-3)
        R.near(layer_norm(x, w_, b_, eps=1e-3), y, bound, dtype)


def test_rows_far_from_zero(dev):
    """A mean a thousand times the deviation: the variance is taken about the mean."""
    x, w, b = inputs(dev, 6, 700, offset=1000.0)
    y, bound = fwd_bound(x, w, b, 1e-5)
    R.near(layer_norm(x, w, b), y, bound)


def test_constant_rows_and_nan(dev):
    x, w, b = inputs(dev, 6, 70)
    x[1] = 3.0
    x[3, 5] = float("nan")
    x[4, 6] = float("inf")
    y = layer_norm(x, w, b)
    assert torch.equal(y[1], b) and bool(y[3].isnan().all()) and bool(y[4].isnan().any())
    assert bool(y[[0, 1, 2, 5]].isfinite().all())


def grad_tols(x, w, eps, dy):
    """dx: g and xh carry the forward's units (50 mean |x| r + 24 relative), each mean 20 more; dw, db: a
    column's sum takes at most a block's rows and parts."""
    _, xh, r = R.norm(x, None, None, eps)
    m = 50 * R.d64(x).abs().mean(-1, keepdim=True) * r
    g = R.d64(dy).abs() * (1 if w is None else R.d64(w).abs())
    e = m + (24 + 1.5 * m) * xh.abs()  # units of xh
    mg, mgx = g.mean(-1, keepdim=True), (g * xh.abs()).mean(-1, keepdim=True)
    dx = r * (30 * g + 30 * mg + xh.abs() * (60 * mgx + (g * e).mean(-1, keepdim=True)) + e * mgx)
    dx = dx + (m + 30) * r * (g + mg + xh.abs() * mgx)
    n = 40 + dy.shape[0] // 2
    ady = R.d64(dy).abs()
    return R.U * dx, R.U * (ady * (e + n * xh.abs())).sum(0), R.U * n * ady.sum(0)


@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("shape", SHAPES + [(300, 96), (1100, 40), (600, 2100)])
def test_gradients(dev, shape, dtype):
    for wdt in {dtype, F32}:
        x, w, b = inputs(dev, *shape, dtype, wdt)
        dy = torch.randn(shape, generator=torch.Generator().manual_seed(3)).to(dtype).to(dev)
        for t in (x, w, b):
            t.requires_grad_()
        got = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)
        for v, r, e, t in zip(got, R.norm_grads(x, w, b, 1e-5, dy), grad_tols(x, w, 1e-5, dy), (x, w, b)):
            assert v.dtype == t.dtype
            R.near(v, r, e, t.dtype)
    (dx,) = torch.autograd.grad(layer_norm(x), x, dy)
    R.near(dx, R.norm_grads(x, None, None, 1e-5, dy)[0], grad_tols(x, None, 1e-5, dy)[0], dtype)


def test_leading_dims_strides_and_partial_gradients(dev):
    x, w, b = inputs(dev, 60, 100, BF)
    dy = torch.randn(60, 100, device=dev).to(BF)
    wide = torch.zeros(5, 12, 210, device=dev, dtype=BF)
    wide[..., 3:103] = x.reshape(5, 12, 100)
    v = wide[..., 3:103]
    flat = layer_norm(x, w, b)
    assert torch.equal(layer_norm(v, w, b).reshape(60, 100), flat)
    t = x.reshape(5, 12, 100).transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(layer_norm(t, w, b).reshape(60, 100), flat)
    w.requires_grad_()
    ref = torch.autograd.grad(layer_norm(x, w, b), w, dy)[0]
    (dw,) = torch.autograd.grad(layer_norm(v, w, b), w, dy.reshape(5, 12, 100).transpose(0, 1).contiguous().transpose(0, 1))
    assert torch.equal(dw, ref)
    e = x[:1].expand(60, 100)  # one row for all
    assert torch.equal(layer_norm(e, w, b)[7], flat[0])
    assert torch.equal(layer_norm(x[0], w, b), flat[0])
    b.requires_grad_()
    (db,) = torch.autograd.grad(layer_norm(x, w, b).sum(), b)
    assert bool((db == 60).all())


def test_graph_replays_and_determinism(dev):
    x, w, b = inputs(dev, 300, 200, BF)
    dy = torch.randn(300, 200, device=dev).to(BF)
    for t in (x, w, b):
        t.requires_grad_()
    from triune_amd.norm import _LayerNorm, _forward

    y, mean, rstd = _forward(x.detach(), w.detach(), b.detach(), 1e-5, True)

    class Ctx:
        saved_tensors, bias_dtype, needs_input_grad = (x.detach(), w.detach(), mean, rstd), b.dtype, (True,) * 4

    call = lambda: _LayerNorm.backward.__wrapped__(Ctx, dy)[:3]  # noqa: E731
    eager = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)
    g = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(g):
        out = call()
        yg = layer_norm(x, w, b)
    for n in range(3):
        for t in (*out, yg):
            t.fill_(float("nan"))
        g.replay()
        again = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)
        torch.cuda.synchronize()
        assert torch.equal(yg, y) and all(torch.equal(p, q) for p, q in zip(out, eager))
        assert all(torch.equal(p, q) for p, q in zip(again, eager))


def test_empty_and_refusals(dev):
    x, w, b = inputs(dev, 4, 8)
    assert layer_norm(x[:0], w, b).shape == (0, 8)
    leaves = [t.clone().requires_grad_() for t in (x[:0], w, b)]
    for t, g in zip(leaves, torch.autograd.grad(layer_norm(*leaves).sum(), leaves)):
        assert g.shape == t.shape and bool((g == 0).all())
    for a in ((x, w[:4]), (x, w, b[:4]), (x[:, :0],), (torch.zeros(2, 16385, device=dev),)):
        with pytest.raises(ValueError):
            layer_norm(*a)
    with pytest.raises(TypeError):
        layer_norm(x.half(), w.bfloat16())
    with pytest.raises(TypeError):
        layer_norm(x.double())
    with pytest.raises(ValueError):
        layer_norm(x, w, b, eps=-1.0)
    with pytest.raises(ValueError):
        layer_norm(x, w.cpu())
