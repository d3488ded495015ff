"""GPU: the RMS norms against their 64-bit definitions, forward and backward, and refusals."""

import pytest
import torch
import decay_ref as D

from triune_amd import add_rms_norm, gated_rms_norm, rms_norm

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-5
SHAPES = [(1, 1), (3, 2), (5, 7), (40, 8), (9, 63), (100, 64), (33, 120), (17, 128), (9, 256), (7, 384), (9, 511), (2, 513),
          (3, 1001), (5, 1536), (2, 2048), (3, 2050), (2, 4096), (1, 5001), (2, 8192), (2, 8195), (1, 16384)]


def rn(dev, *shape, dtype=F32, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev)


def near_norm(y, h, w, dtype, what=""):
    r, _, _ = D.rms(h, w, EPS)
    D.near(y, r, D.U * (D.XH + 4) * r.abs(), dtype, what)


def near_sum(h, x, r, s, what=""):
    t = D.d64(x) * (D.d64(s) if torch.is_tensor(s) else s)
    D.near(h, D.d64(r) + t, D.U * 2 * (D.d64(r) + t).abs(), r.dtype, what)


@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("shape", SHAPES)
def test_rms_and_add(dev, shape, dtype):
    x, w = rn(dev, *shape, dtype=dtype), (1 + rn(dev, shape[1], seed=1) / 4).to(dtype)
    for weight in (w, w.float(), None):
        near_norm(rms_norm(x, weight, EPS), x, weight, dtype)
    s = rn(dev, shape[1], seed=2).to(dtype)
    for rdt in {dtype, F32}:
        r = rn(dev, *shape, dtype=rdt, seed=3) * 2
        for scale, value in ((None, 1.0), (0.37, 0.37), (s, s), (s.float(), s)):
            y, h = add_rms_norm(x, r, w, scale, EPS)
            assert h.dtype == rdt and y.dtype == dtype
            # a number is taken in float32: half a unit more
            t = D.d64(x) * (D.d64(value) if torch.is_tensor(value) else value)
            D.near(h, D.d64(r) + t, D.U * (2 * (D.d64(r) + t).abs() + t.abs()), rdt, "h")
            near_norm(y, h, w, dtype, "y")
            if rdt == dtype:
                assert torch.equal(rms_norm(h, w, EPS), y)


@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("shape", SHAPES)
def test_gated(dev, shape, dtype):
    x, z, w = rn(dev, *shape, dtype=dtype), rn(dev, *shape, dtype=dtype, seed=1) * 3, rn(dev, shape[1], seed=2)
    for weight in (w.to(dtype), w, None):
        y = gated_rms_norm(x, z, weight, EPS)
        f, _, e, _ = D.silu(D.d64(z))
        r, _, _ = D.rms(x, weight, EPS)
        D.near(y, r * f, D.U * ((D.XH + 5) * (r * f).abs() + r.abs() * e), dtype)


@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("shape", SHAPES + [(3000, 64), (700, 513)])
def test_add_gradients(dev, shape, dtype):
    x, w, s = rn(dev, *shape, dtype=dtype), rn(dev, shape[1], seed=1), rn(dev, shape[1], seed=2)
    dy = rn(dev, *shape, dtype=dtype, seed=4)
    for rdt, wdt, scale in ((dtype, dtype, s.to(dtype)), (F32, F32, s), (dtype, F32, 0.5), (F32, dtype, None)):
        r, dh = rn(dev, *shape, dtype=rdt, seed=3), rn(dev, *shape, dtype=rdt, seed=5)
        leaves = [t.detach().requires_grad_() for t in (x, r, w.to(wdt), *([scale] if torch.is_tensor(scale) else []))]
        y, h = add_rms_norm(*leaves[:3], leaves[3] if len(leaves) > 3 else scale, EPS)
        got = torch.autograd.grad((y, h), leaves, (dy, dh))
        g, dw, bg, bw = D.rms_grads(h, leaves[2], EPS, dy, dh)
        f = D.d64(scale) if torch.is_tensor(scale) else 1.0 if scale is None else scale
        D.near(got[1], g, bg, rdt, "dr")
        D.near(got[0], g * f, (bg + D.U * g.abs()) * abs(f), dtype, "dx")
        D.near(got[2], dw, bw, wdt, "dw")
        if len(leaves) > 3:
            n = 60 + shape[0] / 2
            ds = (g * D.d64(x)).sum(0)
            D.near(got[3], ds, (bg * D.d64(x).abs()).sum(0) + D.U * n * (g * D.d64(x)).abs().sum(0), scale.dtype, "ds")
    leaves = [t.detach().requires_grad_() for t in (x, w)]
    got = torch.autograd.grad(rms_norm(*leaves, EPS), leaves, dy)
    g, dw, bg, bw = D.rms_grads(x, w, EPS, dy)
    D.near(got[0], g, bg, dtype, "dx of rms_norm")
    D.near(got[1], dw, bw, F32, "dw of rms_norm")


@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("shape", SHAPES + [(3000, 64), (700, 513)])
def test_gated_gradients(dev, shape, dtype):
    x, z, w = rn(dev, *shape, dtype=dtype), rn(dev, *shape, dtype=dtype, seed=1) * 2, rn(dev, shape[1], seed=2)
    dy = rn(dev, *shape, dtype=dtype, seed=4)
    for weight in (w.to(dtype), w):
        leaves = [t.detach().requires_grad_() for t in (x, z, weight)]
        got = torch.autograd.grad(gated_rms_norm(*leaves, EPS), leaves, dy)
        f, df, ef, edf = D.silu(D.d64(z))
        _, xh, r = D.rms(x, None, EPS)
        wd, dyd = D.d64(weight), D.d64(dy)
        g, _, bg, _ = D.rms_grads(x, None, EPS, dyd * wd * f)
        # the gate's own error moves d, and with it the mean
        ed = dyd.abs() * wd.abs() * ef
        bg = bg + D.U * r * (ed + xh.abs() * (ed * xh.abs()).mean(-1, keepdim=True))
        D.near(got[0], g, bg, dtype, "dx")
        t = dyd * xh * wd
        D.near(got[1], t * df, D.U * ((D.XH + 6) * (t * df).abs() + t.abs() * edf), dtype, "dz")
        n = D.XH + 60 + shape[0] / 2
        t = dyd * xh
        D.near(got[2], (t * f).sum(0), D.U * (n * (t * f).abs() + t.abs() * ef).sum(0), weight.dtype, "dw")


@pytest.mark.parametrize("dtype", [F32, BF])
def test_layouts(dev, dtype):
    """Heads as views of a projection, sliced tokens, transposed and broadcast rows, unaligned starts: the bits of
    contiguous copies."""
    B, T, H, d = 3, 11, 4, 40
    proj = rn(dev, B, T, 2 * H * d + 7, dtype=dtype)
    x = proj[..., 3:3 + H * d].unflatten(-1, (H, d))
    views = [x, proj[:, 2:9, :H * d].unflatten(-1, (H, d)), x.transpose(1, 2), x[:, ::3], x[:1].expand(3, -1, -1, -1),
             x[:, :, :1].expand(-1, -1, 4, -1), x[..., ::2], x[0], x[0, 0], x[0, 0, 0], x[:, 5]]
    for i, v in enumerate(views):
        z = rn(dev, *v.shape, 2, dtype=dtype, seed=1)[..., 0]
        w = rn(dev, v.shape[-1], 2, seed=2)[:, 0]
        outs = []
        for copy in (False, True):
            a, b, c = (t.detach().clone(memory_format=torch.contiguous_format) if copy else t.detach() for t in (v, z, w))
            a, b, c = (t.requires_grad_() for t in (a, b, c))
            up = rn(dev, *v.shape, 3, dtype=dtype, seed=3)[..., 1]
            up = up.contiguous() if copy else up
            y = gated_rms_norm(a, b, c)
            y2, h = add_rms_norm(a, b, c, c)
            outs.append((y, y2, h, rms_norm(a, c), *torch.autograd.grad((y, y2, h), (a, b, c), (up, up, up))))
        for a, b in zip(*outs):
            assert torch.equal(a, b), i
        assert all(t.is_contiguous() for t in outs[0][:4])


def test_one_output_alone_and_unused_inputs(dev):
    x, r, w, s = rn(dev, 9, 100), rn(dev, 9, 100, seed=1), rn(dev, 100, seed=2), rn(dev, 100, seed=3)
    up = rn(dev, 9, 100, seed=4)
    zero = torch.zeros_like(up)
    for pick in (0, 1):
        leaves = [t.detach().requires_grad_() for t in (x, r, w, s)]
        both = add_rms_norm(*leaves, EPS)
        got = torch.autograd.grad(both[pick], leaves, up, allow_unused=True, retain_graph=True)
        want = torch.autograd.grad(both, leaves, (zero, up) if pick else (up, zero))
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    for k in range(4):  # a gradient of one input alone: the same bits
        leaves = [t.detach() for t in (x, r, w, s)]
        leaves[k].requires_grad_()
        got, = torch.autograd.grad(add_rms_norm(*leaves, EPS), leaves[k], (up, up))
        full = [t.detach().requires_grad_() for t in (x, r, w, s)]
        assert torch.equal(got, torch.autograd.grad(add_rms_norm(*full, EPS), full, (up, up))[k])


def test_rows_at_the_edges(dev):
    """Zero rows, rows with a NaN or an infinity, large and small ones: each row by itself."""
    x = rn(dev, 8, 72)
    x[1], x[2, 5], x[3, 6], x[4], x[5] = 0, float("nan"), float("inf"), x[4] * 1e18, x[5] * 1e-18
    z = rn(dev, 8, 72, seed=1)
    for y in (rms_norm(x), gated_rms_norm(x, z)):
        assert bool((y[1] == 0).all()) and bool(y[2].isnan().all()) and bool(y[3, 6].isnan())
        assert bool(y[[0, 4, 5, 6, 7]].isfinite().all())
    near_norm(rms_norm(x, None, EPS)[[0, 4, 5, 6, 7]], x[[0, 4, 5, 6, 7]], None, F32)
    z[0] = torch.tensor([-300.0, 300.0, -88.0, 0.0], device=dev).repeat(18)
    y = gated_rms_norm(x[:1], z[:1], None, EPS)
    r, _, _ = D.rms(x[:1], None, EPS)
    f, _, e, _ = D.silu(D.d64(z[:1]))
    D.near(y, r * f, D.U * ((D.XH + 5) * (r * f).abs() + r.abs() * e) + 1e-35, F32)


def test_empty_rows(dev):
    x, w = torch.zeros(0, 4, 16, device=dev, requires_grad=True), torch.ones(16, device=dev, requires_grad=True)
    for y in (rms_norm(x, w), gated_rms_norm(x, x, w), add_rms_norm(x, x, w, w)[0]):
        assert y.shape == x.shape
        dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
        assert dx.shape == x.shape and not dw.any()


def test_refusals(dev):
    x, w = torch.zeros(4, 16, device=dev), torch.ones(16, device=dev)
    bad = [
        (ValueError, "rows of 1", lambda: rms_norm(torch.zeros(2, 16385, device=dev))),
        (ValueError, "rows of 1", lambda: rms_norm(torch.zeros(2, 0, device=dev))),
        (ValueError, "weight must be", lambda: rms_norm(x, w[:8])),
        (TypeError, "weight must have", lambda: rms_norm(x, w.half())),
        (TypeError, "dtype", lambda: rms_norm(x.double())),
        (ValueError, "eps", lambda: rms_norm(x, eps=-1.0)),
        (ValueError, "eps", lambda: rms_norm(x, eps=float("nan"))),
        (ValueError, "CPU|device", lambda: rms_norm(x, w.cpu())),
        (ValueError, "residual must", lambda: add_rms_norm(x, x[:2])),
        (TypeError, "residual must", lambda: add_rms_norm(x, x.half())),
        (ValueError, "scale must be", lambda: add_rms_norm(x, x, scale=w[:8])),
        (TypeError, "scale must have", lambda: add_rms_norm(x, x, scale=w.half())),
        (ValueError, "z must", lambda: gated_rms_norm(x, x[:2])),
        (ValueError, "z must", lambda: gated_rms_norm(x, x.half())),
    ]
    for kind, match, call in bad:
        with pytest.raises(kind, match=match):
            call()
    fw = torch.autograd.forward_ad
    with fw.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        gated_rms_norm(x, fw.make_dual(x, x))
