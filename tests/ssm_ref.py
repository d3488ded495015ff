"""64-bit CPU definitions of the state space layer's operators and their gradients, each with the bound
that its roundings allow (in units of u = 2^-24), for the tests of the kernels.

The scan's forward bound is a running error analysis: a decay exp(dt A) carries at most
11 |dt A| + 4 units (dt: 8 from softplus, two products' roundings and A log2(e)'s in the exponent;
exp2: 2; the fma: 1), a term dt u B at most 12.  Gradients are bounded by the same formulas on
absolute values times the number of roundings on the longest chain.
"""

import torch

U = 2.0**-24


def softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def d64(t):
    return None if t is None else t.detach().cpu().double()


def per_channel(x, D):
    """[.., N] or [.., G, N] (with a leading [B, T]) as [B, T, D, N]."""
    if x.dim() == 3:
        return x.unsqueeze(2).expand(-1, -1, D, -1)
    return x.repeat_interleave(D // x.shape[2], 2)


def scan(u, delta, A, B, C, D=None, z=None, bias=None, soft=True, s0=None):
    """(y, final state, bound of y, bound of the state, parts for the gradients), 64-bit CPU."""
    u, delta, A, B, C, D, z, bias, s0 = (d64(t) for t in (u, delta, A, B, C, D, z, bias, s0))
    Bn, T, Dm = u.shape
    N = A.shape[1]
    x = delta if bias is None else delta + bias
    dt = softplus(x) if soft else x
    Bc, Cc = per_channel(B, Dm), per_channel(C, Dm)
    h = torch.zeros(Bn, Dm, N, dtype=torch.float64) if s0 is None else s0.clone()
    M, P = h.abs(), torch.zeros_like(h)
    hs, as_, ys, es = [h], [], [], []
    for t in range(T):
        la = dt[:, t, :, None] * A
        a = torch.exp(la)
        xin = (dt[:, t] * u[:, t])[..., None] * Bc[:, t]
        P = a * (P + (11 * la.abs() + 4) * M) + 12 * xin.abs()
        M = a * M + xin.abs()
        h = a * h + xin
        hs.append(h)
        as_.append(a)
        ys.append((Cc[:, t] * h).sum(-1))
        es.append((Cc[:, t].abs() * (P + (N + 2) * M)).sum(-1))
    y, e = (torch.stack(v, 1) if T else torch.zeros(Bn, 0, Dm, dtype=torch.float64) for v in (ys, es))
    if D is not None:
        y = y + D * u
        e = e + 2 * (D * u).abs()
    raw = y
    if z is not None:
        g = z * torch.sigmoid(z)
        y = y * g
        e = (e + (8 + 2 * z.abs()) * raw.abs()) * g.abs()
    return y, h, U * e, U * (P + M), (dt, x, hs, as_, raw)


def scan_grads(u, delta, A, B, C, D, z, bias, soft, s0, dy, dfin, absolute=False):
    """Gradients in the order of ssm_scan's autograd, by the formulas; absolute: every term's absolute
    value instead (the scale of the roundings)."""
    _, _, _, _, (dt, x, hs, as_, raw) = scan(u, delta, A, B, C, D, z, bias, soft, s0)
    u, delta, A, B, C, D, z, bias, s0, dy, dfin = (d64(t) for t in (u, delta, A, B, C, D, z, bias, s0, dy, dfin))
    Bn, T, Dm = u.shape
    N = A.shape[1]
    Bc, Cc = per_channel(B, Dm), per_channel(C, Dm)
    f = (lambda t: t.abs()) if absolute else (lambda t: t)
    if absolute:
        h, hs = (torch.zeros(Bn, Dm, N, dtype=torch.float64) if s0 is None else s0.abs()), []
        hs.append(h)
        for t in range(T):
            h = as_[t] * h + ((dt[:, t] * u[:, t])[..., None] * Bc[:, t]).abs()
            hs.append(h)
        raw = torch.stack([(Cc[:, t].abs() * hs[t + 1]).sum(-1) for t in range(T)], 1)
        raw = raw if D is None else raw + (D * u).abs()
    gy, dz = f(dy), None
    if z is not None:
        s = torch.sigmoid(z)
        # silu' = s (1 + z (1 - s)) cancels near z = -1.28: its roundings (and z (1 - s)'s, 4 units) are of
        # s (1 + |z| (1 - s)), so in the absolute form both terms count
        dz = f(dy) * raw * s * (1 + f(z) * (1 - s))
        gy = f(dy) * f(z * s)
    E = torch.zeros(Bn, Dm, N, dtype=torch.float64) if dfin is None else f(dfin).clone()
    dA = torch.zeros_like(A)
    dB4, dC4 = (torch.zeros(Bn, T, Dm, N, dtype=torch.float64) for _ in range(2))
    du, ddt = torch.zeros_like(u), torch.zeros_like(u)
    for t in range(T - 1, -1, -1):
        dh = f(Cc[:, t]) * gy[:, t, :, None] + E
        dC4[:, t] = gy[:, t, :, None] * hs[t + 1]
        dB4[:, t] = dh * f(dt[:, t] * u[:, t])[..., None]
        E = dh * as_[t]
        p = E * hs[t]
        b = (dh * f(Bc[:, t])).sum(-1)
        ddt[:, t] = (p * f(A)).sum(-1) + b * f(u[:, t])
        du[:, t] = b * f(dt[:, t]) + (0 if D is None else f(D) * gy[:, t])
        dA += (p * f(dt[:, t])[..., None]).sum(0)
    dd = ddt * torch.sigmoid(x) if soft else ddt

    def grp(v):
        return v.sum(2) if B.dim() == 3 else v.unflatten(2, (B.shape[2], -1)).sum(3)

    return (du, dd, dA, grp(dB4), grp(dC4), None if D is None else (gy * f(u)).sum((0, 1)), dz,
            None if bias is None else dd.sum((0, 1)), None if s0 is None else E)


def conv(x, w, bias=None, s0=None, silu=True):
    """(y, final state, bound of y, parts): W products, a bias, and silu's 8 + 2 |p| units."""
    x, w, bias, s0 = (d64(t) for t in (x, w, bias, s0))
    Bn, T, Dm = x.shape
    W = w.shape[1]
    prev = torch.zeros(Bn, W - 1, Dm, dtype=torch.float64) if s0 is None else s0
    full = torch.cat((prev, x), 1)
    b = torch.zeros(Dm, dtype=torch.float64) if bias is None else bias
    p = b.expand(Bn, T, Dm)
    e = b.abs().expand(Bn, T, Dm)
    for j in range(W):
        p = p + full[:, j:j + T] * w[:, j]
        e = e + (full[:, j:j + T] * w[:, j]).abs()
    e = (W + 1) * e
    fin = full[:, T:]
    if not silu:
        return p, fin, U * e, (full, p)
    s = torch.sigmoid(p)
    return p * s, fin, U * (1.1 * e + (8 + 2 * p.abs()) * (p * s).abs()), (full, p)


def conv_grads(x, w, bias, s0, silu, dy, dfin, absolute=False):
    _, _, _, (full, p) = conv(x, w, bias, s0, silu)
    w, dy, dfin = d64(w), d64(dy), d64(dfin)
    f = (lambda t: t.abs()) if absolute else (lambda t: t)
    T, W = p.shape[1], w.shape[1]
    dp = f(dy)
    if silu:
        s = torch.sigmoid(p)
        dp = dp * f(s * (1 + p * (1 - s)))
    dfull = torch.zeros_like(full)
    if dfin is not None:
        dfull[:, T:] += f(dfin)
    dw = torch.zeros_like(w)
    for j in range(W):
        dfull[:, j:j + T] += dp * f(w[:, j])
        dw[:, j] = (dp * f(full[:, j:j + T])).sum((0, 1))
    return dfull[:, W - 1:], dw, None if bias is None else dp.sum((0, 1)), None if s0 is None else dfull[:, :W - 1]


def norm(x, w, b, eps):
    """(y, xh, rstd), 64-bit."""
    x, w, b = (d64(t) for t in (x, w, b))
    c = x - x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    xh = c * r
    y = xh if w is None else xh * w
    return (y if b is None else y + b), xh, r


def norm_grads(x, w, b, eps, dy):
    _, xh, r = norm(x, w, b, eps)
    dy, w = d64(dy), d64(w)
    g = dy if w is None else dy * w
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    lead = tuple(range(dy.dim() - 1))
    return dx, (dy * xh).sum(lead), dy.sum(lead)


def half_step(t, dtype):
    """The error of rounding t once to dtype (fp32: within the bounds' units); below the smallest
    normal number the spacing stays that number's."""
    if dtype == torch.float32:
        return U * t.abs()
    fi = torch.finfo(dtype)
    return fi.eps / 2 * t.abs().clamp_min(fi.tiny)


def near(got, ref, bound, dtype=torch.float32, what=""):
    """got within bound of ref, plus one rounding to dtype (of a value that the bound may move)."""
    got = d64(got)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    tol = bound + half_step(ref.abs() + bound, dtype) + 1e-37
    bad = ~((got - ref).abs() <= tol)
    if bool(bad.any()):
        i = int(torch.argmax(torch.where(bad, (got - ref).abs() / tol, torch.zeros_like(tol)).nan_to_num(nan=1e30)))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, worst at {i}: {got.flatten()[i]} for "
                             f"{ref.flatten()[i]}, allowed {tol.flatten()[i]}")
