"""64-bit CPU definitions of decay attention and the RMS norms, their gradients, and the bounds that their roundings
allow, for the tests of the kernels.  U is 2^-24, half the spacing of float32 in [1/2, 1).

Decay attention is taken in its closed form: with D_ij = e^{G_i - G_j} (j <= i), G the sums of g,
    o = scale ((q k^T . D) v + d0 q S_0),   S_T = aT S_0 + (k dT)^T v
and every output and gradient is a sum of products of inputs with one of the decays D_ij, d0_i = e^{G_i},
dT_j = e^{G_T - G_j}, aT = e^{G_T}.  The same sums over absolute values, with every decay times the roundings on its
way, bound the error.  Units of U, of the product with a decay over m tokens whose gates sum to G:
    exponents  g log2(e) is off by two roundings of |g| log2(e), and the constant; sums of the parts below 2^-8 and their
               difference by under one: 3 |G| + 3 m with the factors of the chunks and segments (exp2: 2, products: 1)
    sums       a state takes at most three products of parts for each token, each added with a rounding (or a cut, two
               halves) of the sum of absolute values so far: 4 m
    ends       sums over the head dims, the chunk and the slices, and the parts of derived operands in bf16, which leave
               2^-17 of the value (128 units) at two uses: Dk + Dv + 80 + 260
    underflow  a decay below 2^-126, the smallest normal number, may count as 0, and so may each part of a weighted value
               and of a score below it (at most 6): 8 times 2^-126 of the product without its decay
"""

import torch
from ssm_ref import U, d64, half_step, near  # noqa: F401


def _gate(g, H, T):
    g = torch.where(g > 0, torch.zeros_like(g), torch.clamp(g, min=-1e4))
    return g.expand(T, H) if g.dim() == 1 else g


def _decays(g, units):
    """(D, d0, dT, aT) of one head, g [T]; with `units`, each times its roundings."""
    T = g.shape[0]
    G = g.cumsum(0)
    n = torch.arange(1, T + 1, dtype=torch.float64)

    def times(x, m):
        return torch.exp(x) if units is None else torch.exp(x) * (units + 3 * x.abs() + 7 * m) + 2.0**-123 / U

    D = times((G[:, None] - G[None, :]).tril(), (n[:, None] - n[None, :]).tril()).tril()
    return D, times(G, n), times(G[-1] - G, T - n), times(G[-1], n[-1])


def attn(q, k, v, g, scale, s0=None, do=None, dfin=None, bound=None):
    """One sequence: q, k [T, Hk, Dk], v [T, H, Dv], g [T, H] or [H], s0 [H, Dk, Dv] or None.  Returns (o, final state) or
    with do and dfin (o, final, dq, dk, dv, dg, ds0); bound: the sums over absolute values in these units (1 + those of
    the ends)."""
    q, k, v, g, s0, do, dfin = (d64(t) for t in (q, k, v, g, s0, do, dfin))
    T, Hk, Dk = q.shape
    H, Dv = v.shape[1:]
    per = H // Hk
    if s0 is None:
        s0 = torch.zeros(H, Dk, Dv, dtype=torch.float64)
    raw, g = g, _gate(g, H, T)
    if bound is not None:
        q, k, v, s0, scale = q.abs(), k.abs(), v.abs(), s0.abs(), abs(scale)
        do, dfin = (None if t is None else t.abs() for t in (do, dfin))
    outs = []
    for h in range(H):
        qh, kh, vh, sh = q[:, h // per], k[:, h // per], v[:, h], s0[h]
        D, d0, dT, aT = _decays(g[:, h], bound)
        qk = qh @ kh.T
        o = scale * ((qk * D) @ vh + d0[:, None] * (qh @ sh))
        fin = aT * sh + (kh * dT[:, None]).T @ vh
        if do is None:
            outs.append((o, fin))
            continue
        doh, dfh = do[:, h], dfin[h]
        B = scale * (doh @ vh.T) * D
        dq = B @ kh + scale * d0[:, None] * (doh @ sh.T)
        dk = B.T @ qh + dT[:, None] * (vh @ dfh.T)
        dv = scale * (qk * D).T @ doh + dT[:, None] * (kh @ dfh)
        ds0 = aT * dfh + scale * (qh * d0[:, None]).T @ doh
        # pairs that span t: written before it, read at it or behind
        M = torch.zeros(T + 2, T + 2, dtype=torch.float64)  # row T + 1: the final state; column 0: the initial one
        M[1:T + 1, 1:T + 1] = qk * B
        M[1:T + 1, 0] = (qh * (scale * d0[:, None] * (doh @ sh.T))).sum(-1)
        M[T + 1, 1:T + 1] = (kh * (dT[:, None] * (vh @ dfh.T))).sum(-1)
        M[T + 1, 0] = aT * (sh * dfh).sum()
        before = M.cumsum(1)
        dg = torch.stack([before[t:, t - 1].sum() for t in range(1, T + 1)])
        outs.append((o, fin, dq, dk, dv, dg, ds0))
    o, fin = torch.stack([x[0] for x in outs], 1), torch.stack([x[1] for x in outs])
    if do is None:
        return o, fin
    dq, dk, dv = (torch.stack([x[i] for x in outs], 1) for i in (2, 3, 4))
    dg, ds0 = torch.stack([x[5] for x in outs], 1), torch.stack([x[6] for x in outs])
    dq, dk = (x.unflatten(1, (Hk, per)).sum(2) for x in (dq, dk))
    if raw.dim() == 1:
        dg = dg.sum(0)
    return o, fin, dq, dk, dv, torch.where(raw > 0, torch.zeros_like(dg), dg), ds0


def ends(Dk, Dv, T=0, shared=False):
    """Units of the ends; a constant gate's gradient is a sum over T tokens of a batch in parts of at most 64."""
    return Dk + Dv + 340 + T / 16 + (64 if shared else 0)


def batch(q, k, v, g, scale, s0=None, do=None, dfin=None, bound=None):
    """attn over [B, T, ...]."""
    at = lambda t, b: None if t is None else t[b]  # noqa: E731
    got = [attn(q[b], k[b], v[b], g if g.dim() == 1 else g[b], scale, at(s0, b), at(do, b), at(dfin, b), bound)
           for b in range(q.shape[0])]
    out = [torch.stack(x) for x in zip(*got)]
    if do is not None and g.dim() == 1:
        out[5] = out[5].sum(0)
    return out


# ---- norms ---------------------------------------------------------------------------------------------------
def rms(x, w, eps):
    """(y, xh, rstd)."""
    x, w = d64(x), d64(w)
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return (x * r if w is None else x * r * w), x * r, r


# The mean square is a sum of positive terms: at most 2 K <= 64 in a row in a thread and ten levels of a tree, half of
# whose roundings reach rstd, then a division, a root and a reciprocal
XH = 45


def rms_grads(h, w, eps, dy, dh=None):
    """(g, dw, bound of g, bound of dw) of y = rms(h): g the gradient of h."""
    _, xh, r = rms(h, None, eps)
    dy, w, dh = d64(dy), d64(w), d64(dh)
    d = dy if w is None else dy * w
    m = (d * xh).mean(-1, keepdim=True)
    g = r * (d - xh * m)
    ma = (d * xh).abs().mean(-1, keepdim=True)
    b = r * ((XH + 6) * d.abs() + (3 * XH + 90) * xh.abs() * ma)
    if dh is not None:
        g, b = g + dh, b + 2 * dh.abs()
    lead = tuple(range(dy.dim() - 1))
    n = XH + 60 + dy[..., 0].numel() / 2  # rows of a block and parts in a row
    return g, (dy * xh).sum(lead), U * (b + 2 * g.abs()), U * n * (dy * xh).abs().sum(lead)


def silu(z):
    """(silu, silu', units of each against their terms' absolute values): exp2's argument is rounded, so the sigmoid's
    error grows with |z|."""
    s = torch.sigmoid(z)
    return z * s, s * (1 + z * (1 - s)), (8 + 2 * z.abs()) * (z * s).abs(), (14 + 4 * z.abs()) * s * (1 + z.abs() * (1 - s))
