"""CPU: the 64-bit formulas that decay attention and the RMS norms are tested with, against the recurrence token by token
and its gradients by torch."""

import pytest
import torch
import decay_ref as D


def inputs(seed, B=2, T=9, H=4, Hk=2, Dk=3, Dv=5, head=False):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    gate = -rn(H).abs() if head else 0.4 - rn(B, T, H).abs()  # some above 0, which count as 0
    return rn(B, T, Hk, Dk), rn(B, T, Hk, Dk), rn(B, T, H, Dv), gate, rn(B, H, Dk, Dv)


def recurrence(q, k, v, g, scale, s0):
    H, per = v.shape[2], v.shape[2] // q.shape[2]
    q, k = (x.repeat_interleave(per, 2) for x in (q, k))
    g = g.expand(*v.shape[:-1]).clamp(max=0)
    h, outs = s0, []
    for t in range(q.shape[1]):
        h = torch.exp(g[:, t])[..., None, None] * h + k[:, t, :, :, None] * v[:, t, :, None, :]
        outs.append(scale * (q[:, t, :, :, None] * h).sum(-2))
    return torch.stack(outs, 1), h


@pytest.mark.parametrize("head", [False, True])
def test_closed_form_and_gradients(head):
    args = [x.requires_grad_() for x in inputs(1, head=head)]
    o, fin = recurrence(*args[:4], 0.7, args[4])
    do, dfin = torch.randn_like(o), torch.randn_like(fin)
    want = [o, fin, *torch.autograd.grad((o, fin), args, (do, dfin))]
    got = D.batch(*args[:4], 0.7, args[4], do, dfin)
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b.detach(), rtol=1e-12, atol=1e-12)
    for a, b in zip(D.batch(*args[:4], 0.7, args[4]), want):
        torch.testing.assert_close(a, b.detach(), rtol=1e-12, atol=1e-12)


def test_a_gate_of_minus_infinity_forgets():
    q, k, v, g, s0 = inputs(2)
    g[:, 4] = float("-inf")
    o, fin = D.batch(q, k, v, g, 1.0, s0)
    o2, fin2 = D.batch(q[:, 4:], k[:, 4:], v[:, 4:], g[:, 4:], 1.0)
    torch.testing.assert_close(o[:, 4:], o2)
    torch.testing.assert_close(fin, fin2)


def test_gradients_against_differences():
    args = inputs(3, B=1, T=5)
    g = torch.Generator().manual_seed(4)
    do, dfin = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((1, 5, 4, 5), (1, 4, 3, 5)))

    def loss(a):
        o, fin = D.batch(*a[:4], 0.5, a[4])
        return float((o * do).sum() + (fin * dfin).sum())

    grads = D.batch(*args[:4], 0.5, args[4], do, dfin)[2:]
    for i, grad in enumerate(grads):
        step = torch.randn(args[i].shape, generator=g, dtype=torch.float64)
        up, down = (list(args) for _ in range(2))
        up[i], down[i] = args[i] + 1e-6 * step, args[i] - 1e-6 * step
        diff = (loss(up) - loss(down)) / 2e-6
        assert abs(diff - float((grad * step).sum())) < 1e-6 * max(1.0, abs(diff))


@pytest.mark.parametrize("w", [None, 1])
def test_norm_gradients(w):
    g = torch.Generator().manual_seed(5)
    rn = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    h, dy, dh = rn(6, 7).requires_grad_(), rn(6, 7), rn(6, 7)
    w = None if w is None else rn(7).requires_grad_()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-3) * (1 if w is None else w)
    got = torch.autograd.grad((y, h), [h] if w is None else [h, w], (dy, dh))
    grad, dw, _, _ = D.rms_grads(h, w, 1e-3, dy, dh)
    torch.testing.assert_close(grad, got[0])
    if w is not None:
        torch.testing.assert_close(dw, got[1])
    z = rn(50).requires_grad_()
    f, df, _, _ = D.silu(z)
    torch.testing.assert_close(df.detach(), torch.autograd.grad(torch.nn.functional.silu(z).sum(), z)[0])
