"""CPU: the 64-bit formulas that the state space layer's kernels are tested with, against differences
and against torch."""

import pytest
import torch
import ssm_ref as R


def _scan_inputs(seed, B=2, T=6, D=4, N=3, G=1, z=True):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    bc = (B, T, N) if G == 1 else (B, T, G, N)
    return [rn(B, T, D), rn(B, T, D), -torch.exp(rn(D, N)), rn(*bc), rn(*bc), rn(D), rn(B, T, D) if z else None, rn(D),
            rn(B, D, N)]


def _difference(f, args, k, v, step=1e-6):
    hi, lo = (list(args) for _ in range(2))
    hi[k], lo[k] = args[k] + step * v, args[k] - step * v
    return (f(*hi) - f(*lo)) / (2 * step)


@pytest.mark.parametrize("G", [1, 2])
@pytest.mark.parametrize("z", [True, False])
@pytest.mark.parametrize("soft", [True, False])
def test_scan_gradients_against_differences(G, z, soft):
    args = _scan_inputs(3, G=G, z=z)
    g = torch.Generator().manual_seed(4)
    dy, ds = (torch.randn(s, generator=g, dtype=torch.float64) for s in (args[0].shape, args[8].shape))

    def loss(u, delta, A, B, C, D, z_, bias, s0):
        y, s, *_ = R.scan(u, delta, A, B, C, D, z_, bias, soft, s0)
        return float((y * dy).sum() + (s * ds).sum())

    # a difference of two losses keeps their rounding (a few 2^-53 of the sum of their terms, which grow
    # without softplus, where dt < 0 makes decays of more than 1) over the step
    y, s, *_ = R.scan(*args[:8], soft, args[8])
    rounding = 2.0**-50 * float((y * dy).abs().sum() + (s * ds).abs().sum()) / 1e-6
    grads = R.scan_grads(*args[:8], soft, args[8], dy, ds)
    for k, grad in enumerate(grads):
        if args[k] is None:
            assert grad is None
            continue
        v = torch.randn(args[k].shape, generator=g, dtype=torch.float64)
        want = _difference(loss, args, k, v)
        assert abs(float((grad * v).sum()) - want) <= 1e-7 * (1 + abs(want)) + rounding, k


@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("T", [1, 2, 7])
@pytest.mark.parametrize("silu", [True, False])
def test_conv_gradients_against_differences(W, T, silu):
    g = torch.Generator().manual_seed(W * 10 + T)
    rn = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    args = [rn(2, T, 3), rn(3, W), rn(3), rn(2, W - 1, 3)]
    dy, ds = rn(2, T, 3), rn(2, W - 1, 3)

    def loss(x, w, b, s0):
        y, s, *_ = R.conv(x, w, b, s0, silu)
        return float((y * dy).sum() + (s * ds).sum())

    for k, grad in enumerate(R.conv_grads(*args, silu, dy, ds)):
        v = rn(*args[k].shape)
        want = _difference(loss, args, k, v)
        assert abs(float((grad * v).sum()) - want) <= 1e-7 * (1 + abs(want)), k


def test_norm_against_torch():
    g = torch.Generator().manual_seed(1)
    x, w, b, dy = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((5, 9), (9,), (9,), (5, 9)))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = torch.nn.functional.layer_norm(leaves[0], (9,), leaves[1], leaves[2], 1e-5)
    torch.testing.assert_close(R.norm(x, w, b, 1e-5)[0], y.detach(), rtol=1e-12, atol=1e-12)
    for got, want in zip(R.norm_grads(x, w, b, 1e-5, dy), torch.autograd.grad(y, leaves, dy)):
        torch.testing.assert_close(got, want, rtol=1e-11, atol=1e-12)
