"""CPU: the bound of a few terms in test_gpu_decay_bits.py is passed by operands of 16 bits, which two bf16 parts hold."""

import decay_ref as D
import pytest
import torch
from ssm_ref import U


def cut(x):
    """The sum of two bf16 parts."""
    hi = x.float().to(torch.bfloat16).float()
    return (hi + (x.float() - hi).to(torch.bfloat16).float()).to(x.dtype)


@pytest.mark.parametrize("T,Dk,Dv", [(1, 1, 1), (2, 1, 2), (3, 2, 1)])
def test_two_parts_pass_the_bound(T, Dk, Dv):
    gen = torch.Generator().manual_seed(0)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    q, k, v, do = rn(T, 64, Dk), rn(T, 64, Dk), rn(T, 64, Dv), rn(T, 64, Dv)
    g, s0, dfin = -0.2 * rn(T, 64).abs(), rn(64, Dk, Dv), rn(64, Dk, Dv)
    ref = D.attn(q, k, v, g, 0.3, s0, do, dfin)
    bound = D.attn(q, k, v, g, 0.3, s0, do, dfin, bound=2 * (Dk + Dv + T) + 16)
    bad = D.attn(q, cut(k), cut(v), g, 0.3, cut(s0), cut(do), cut(dfin))
    for name, a, r, b in zip("o final dq dk dv dg ds0".split(), bad, ref, bound):
        assert bool(((a - r).abs() > U * (b + r.abs())).any()), name
