"""GPU: the gradients of decay attention stay inside a workspace of exactly the size that they ask for, with and without
what the forward left, which they do not write."""

import pytest
import torch

import triune_amd.decay as M
from triune_amd._lib import plan_on

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("head", [False, True])
def test_bounds_of_the_scratch(dev, monkeypatch, dtype, head):
    gen = torch.Generator().manual_seed(0)
    rn = lambda *s: torch.randn(*s, generator=gen).to(dev)  # noqa: E731
    B, T, H, Hk, Dk, Dv = 2, 700, 4, 2, 48, 80
    q, k, v, do = (rn(B, T, n, d).to(dtype) for n, d in ((Hk, Dk), (Hk, Dk), (H, Dv), (H, Dv)))
    g, s0, dfin = -(rn(H) if head else rn(B, T, H)).abs(), rn(B, H, Dk, Dv), rn(B, H, Dk, Dv)
    _, _, kept = M._attn(q, k, v, g, 0.2, s0, None)
    before = kept.clone()
    spaces = []

    def space(*shape, dtype=None, device=None):  # workspaces are the tensors of bytes
        if dtype is not torch.uint8:
            return torch.empty(*shape, dtype=dtype, device=device)
        wide = torch.full((shape[0] + 4096,), 0xA5, dtype=dtype, device=device)
        spaces.append((wide, shape[0]))
        return wide[:shape[0]]

    class Torch:
        empty = staticmethod(space)

        def __getattr__(self, name):
            return getattr(torch, name)

    monkeypatch.setattr(M, "torch", Torch())
    full = M._attn_bwd(q, k, v, g, 0.2, s0, do, dfin, True)
    less = M._attn_bwd(q, k, v, g, 0.2, s0, do, dfin, True, 0, kept)
    assert all(torch.equal(a, b) for a, b in zip(full, less)) and torch.equal(kept, before)
    (_, m), (_, n) = spaces
    assert m - n == kept.numel() == plan_on(q, "triune_hip_decay_attn_workspace_size", B, T, H, Hk, Dk, Dv, 0) > 0
    assert all(bool((wide[used:] == 0xA5).all()) for wide, used in spaces)
