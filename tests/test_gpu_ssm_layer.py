"""GPU: the state space layer's operators together, as a model runs them: norm, projection, short
convolution, projections of its output, scan, projection.  Trained against a 64-bit layer on the CPU,
prefilled packed over pools and decoded token by token against the whole prompts, and the decode
step captured in a graph."""

import pytest
import torch
import torch.nn.functional as F
import ssm_ref as R

from triune_amd import (layer_norm, short_conv, short_conv_decode_step, short_conv_varlen, ssm_decode_step, ssm_scan,
                        ssm_scan_varlen)

pytestmark = pytest.mark.gpu

WIDTH, INNER, N, W, RANK = 48, 72, 16, 4, 8


def parameters(seed=0):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return {"norm_w": 1 + rn(WIDTH) / 8, "norm_b": rn(WIDTH) / 8, "in": rn(2 * INNER, WIDTH) / WIDTH**0.5,
            "conv_w": rn(INNER, W) / 2, "conv_b": rn(INNER) / 8, "x": rn(RANK + 2 * N, INNER) / INNER**0.5,
            "dt": rn(INNER, RANK) / RANK**0.5, "dt_b": rn(INNER) - 3, "A_log": rn(INNER, N) / 2,
            "D": 1 + rn(INNER) / 8, "out": rn(WIDTH, INNER) / INNER**0.5}


def project(p, x):
    """x and gate halves; delta, B, C of the convolution's output."""
    xz = F.linear(x, p["in"])
    return xz[..., :INNER], xz[..., INNER:]


def scan_operands(p, u):
    dbc = F.linear(u, p["x"])
    return F.linear(dbc[..., :RANK], p["dt"]), dbc[..., RANK:RANK + N], dbc[..., RANK + N:]


def layer(p, x):
    u, z = project(p, layer_norm(x, p["norm_w"], p["norm_b"]))
    u, cs = short_conv(u, p["conv_w"], p["conv_b"])
    delta, B, C = scan_operands(p, u)
    y, hs = ssm_scan(u, delta, -torch.exp(p["A_log"]), B, C, D=p["D"], z=z, delta_bias=p["dt_b"])
    return x + F.linear(y, p["out"]), cs, hs


def layer64(p, x):
    """The same from the definitions, in 64 bits."""
    m = x.mean(-1, keepdim=True)
    v = ((x - m) ** 2).mean(-1, keepdim=True)
    u, z = project(p, (x - m) / torch.sqrt(v + 1e-5) * p["norm_w"] + p["norm_b"])
    T = x.shape[1]
    full = F.pad(u, (0, 0, W - 1, 0))
    c = p["conv_b"] + sum(full[:, j:j + T] * p["conv_w"][:, j] for j in range(W))
    u = c * torch.sigmoid(c)
    delta, B, C = scan_operands(p, u)
    dt, A = R.softplus(delta + p["dt_b"]), -torch.exp(p["A_log"])
    h, ys = torch.zeros(x.shape[0], INNER, N, dtype=x.dtype), []
    for t in range(T):
        h = torch.exp(dt[:, t, :, None] * A) * h + (dt[:, t] * u[:, t])[..., None] * B[:, t, None]
        ys.append((h * C[:, t, None]).sum(-1))
    y = (torch.stack(ys, 1) + p["D"] * u) * z * torch.sigmoid(z)
    return x + F.linear(y, p["out"]), full[:, T:], h


def close(got, ref, units, what):
    """Relative 2-norm: `units` roundings of 2^-24 at most in a row, on sums of terms of random signs,
    whose norm is at least a quarter of their absolute values'."""
    got = R.d64(got)
    assert float((got - ref).norm()) <= 4 * units * R.U * float(ref.norm()), what


def test_training_step_against_64_bits(dev):
    """Two layers, forward and every gradient.  Roundings in a row: the scans' 24 (T + 16) each way, the
    products' sums of at most 2 INNER terms, the norms' and convolutions' under 100."""
    B, T = 2, 45
    ps = [parameters(1), parameters(2)]
    x = torch.randn(B, T, WIDTH, generator=torch.Generator().manual_seed(3))
    dy = torch.randn(B, T, WIDTH, generator=torch.Generator().manual_seed(4))
    dev_ps = [{k: v.to(dev).requires_grad_() for k, v in p.items()} for p in ps]
    ref_ps = [{k: v.double().requires_grad_() for k, v in p.items()} for p in ps]
    xd, xr = x.to(dev).requires_grad_(), x.double().requires_grad_()
    yd, yr = xd, xr
    for a, b in zip(dev_ps, ref_ps):
        yd, yr = layer(a, yd)[0], layer64(b, yr)[0]
    units = 2 * (2 * 24 * (T + 16) + 8 * 2 * INNER + 200)
    close(yd, yr.detach(), units, "y")
    keys = list(ps[0])
    gd = torch.autograd.grad(yd, [xd, *(p[k] for p in dev_ps for k in keys)], dy.to(dev))
    gr = torch.autograd.grad(yr, [xr, *(p[k] for p in ref_ps for k in keys)], dy.double())
    for name, a, b in zip(["x", *(f"{i}.{k}" for i in (0, 1) for k in keys)], gd, gr):
        close(a, b, units, name)


@torch.no_grad()
def test_packed_prefill_and_decode_against_whole_prompts(dev):
    """Ragged prompts prefilled in one packed call into slots of pools, then three tokens each."""
    p = {k: v.to(dev) for k, v in parameters(5).items()}
    lens, extra = [7, 40, 1, 18], 3
    A, n = -torch.exp(p["A_log"]), len(lens)
    whole = [torch.randn(1, ln + extra, WIDTH, generator=torch.Generator().manual_seed(i)).to(dev)
             for i, ln in enumerate(lens)]
    pool_c, pool_h = torch.zeros(6, W - 1, INNER, device=dev), torch.zeros(6, INNER, N, device=dev)
    slots = torch.tensor([5, 0, 3, 2], device=dev, dtype=torch.int32)
    cu = torch.tensor([0, *lens]).cumsum(0).to(torch.int32).to(dev)
    x = torch.cat([w[0, :ln] for w, ln in zip(whole, lens)])
    u, z = project(p, layer_norm(x, p["norm_w"], p["norm_b"]))
    u, _ = short_conv_varlen(u, p["conv_w"], cu, p["conv_b"], state_pool=pool_c, slots=slots)
    delta, B, C = scan_operands(p, u)
    y, _ = ssm_scan_varlen(u, delta, A, B, C, cu, D=p["D"], z=z, delta_bias=p["dt_b"], state_pool=pool_h, slots=slots)
    outs = [[o] for o in (x + F.linear(y, p["out"])).split(lens)]
    for t in range(extra):
        x = torch.cat([w[:, ln + t] for w, ln in zip(whole, lens)])
        u, z = project(p, layer_norm(x, p["norm_w"], p["norm_b"]))
        u, _ = short_conv_decode_step(u, p["conv_w"], pool_c, p["conv_b"], inplace=True, slots=slots)
        delta, B, C = scan_operands(p, u)
        y, _ = ssm_decode_step(u, delta, A, B, C, pool_h, D=p["D"], z=z, delta_bias=p["dt_b"], inplace=True, slots=slots)
        for o, row in zip(outs, x + F.linear(y, p["out"])):
            o.append(row[None])
    ref_p = {k: v.cpu().double() for k, v in p.items()}
    for i, w in enumerate(whole):
        ref, cs, hs = layer64(ref_p, w.cpu().double())
        units = 24 * (w.shape[1] + 16) + 8 * 2 * INNER + 200
        close(torch.cat(outs[i]), ref[0], units, f"sequence {i}")
        close(pool_c[slots[i]], cs[0], units, f"convolution state {i}")
        close(pool_h[slots[i]], hs[0], units, f"scan state {i}")
    assert bool((pool_h[[1, 4]] == 0).all()) and bool((pool_c[[1, 4]] == 0).all())


@torch.no_grad()
def test_captured_decode_step(dev):
    """The layer's step for four sessions in a graph, replayed with new tokens and eager work between, against eager
    steps on other pools."""
    p = {k: v.to(dev) for k, v in parameters(6).items()}
    A = -torch.exp(p["A_log"])
    slots = torch.tensor([4, 1, 0, 3], device=dev, dtype=torch.int32)
    pools = [(torch.zeros(5, W - 1, INNER, device=dev), torch.zeros(5, INNER, N, device=dev)) for _ in range(2)]

    def step(x, pc, ph):
        u, z = project(p, layer_norm(x, p["norm_w"], p["norm_b"]))
        u, _ = short_conv_decode_step(u, p["conv_w"], pc, p["conv_b"], inplace=True, slots=slots)
        delta, B, C = scan_operands(p, u)
        y, _ = ssm_decode_step(u, delta, A, B, C, ph, D=p["D"], z=z, delta_bias=p["dt_b"], inplace=True, slots=slots)
        return x + F.linear(y, p["out"])

    x = torch.randn(4, WIDTH, device=dev)
    side = torch.cuda.Stream(device=dev)  # the projections' library picks its kernels before the capture
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step(x, *(t.clone() for t in pools[0]))
    torch.cuda.current_stream(dev).wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(x, *pools[0])
    for t in pools[0]:
        t.zero_()
    for k in range(4):
        x.copy_(torch.randn(4, WIDTH, generator=torch.Generator().manual_seed(k)))
        g.replay()
        eager = step(x, *pools[1])
        torch.cuda.synchronize()
        torch.testing.assert_close(out, eager, rtol=0, atol=0)
        assert all(torch.equal(a, b) for a, b in zip(*pools))
