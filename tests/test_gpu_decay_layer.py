"""GPU: the decay attention layer's operators together, as a model runs them: residual sum and norm, projections, decay
attention, gated norm of each head, projection.  Trained against a 64-bit layer on the CPU, prefilled packed over a
pool and decoded token by token against the whole prompts, and steps captured in graphs."""

import pytest
import torch
import torch.nn.functional as F
import decay_ref as D

from triune_amd import (add_rms_norm, decay_attn, decay_attn_decode_step, decay_attn_varlen, gated_rms_norm, rms_norm)

pytestmark = pytest.mark.gpu

WIDTH, H, HK, DK, DV, EPS = 48, 4, 2, 16, 24, 1e-6
SPLIT = [HK * DK, HK * DK, H * DV, H * DV, H]


def parameters(seed=0):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return {"w": 1 + rn(WIDTH) / 8, "in": rn(sum(SPLIT), WIDTH) / WIDTH**0.5, "gate_b": rn(H), "head_w": 1 + rn(DV) / 8,
            "out": rn(WIDTH, H * DV) / (H * DV)**0.5, "res": 0.5 + rn(WIDTH) / 8}


def operands(p, x):
    """q, k, v, gate and log-decay of normalised rows [..., WIDTH]."""
    q, k, v, z, g = F.linear(x, p["in"]).split(SPLIT, -1)
    heads = lambda t, n: t.unflatten(-1, (n, -1))  # noqa: E731
    return heads(q, HK), heads(k, HK), heads(v, H), heads(z, H), F.logsigmoid(g.float() + p["gate_b"])


def finish(p, o, z):
    return F.linear(gated_rms_norm(o, z, p["head_w"], EPS).flatten(-2), p["out"])


def model(ps, x):
    """Blocks behind one another; the residual sums belong to the next block's norm."""
    y, h, finals = rms_norm(x, ps[0]["w"], EPS), x, []
    for i, p in enumerate(ps):
        q, k, v, z, g = operands(p, y)
        o, fin = decay_attn(q, k, v, g, scale=DK**-0.5)
        finals.append(fin)
        last = i + 1 == len(ps)
        y, h = add_rms_norm(finish(p, o, z), h, None if last else ps[i + 1]["w"], p["res"], EPS)
    return h, finals


def model64(ps, x):
    norm = lambda t, w=1.0: t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS) * w  # noqa: E731
    y, h, finals = norm(x, ps[0]["w"]), x, []
    for i, p in enumerate(ps):
        q, k, v, z, g = F.linear(y, p["in"]).split(SPLIT, -1)
        q, k, v, z = q.unflatten(-1, (HK, -1)), k.unflatten(-1, (HK, -1)), v.unflatten(-1, (H, -1)), z.unflatten(-1, (H, -1))
        g = F.logsigmoid(g + p["gate_b"])
        q, k = (t.repeat_interleave(H // HK, -2) for t in (q, k))
        s, outs = torch.zeros(x.shape[0], H, DK, DV, dtype=x.dtype), []
        for t in range(x.shape[1]):
            s = torch.exp(g[:, t])[..., None, None] * s + k[:, t, :, :, None] * v[:, t, :, None, :]
            outs.append((q[:, t, :, :, None] * s).sum(-2) * DK**-0.5)
        finals.append(s)
        o = norm(torch.stack(outs, 1), p["head_w"]) * z * torch.sigmoid(z)
        h = h + p["res"] * F.linear(o.flatten(-2), p["out"])
        y = norm(h, ps[i + 1]["w"]) if i + 1 < len(ps) else None
    return h, finals


def close(got, ref, units, what):
    """Relative 2-norm: `units` roundings of 2^-24 at most in a row, on sums of terms of random signs, whose norm is at
    least a quarter of their absolute values'."""
    got = D.d64(got)
    assert float((got - ref).norm()) <= 4 * units * D.U * float(ref.norm()), what


def units(T, blocks, ways=1):
    """Roundings in a row: 7 T + 3 |G| (at most 2 T here) + ends of the attention, the projections' sums of at most
    H DV terms twice, the norms' under 200; each way of each block."""
    return blocks * ways * (9 * T + D.ends(DK, DV) + 3 * H * DV + 400)


def test_training_step_against_64_bits(dev):
    B, T = 2, 45
    ps = [parameters(1), parameters(2)]
    x = torch.randn(B, T, WIDTH, generator=torch.Generator().manual_seed(3))
    up = torch.randn(B, T, WIDTH, generator=torch.Generator().manual_seed(4))
    dev_ps = [{k: v.to(dev).requires_grad_() for k, v in p.items()} for p in ps]
    ref_ps = [{k: v.double().requires_grad_() for k, v in p.items()} for p in ps]
    xd, xr = x.to(dev).requires_grad_(), x.double().requires_grad_()
    (hd, fd), (hr, fr) = model(dev_ps, xd), model64(ref_ps, xr)
    close(hd, hr.detach(), units(T, 2), "h")
    for a, b in zip(fd, fr):
        close(a, b.detach(), units(T, 2), "state")
    leaves = lambda first, qs: [first, *(q[k] for q in qs for k in sorted(ps[0]))]  # noqa: E731
    gd = torch.autograd.grad(hd, leaves(xd, dev_ps), up.to(dev))
    gr = torch.autograd.grad(hr, leaves(xr, ref_ps), up.double())
    for i, (a, b) in enumerate(zip(gd, gr)):
        close(a, b, units(T, 2, 2), f"gradient {i}")


def step(ps, x, pools, slots, varlen=None):
    """Rows x [N, WIDTH]: packed prompts (varlen: their offsets), or one token for each slot."""
    y, h = rms_norm(x, ps[0]["w"], EPS), x
    for i, (p, pool) in enumerate(zip(ps, pools)):
        q, k, v, z, g = operands(p, y)
        if varlen is None:
            o, _ = decay_attn_decode_step(q, k, v, g, pool, DK**-0.5, inplace=True, slots=slots)
        else:
            o, _ = decay_attn_varlen(q, k, v, g, varlen, scale=DK**-0.5, state_pool=pool, slots=slots)
        last = i + 1 == len(ps)
        y, h = add_rms_norm(finish(p, o, z), h, None if last else ps[i + 1]["w"], p["res"], EPS)
    return h


@torch.no_grad()
def test_packed_prefill_and_decode_against_whole_prompts(dev):
    ps = [{k: v.to(dev) for k, v in parameters(s).items()} for s in (5, 6)]
    lens, extra = [7, 40, 1, 70], 3
    whole = [torch.randn(1, n + extra, WIDTH, generator=torch.Generator().manual_seed(i)).to(dev) for i, n in enumerate(lens)]
    pools = [torch.zeros(6, H, DK, DV, device=dev) for _ in ps]
    slots = torch.tensor([5, 0, 3, 2], device=dev, dtype=torch.int32)
    cu = torch.tensor([0, *lens]).cumsum(0).to(torch.int32).to(dev)
    outs = [[o] for o in step(ps, torch.cat([w[0, :n] for w, n in zip(whole, lens)]), pools, slots, cu).split(lens)]
    for t in range(extra):
        for o, row in zip(outs, step(ps, torch.cat([w[:, n + t] for w, n in zip(whole, lens)]), pools, slots)):
            o.append(row[None])
    ref_ps = [{k: v.cpu().double() for k, v in p.items()} for p in ps]
    for i, w in enumerate(whole):
        ref, finals = model64(ref_ps, w.cpu().double())
        close(torch.cat(outs[i]), ref[0], units(w.shape[1], 2), f"sequence {i}")
        for pool, s in zip(pools, finals):
            close(pool[slots[i]], s[0], units(w.shape[1], 2), f"state {i}")
    assert all(bool((pool[[1, 4]] == 0).all()) for pool in pools)


def warm(dev, fn):
    """The projections' library picks its kernels before the capture."""
    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream(dev).wait_stream(side)


@torch.no_grad()
@pytest.mark.parametrize("packed", [False, True])
def test_captured_serving_steps(dev, packed):
    """The step for four sessions (a packed prefill of four prompts) in a graph, replayed with new rows and eager work
    between, against eager steps on other pools."""
    ps = [{k: v.to(dev) for k, v in parameters(s).items()} for s in (7, 8)]
    slots = torch.tensor([4, 1, 0, 3], device=dev, dtype=torch.int32)
    cu = torch.tensor([0, 3, 300, 301, 900], device=dev, dtype=torch.int32) if packed else None
    pools = [[torch.zeros(5, H, DK, DV, device=dev) for _ in ps] for _ in range(2)]
    x = torch.randn(900 if packed else 4, WIDTH, device=dev)
    warm(dev, lambda: step(ps, x, [t.clone() for t in pools[0]], slots, cu))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(ps, x, pools[0], slots, cu)
    for t in pools[0]:
        t.zero_()
    for n in range(4):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(n)))
        graph.replay()
        eager = step(ps, x, pools[1], slots, cu)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and all(torch.equal(a, b) for a, b in zip(*pools))


def test_captured_training_steps(dev):
    """Forward and backward of each operator through its public call, captured together and replayed with new inputs and
    eager steps (on leaves of their own) between."""
    rn = lambda *s: torch.randn(*s, device=dev)  # noqa: E731
    bf = torch.bfloat16
    B, T = 2, 333
    ops = [
        (lambda q, k, v, g, s: decay_attn(q, k, v, F.logsigmoid(g), s),
         [rn(B, T, 2, 64).to(bf), rn(B, T, 2, 64).to(bf), rn(B, T, 4, 32).to(bf), rn(B, T, 4), rn(B, 4, 64, 32)]),
        (lambda q, k, v, g: decay_attn(q, k, v, F.logsigmoid(g)),
         [rn(B, T, 1, 20), rn(B, T, 1, 20), rn(B, T, 2, 36), rn(2)]),
        (lambda x, r, w, s: add_rms_norm(x, r, w, s), [rn(B, T, 200).to(bf), rn(B, T, 200), rn(200), rn(200).to(bf)]),
        (lambda x, z, w: (gated_rms_norm(x, z, w),), [rn(B, T, 4, 32).to(bf), rn(B, T, 4, 32).to(bf), rn(32)]),
    ]
    for op, data in ops:
        with torch.no_grad():
            ups = [torch.randn_like(t) for t in op(*data)]

        def run(inputs, ups=ups, op=op):
            leaves = [t.detach().requires_grad_() for t in inputs]
            return torch.autograd.grad(op(*leaves), leaves, ups)

        warm(dev, lambda: run(data))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(data)
        for n in range(3):
            data[0].copy_(torch.randn(data[0].shape, generator=torch.Generator().manual_seed(n)))
            for t in out:
                t.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, run(data)):
                assert torch.equal(a, b)
        del graph
