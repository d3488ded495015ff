"""The state space layer's operators as they are timed: the selective scan, the short causal
convolution and layer norm, each from its smallest call to its largest, with a plain form in torch and
64-bit results to compare with.

A case is a dict of plain values; `kind` names the call:

  scan         ssm_scan without gradients: prompts of one length, from a carried-in state
  scan_packed  ssm_scan_varlen: ragged prompts packed end to end, states in a pool
  scan_step    ssm_decode_step: one token for each of B sessions, states in a pool, in place
  scan_train   ssm_scan forward and backward
  conv         short_conv without gradients, over a carried-in state
  conv_packed  short_conv_varlen over a pool
  conv_step    short_conv_decode_step over a pool, in place
  conv_train   short_conv forward and backward
  norm         layer_norm without gradients
  norm_train   layer_norm forward and backward

Distributions are those of a layer at the start of its training: step sizes dt log-uniform in
[1e-3, 0.1] through the bias of their softplus, A near -(1 .. N), everything that a projection gives
~ N(0, 1); x and z are the two halves of one projection, B and C parts of another, so they come as
views.  Widths are heads times head dim of the framework's configurations (6 x 64, 12 x 128 and
multiples) or generic.
"""

from __future__ import annotations

import math
import random

import torch

DEV = "cuda"
own = False
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_MOST_STATES = 201_326_592  # (token, channel, state) triples of the largest listed scan
_MOST_VALUES = 50_331_648  # values of the largest listed convolution or norm


def listed():
    return [
        # one session generating a token through a small layer: all latency
        {"name": "scan_step_one", "kind": "scan_step", "B": 1, "D": 768, "N": 16, "io": "bf16"},
        # batched decode: 256 sessions of a 12 x 128 wide layer, one state read and written each
        {"name": "scan_step_batch", "kind": "scan_step", "B": 256, "D": 1536, "N": 16, "io": "bf16"},
        # one long prompt: few channels, so the time axis has to be split
        {"name": "scan_long", "kind": "scan", "B": 1, "T": 16384, "D": 768, "N": 16, "G": 1, "io": "bf16", "gate": True},
        # continuous batching: 16 ragged prompts, states kept in the pool's slots
        {"name": "scan_packed", "kind": "scan_packed", "n": 16, "lo": 16, "hi": 2048, "lseed": 4, "D": 1536, "N": 16,
         "G": 1, "io": "bf16", "gate": True},
        # a training step's scan at the prompt length of the recall benchmark
        {"name": "scan_train", "kind": "scan_train", "B": 4, "T": 2048, "D": 1536, "N": 16, "G": 1, "io": "bf16",
         "gate": True},
        # fp32 training at odd sizes, two groups of B and C, no gate
        {"name": "scan_train_odd", "kind": "scan_train", "B": 3, "T": 777, "D": 200, "N": 24, "G": 2, "io": "fp32",
         "gate": False},
        # one token of 256 sessions through the convolution
        {"name": "conv_step", "kind": "conv_step", "B": 256, "D": 1536, "W": 4, "io": "bf16", "silu": True, "bias": True},
        # long prompts, the headline benchmark's batch and length
        {"name": "conv_long", "kind": "conv", "B": 4, "T": 16384, "D": 768, "W": 4, "io": "bf16", "silu": True,
         "bias": True},
        # a training step's convolution
        {"name": "conv_train", "kind": "conv_train", "B": 8, "T": 2048, "D": 1536, "W": 4, "io": "bf16", "silu": True,
         "bias": True},
        # the norm of a decode batch of 256 sessions
        {"name": "norm_step", "kind": "norm", "R": 256, "D": 384, "io": "bf16", "affine": True},
        # a training step's norm
        {"name": "norm_train", "kind": "norm_train", "R": 16384, "D": 1536, "io": "bf16", "affine": True},
        # fp32 rows of an odd number and width
        {"name": "norm_train_odd", "kind": "norm_train", "R": 9003, "D": 1001, "io": "fp32", "affine": True},
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random):
    kind = rng.choice(["scan", "scan", "scan_packed", "scan_step", "scan_train", "scan_train", "conv", "conv_packed",
                       "conv_step", "conv_train", "norm", "norm_train"])
    io = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    case = {"kind": kind, "io": io}
    if kind.startswith("norm"):
        D = _log(rng, 8, 16384)
        case.update(R=_log(rng, 1, max(1, min(65536, _MOST_VALUES // (2 * D)))), D=D, affine=rng.random() < 0.8)
        return case
    if kind.startswith("conv"):
        D = _log(rng, 16, 8192)
        case.update(D=D, W=rng.choice([2, 3, 4, 4]), silu=rng.random() < 0.8, bias=rng.random() < 0.7)
        if kind == "conv_step":
            case["B"] = _log(rng, 1, 1024)
        elif kind == "conv_packed":
            case.update(n=_log(rng, 1, 64), lo=1, hi=_log(rng, 2, 2048), lseed=rng.randrange(1000))
        else:
            case.update(B=_log(rng, 1, 16), T=_log(rng, 1, 16384))
            case["T"] = max(1, min(case["T"], _MOST_VALUES // (2 * case["B"] * D)))
        return case
    G = rng.choice([1, 1, 1, 2, 4])
    D, N = G * _log(rng, 16, 4096 // G), rng.choice([4, 8, 16, 16, 16, 24, 32, 64, rng.randint(1, 40)])
    case.update(D=D, N=N)
    if kind == "scan_step":
        case["B"] = _log(rng, 1, 1024)
        return case
    case.update(G=G, gate=rng.random() < 0.7)
    most = max(1, _MOST_STATES // (2 * D * N))
    if kind == "scan_packed":
        case["n"] = min(_log(rng, 1, 64), max(1, most // 2))
        case.update(lo=1, hi=max(1, min(_log(rng, 1, 8192), most // case["n"])), lseed=rng.randrange(1000))
    else:
        case["B"] = min(_log(rng, 1, 32), most)
        case["T"] = max(1, min(_log(rng, 1, 16384 if kind == "scan" else 8192), most // case["B"]))
    return case


def _lengths(case) -> list[int]:
    r = random.Random(case["lseed"])
    return [_log(r, case["lo"], case["hi"]) for _ in range(case["n"])]


# ---- inputs ------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    kind, dt, D = case["kind"], _DT[case["io"]], case["D"]
    train = kind.endswith("_train")
    s = {"case": dict(case), "dt": dt}
    leaf = lambda x: x.requires_grad_() if train else x  # noqa: E731
    if kind.startswith("norm"):
        R = case["R"]
        # a residual stream: rows of differing scale and offset, a few wide channels
        x = rn(R, D) * (0.5 + 2.0 * torch.rand(R, 1, generator=gen, device=DEV)) + 0.5 * rn(R, 1) + rn(D)
        s["x"] = leaf(x.to(dt))
        s["w"] = leaf((1.0 + 0.1 * rn(D)).to(dt)) if case["affine"] else None
        s["b"] = leaf((0.1 * rn(D)).to(dt)) if case["affine"] else None
        if train:
            s["dy"] = rn(R, D).to(dt)
        return s
    if "lseed" in case:
        lens = _lengths(case)
        s["cu"] = torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(torch.int32).to(DEV)
        lead, nseq = (sum(lens),), case["n"]
    elif kind.endswith("_step"):
        lead, nseq = (case["B"],), case["B"]
    else:
        lead, nseq = (case["B"], case["T"]), case["B"]
    if kind.endswith("_step") or "lseed" in case:  # sessions in scattered slots of a larger pool
        rows = nseq + 3
        s["slots"] = torch.randperm(rows, generator=gen, device=DEV)[:nseq].to(torch.int32)
    else:
        rows = nseq
    if kind.startswith("conv"):
        W = case["W"]
        x = rn(*lead, 2 * D).to(dt)[..., :D]
        s["x"] = leaf(x.contiguous() if train else x)
        s["w"] = leaf((rn(D, W) / math.sqrt(W)).to(dt))
        s["b"] = leaf((0.1 * rn(D)).to(dt)) if case["bias"] else None
        s["state"] = leaf(rn(rows, W - 1, D).to(dt))
        if train:
            s["dy"], s["dstate"] = rn(*lead, D).to(dt), rn(nseq, W - 1, D).to(dt)
        return s
    N, G = case["N"], case.get("G", 1)
    gate = case.get("gate", True)
    u = rn(*lead, D)
    s["u"] = leaf((u * torch.sigmoid(u)).to(dt))  # what the convolution gives
    s["delta"] = leaf((0.5 * rn(*lead, D)).to(dt))
    bc = rn(*lead, 2 * G * N).to(dt)
    bs, cs = bc[..., :G * N], bc[..., G * N:]
    shape = (*lead, G, N) if G > 1 else (*lead, N)
    s["B"], s["C"] = (leaf((x.contiguous() if train else x).reshape(shape)) for x in (bs, cs))
    s["z"] = None
    if gate:
        z = rn(*lead, 2 * D).to(dt)[..., D:]
        s["z"] = leaf(z.contiguous() if train else z)
    s["A"] = leaf(-torch.arange(1, N + 1, device=DEV).float() * torch.exp(0.1 * rn(D, N)))
    s["Dp"] = leaf(1.0 + 0.1 * rn(D))
    step = torch.exp(torch.rand(D, generator=gen, device=DEV) * math.log(100.0) + math.log(1e-3))
    s["bias"] = leaf(step + torch.log(-torch.expm1(-step)))
    s["state"] = leaf(0.1 * rn(rows, D, N))
    if train:
        s["dy"], s["dstate"] = rn(*lead, D).to(dt), 0.1 * rn(nseq, D, N)
    return s


# ---- the plain forms -----------------------------------------------------------------------------
def _linear_scan(a, x):
    """h_t = a_t h_{t-1} + x_t along dim 1 from h = 0, by doubling."""
    step = 1
    while step < x.shape[1]:
        x = torch.cat((x[:, :step], x[:, step:] + a[:, step:] * x[:, :-step]), 1)
        a = torch.cat((a[:, :step], a[:, step:] * a[:, :-step]), 1)
        step *= 2
    return x


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def _f(t):
    return None if t is None else t.detach().float()


def _per_channel(x, D):
    """B or C [..., N] or [..., G, N] as [..., D or 1, N]."""
    if x.dim() == 3:
        return x.unsqueeze(-2)
    return x.repeat_interleave(D // x.shape[-2], -2)


def _per_group(x, like):
    """The sum over the channels that share a row of `like`: [B, T, D, N] to like's shape."""
    if like.dim() == 3:
        return x.sum(2)
    return x.unflatten(2, (like.shape[2], -1)).sum(3)


def _scan_fwd(u, delta, A, B, C, Dp, z, bias, h0, starts=None):
    dt = _softplus(delta + bias)
    a = torch.exp(dt.unsqueeze(-1) * A)
    x = (dt * u).unsqueeze(-1) * _per_channel(B, u.shape[-1])
    if starts is None:
        x[:, 0] += a[:, 0] * h0
        h = _linear_scan(a, x)
    else:  # packed: a sequence starts from its own state
        x[0, starts] += a[0, starts] * h0
        cut = a.clone()
        cut[0, starts] = 0
        h = _linear_scan(cut, x)
    y = (h * _per_channel(C, u.shape[-1])).sum(-1) + Dp * u
    return (y if z is None else y * z * torch.sigmoid(z)), y, h, a, dt


def _scan_plain(s):
    case, dt_ = s["case"], s["dt"]
    u, delta, A, B, C, Dp, z, bias, h0 = (_f(s[k]) for k in ("u", "delta", "A", "B", "C", "Dp", "z", "bias", "state"))
    kind = case["kind"]
    if kind == "scan_step":
        rows = s["slots"].long()
        dt = _softplus(delta + bias)
        h = torch.exp(dt.unsqueeze(-1) * A) * h0[rows] + (dt * u).unsqueeze(-1) * B.unsqueeze(1)
        y = (h * C.unsqueeze(1)).sum(-1) + Dp * u
        s["state"][rows] = h
        return (y * z * torch.sigmoid(z)).to(dt_), s["state"]
    if kind == "scan_packed":
        rows, cu = s["slots"].long(), s["cu"].long()
        one = [None if x is None else x.unsqueeze(0) for x in (u, delta, B, C, z)]
        out, _, h, _, _ = _scan_fwd(one[0], one[1], A, one[2], one[3], Dp, one[4], bias, h0[rows], cu[:-1])
        s["state"][rows] = h[0, cu[1:] - 1]
        return out[0].to(dt_), s["state"]
    out, y, h, a, dt = _scan_fwd(u, delta, A, B, C, Dp, z, bias, h0)
    final = h[:, -1].clone()
    if kind == "scan":
        return out.to(dt_), final
    dy, dstate = _f(s["dy"]), _f(s["dstate"])
    D = u.shape[-1]
    dz = None
    if z is not None:
        sg = torch.sigmoid(z)
        dz = (dy * y * sg * (1 + z * (1 - sg))).to(dt_)
        dy = dy * z * sg
    g = dy.unsqueeze(-1) * _per_channel(C, D)
    g[:, -1] += dstate
    after = torch.cat((a[:, 1:], torch.zeros_like(a[:, :1])), 1)
    dh = _linear_scan(after.flip(1), g.flip(1)).flip(1)
    dC = _per_group(dy.unsqueeze(-1) * h, C)
    before = torch.cat((h0.unsqueeze(1), h[:, :-1]), 1)
    dB = _per_group(dh * (dt * u).unsqueeze(-1), B)
    db = (dh * _per_channel(B, D)).sum(-1)
    dh0 = a[:, 0] * dh[:, 0]
    p = dh * a * before
    ddelta = ((p * A).sum(-1) + db * u) * torch.sigmoid(delta + bias)
    return {"y": out.to(dt_), "final": final, "du": (db * dt + Dp * dy).to(dt_), "ddelta": ddelta.to(dt_),
            "dA": (p * dt.unsqueeze(-1)).sum((0, 1)), "dB": dB.to(dt_), "dC": dC.to(dt_), "dD": (dy * u).sum((0, 1)),
            "dz": dz, "dbias": ddelta.sum((0, 1)), "dstate0": dh0}


def _conv_plain(s):
    case, dt_, W = s["case"], s["dt"], s["case"]["W"]
    x, w, b, st = (_f(s[k]) for k in ("x", "w", "b", "state"))
    kind = case["kind"]
    if kind == "conv_packed":
        rows, cu = s["slots"].long(), s["cu"].long()
        at = torch.arange(x.shape[0], device=x.device)
        seq = torch.searchsorted(cu, at, right=True) - 1
        back = torch.arange(W, device=x.device) - (W - 1)
        pos = at[:, None] + back  # [N, W]; before a sequence's start the pool's rows
        into = pos - cu[seq][:, None]
        old = st[rows[seq][:, None], (into + W - 1).clamp(0, W - 2)]
        win = torch.where((into >= 0)[..., None], x[pos.clamp(min=0)], old).transpose(1, 2)
        p = (win * w).sum(-1)
        last = cu[1:, None] + back[:-1] + 0  # the last W - 1 tokens of [state, sequence]
        into = last - cu[:-1, None]
        old = s["state"][rows[:, None], (into + W - 1).clamp(0, W - 2)]
        s["state"][rows] = torch.where((into >= 0)[..., None], s["x"][last.clamp(min=0)], old)
        final = s["state"]
    else:
        step = kind == "conv_step"
        rows = s["slots"].long() if step else None
        cur, prev = (s["x"].unsqueeze(1), s["state"][rows]) if step else (s["x"], s["state"])
        full = torch.cat((prev, cur), 1).detach()
        p = (full.float().unfold(1, W, 1) * w).sum(-1)
        final = full[:, full.shape[1] - (W - 1):].clone()
        if step:
            s["state"][rows] = final
            p, final = p[:, 0], s["state"]
    if b is not None:
        p = p + b
    sg = torch.sigmoid(p) if case["silu"] else None
    y = (p if sg is None else p * sg).to(dt_)
    if kind != "conv_train":
        return y, final
    dp = _f(s["dy"])
    if sg is not None:
        dp = dp * sg * (1 + p * (1 - sg))
    pad = torch.zeros_like(dp[:, :1]).expand(-1, W - 1, -1)
    dfull = (torch.cat((pad, dp, pad), 1).unfold(1, W, 1) * w.flip(1)).sum(-1)
    dfull[:, dfull.shape[1] - (W - 1):] += _f(s["dstate"])
    dw = (full.float().unfold(1, W, 1) * dp.unsqueeze(-1)).sum((0, 1))
    return {"y": y, "final": final, "dx": dfull[:, W - 1:].to(dt_), "dw": dw.to(dt_),
            "db": None if b is None else dp.sum((0, 1)).to(dt_), "dstate0": dfull[:, :W - 1].to(dt_)}


_EPS = 1e-5


def _norm_plain(s):
    x, w, b, dt_ = _f(s["x"]), _f(s["w"]), _f(s["b"]), s["dt"]
    c = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((c * c).mean(-1, keepdim=True) + _EPS)
    xh = c * r
    y = (xh if w is None else xh * w + b).to(dt_)
    if s["case"]["kind"] == "norm":
        return y
    dy = _f(s["dy"])
    g = dy if w is None else dy * w
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return {"y": y, "dx": dx.to(dt_), "dw": None if w is None else (dy * xh).sum(0).to(dt_),
            "db": None if w is None else dy.sum(0).to(dt_)}


# ---- the framework's calls -----------------------------------------------------------------------
def _grads(outs, ups, names, s, keys):
    have = [(n, s[k]) for n, k in zip(names, keys) if s[k] is not None]
    got = dict(zip([n for n, _ in have], torch.autograd.grad(outs, [x for _, x in have], ups)))
    return {n: got.get(n) for n in names}


def _own(s):
    import triune_amd as fw

    kind, case = s["case"]["kind"], s["case"]
    if kind.startswith("norm"):
        y = fw.layer_norm(s["x"], s["w"], s["b"], eps=_EPS)
        if kind == "norm":
            return y
        return {"y": y.detach(), **_grads((y,), (s["dy"],), ("dx", "dw", "db"), s, ("x", "w", "b"))}
    if kind.startswith("conv"):
        act = "silu" if case["silu"] else None
        if kind == "conv_step":
            return fw.short_conv_decode_step(s["x"], s["w"], s["state"], bias=s["b"], activation=act, inplace=True,
                                             slots=s["slots"])
        if kind == "conv_packed":
            return fw.short_conv_varlen(s["x"], s["w"], s["cu"], bias=s["b"], activation=act, state_pool=s["state"],
                                        slots=s["slots"])
        y, final = fw.short_conv(s["x"], s["w"], bias=s["b"], initial_state=s["state"], activation=act)
        if kind == "conv":
            return y, final
        return {"y": y.detach(), "final": final.detach(),
                **_grads((y, final), (s["dy"], s["dstate"]), ("dx", "dw", "db", "dstate0"), s,
                         ("x", "w", "b", "state"))}
    kw = {"D": s["Dp"], "z": s["z"], "delta_bias": s["bias"]}
    args = (s["u"], s["delta"], s["A"], s["B"], s["C"])
    if kind == "scan_step":
        return fw.ssm_decode_step(*args, s["state"], inplace=True, slots=s["slots"], **kw)
    if kind == "scan_packed":
        return fw.ssm_scan_varlen(*args, s["cu"], state_pool=s["state"], slots=s["slots"], **kw)
    y, final = fw.ssm_scan(*args, initial_state=s["state"], **kw)
    if kind == "scan":
        return y, final
    return {"y": y.detach(), "final": final.detach(),
            **_grads((y, final), (s["dy"], s["dstate"]),
                     ("du", "ddelta", "dA", "dB", "dC", "dD", "dz", "dbias", "dstate0"), s,
                     ("u", "delta", "A", "B", "C", "Dp", "z", "bias", "state"))}


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    return (_norm_plain if kind.startswith("norm") else _conv_plain if kind.startswith("conv") else _scan_plain)(state)


# ---- what a pass cannot do without -----------------------------------------------------------------
def work(case):
    kind, D, E = case["kind"], case["D"], _DT[case["io"]].itemsize
    train = kind.endswith("_train")
    if kind.startswith("norm"):
        v, par = case["R"] * D, 2 * D * E if case["affine"] else 0
        if not train:
            return {"bytes": 2 * v * E + par, "flops": 8 * v}
        return {"bytes": 4 * v * E + 2 * par, "flops": 21 * v}
    if "lseed" in case:
        tok, nseq = sum(_lengths(case)), case["n"]
    else:
        tok, nseq = case["B"] * case.get("T", 1), case["B"]
    v = tok * D
    if kind.startswith("conv"):
        W = case["W"]
        state, par = 2 * nseq * (W - 1) * D * E, D * (W + int(case["bias"])) * E
        if not train:
            return {"bytes": 2 * v * E + state + par, "flops": v * (2 * W + 5)}
        return {"bytes": 4 * v * E + 2 * state + 2 * par, "flops": v * (6 * W + 16)}
    N, G = case["N"], case.get("G", 1)
    acts = 3 + int(case.get("gate", True))  # u, delta, (z), y
    state, par = 2 * nseq * D * N * 4, D * (N + 2) * 4
    fwd = acts * v * E + 2 * tok * G * N * E + state + par
    if not train:
        return {"bytes": fwd, "flops": v * (7 * N + 16)}
    # gradients of u, delta, (z), B, C, the parameters and the entering state, upstream of y and the final state
    return {"bytes": 2 * fwd, "flops": v * (25 * N + 50)}


# ---- 64-bit results ---------------------------------------------------------------------------------
def _steps64(u, delta, A, B, C, Dp, z, bias, h):
    """The definition, a token at a time: u ... [B, T, *] -> (y, last state)."""
    D = u.shape[-1]
    if B.dim() == 4:
        g = torch.arange(D, device=u.device) // (D // B.shape[2])
    outs = []
    for t in range(u.shape[1]):
        x = delta[:, t] + bias
        dt = torch.where(x > 30, x, torch.log1p(torch.exp(torch.clamp(x, max=30))))
        b, c = (v[:, t, g] if v.dim() == 4 else v[:, t, None] for v in (B, C))
        h = torch.exp(dt[..., None] * A) * h + (dt * u[:, t])[..., None] * b
        y = (h * c).sum(-1) + Dp * u[:, t]
        if z is not None:
            y = y * z[:, t] / (1 + torch.exp(-z[:, t]))
        outs.append(y)
    return torch.stack(outs, 1), h


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    train = kind.endswith("_train")
    d = {k: v.detach().double().requires_grad_(train) for k, v in s.items()
         if torch.is_tensor(v) and v.is_floating_point()}
    for k in ("w", "b", "z"):
        d.setdefault(k, None)
    if kind.startswith("norm"):
        y = torch.nn.functional.layer_norm(d["x"], (case["D"],), d["w"], d["b"], _EPS)
        if not train:
            return y
        return {"y": y.detach(), **_grads((y,), (s["dy"].double(),), ("dx", "dw", "db"), d, ("x", "w", "b"))}
    rows = s["slots"].long() if "slots" in s else None
    if kind.startswith("conv"):
        W, w = case["W"], d["w"]

        def conv(x, prev):  # x [B, T, D], prev [B, W - 1, D]
            full = torch.cat((prev, x), 1)
            p = 0 if d["b"] is None else d["b"]
            for j in range(W):
                p = p + w[:, j] * full[:, j:j + x.shape[1]]
            return (p / (1 + torch.exp(-p)) if case["silu"] else p), full[:, x.shape[1]:]

        if rows is None:
            y, final = conv(d["x"], d["state"])
            if not train:
                return y, final
            return {"y": y.detach(), "final": final.detach(),
                    **_grads((y, final), (s["dy"].double(), s["dstate"].double()), ("dx", "dw", "db", "dstate0"), d,
                             ("x", "w", "b", "state"))}
        cu = s["cu"].tolist() if "cu" in s else list(range(case["B"] + 1))
        if "cu" not in s:
            y, d["state"][rows] = conv(d["x"].unsqueeze(1), d["state"][rows])
            return y[:, 0], d["state"]
        ys = []
        for i, r in enumerate(rows.tolist()):
            y, d["state"][r:r + 1] = conv(d["x"][None, cu[i]:cu[i + 1]], d["state"][r:r + 1].clone())
            ys.append(y[0])
        return torch.cat(ys), d["state"]
    args = lambda pick: [None if d[k] is None else pick(d[k]) for k in ("u", "delta", "B", "C", "z")]  # noqa: E731
    par = (d["A"], d["Dp"], d["bias"])

    def steps(u, delta, B, C, z, h):
        return _steps64(u, delta, par[0], B, C, par[1], z, par[2], h)

    if kind == "scan_step":
        y, d["state"][rows] = steps(*args(lambda x: x.unsqueeze(1)), d["state"][rows])
        return y[:, 0], d["state"]
    if kind == "scan_packed":
        cu, ys = s["cu"].tolist(), []
        if cu[-1] > 50000:
            return None
        for i, r in enumerate(rows.tolist()):
            y, d["state"][r:r + 1] = steps(*args(lambda x: x[None, cu[i]:cu[i + 1]]), d["state"][r:r + 1].clone())
            ys.append(y[0])
        return torch.cat(ys), d["state"]
    y, final = steps(*args(lambda x: x), d["state"])
    if kind == "scan":
        return y, final
    return {"y": y.detach(), "final": final.detach(),
            **_grads((y, final), (s["dy"].double(), s["dstate"].double()),
                     ("du", "ddelta", "dA", "dB", "dC", "dD", "dz", "dbias", "dstate0"), d,
                     ("u", "delta", "A", "B", "C", "Dp", "z", "bias", "state"))}
