"""A decay attention layer's operators as they are timed: linear attention whose state decays by one factor per
head and token, and the norms before and after it with the residual sum and the gate, each from its smallest call to
its largest, with a plain form in torch and 64-bit results to compare with.

A case is a dict of plain values; `kind` names the call:

  attn             decay_attn without gradients: prompts of one length, from a carried-in state
  attn_packed      decay_attn_varlen: ragged prompts packed end to end, states in a pool
  attn_step        decay_attn_decode_step: one token for each of B sessions, states in a pool, in place
  attn_train       decay_attn forward and backward
  add_norm         add_rms_norm (rms_norm where there is no residual) without gradients
  add_norm_train   the same forward and backward
  gate_norm        gated_rms_norm without gradients
  gate_norm_train  gated_rms_norm forward and backward

H heads of v share Hk heads of q and k.  gate "token" is a log-decay for every token and head, -softplus(.) a with
a in [1, 16] and steps from 1e-3 to 0.1; "head" is one constant per head, log(1 - 2^-(5 + h)).  Heads and their dims
are those of the framework's configurations (6 x 64, 12 x 128) or generic.
"""

from __future__ import annotations

import math
import random

import torch

DEV = "cuda"
own = False
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_MOST_ROWS = 50_331_648  # q and v values of the largest listed prompts
_MOST_STATE = 50_331_648  # state values of the largest listed decode batch
_MOST_VALUES = 50_331_648  # values of the largest listed norm
_EPS = 1e-6


def listed():
    return [
        # one session generating a token through a small layer: all latency
        {"name": "attn_step_one", "kind": "attn_step", "B": 1, "H": 6, "Hk": 6, "Dk": 64, "Dv": 64, "io": "bf16",
         "gate": "token"},
        # batched decode: 256 sessions of a 12 x 128 layer, one state read and written each
        {"name": "attn_step_batch", "kind": "attn_step", "B": 256, "H": 12, "Hk": 12, "Dk": 128, "Dv": 128,
         "io": "bf16", "gate": "token"},
        # the headline benchmark's prompts
        {"name": "attn_prompts", "kind": "attn", "B": 4, "T": 16384, "H": 6, "Hk": 6, "Dk": 64, "Dv": 64, "io": "bf16",
         "gate": "token"},
        # a prompt through a layer whose 24 heads share one head of q and k
        {"name": "attn_shared", "kind": "attn", "B": 1, "T": 8192, "H": 24, "Hk": 1, "Dk": 128, "Dv": 64, "io": "bf16",
         "gate": "token"},
        # continuous batching: 16 ragged prompts, states kept in the pool's slots
        {"name": "attn_packed", "kind": "attn_packed", "n": 16, "lo": 16, "hi": 2048, "lseed": 4, "H": 12, "Hk": 12,
         "Dk": 128, "Dv": 128, "io": "bf16", "gate": "token"},
        # a training step's attention at the prompt length of the recall benchmark
        {"name": "attn_train", "kind": "attn_train", "B": 4, "T": 2048, "H": 12, "Hk": 12, "Dk": 128, "Dv": 128,
         "io": "bf16", "gate": "token"},
        # fp32 training at odd sizes, shared heads, one constant decay per head
        {"name": "attn_train_odd", "kind": "attn_train", "B": 3, "T": 777, "H": 6, "Hk": 2, "Dk": 48, "Dv": 80,
         "io": "fp32", "gate": "head"},
        # the residual sum and norm of a decode batch of 256 sessions
        {"name": "add_norm_step", "kind": "add_norm", "R": 256, "D": 384, "io": "bf16", "res": "io", "scale": "none"},
        # a training step's residual sum and norm, with a residual scale for each channel
        {"name": "add_norm_train", "kind": "add_norm_train", "R": 16384, "D": 1536, "io": "bf16", "res": "io",
         "scale": "channel"},
        # a float32 residual stream of an odd number of odd rows under fp16 activations
        {"name": "add_norm_odd", "kind": "add_norm_train", "R": 9003, "D": 1001, "io": "fp16", "res": "fp32",
         "scale": "number"},
        # the norm of every head behind the headline prompts, and its gate
        {"name": "gate_norm_prompts", "kind": "gate_norm", "R": 65536, "H": 6, "D": 64, "io": "bf16"},
        # a training step's
        {"name": "gate_norm_train", "kind": "gate_norm_train", "R": 8192, "H": 12, "D": 128, "io": "bf16"},
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random):
    kind = rng.choice(["attn", "attn", "attn_packed", "attn_step", "attn_train", "attn_train", "add_norm",
                       "add_norm_train", "gate_norm", "gate_norm_train"])
    io = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    case = {"kind": kind, "io": io}
    train = kind.endswith("_train")
    if kind.startswith("add_norm"):
        D = _log(rng, 8, 16384)
        case.update(R=_log(rng, 1, max(1, min(65536, _MOST_VALUES // (2 * D)))), D=D,
                    res=rng.choice(["io", "io", "fp32", "none"]), scale=rng.choice(["none", "number", "channel"]))
        return case
    if kind.startswith("gate_norm"):
        H, D = _log(rng, 1, 32), rng.choice([32, 64, 64, 128, 128, 256, _log(rng, 8, 2048)])
        case.update(R=_log(rng, 1, max(1, min(65536, _MOST_VALUES // (2 * H * D)))), H=H, D=D)
        return case
    Hk = rng.choice([1, 2, 4, 6, 8, 12, rng.randint(1, 16)])
    H = Hk * rng.choice([1, 1, 1, 2, 3, 4, 8])
    Dk = rng.choice([16, 32, 64, 64, 128, 128, rng.randint(8, 128)])
    Dv = rng.choice([Dk, Dk, 64, 128, 256, rng.randint(8, 200)])
    case.update(H=H, Hk=Hk, Dk=Dk, Dv=Dv, gate=rng.choice(["token", "token", "head"]))
    if kind == "attn_step":
        case["B"] = _log(rng, 1, max(1, min(1024, _MOST_STATE // (H * Dk * Dv))))
        return case
    most = max(1, _MOST_ROWS // ((4 if train else 2) * H * (Dk + Dv)))
    if kind == "attn_packed":
        case["n"] = min(_log(rng, 1, 64), most)
        case.update(lo=1, hi=max(1, min(_log(rng, 1, 8192), most // case["n"])), lseed=rng.randrange(1000))
    else:
        case["B"] = min(_log(rng, 1, 32), most)
        case["T"] = max(1, min(_log(rng, 1, 4096 if train else 16384), most // case["B"]))
    return case


def _lengths(case) -> list[int]:
    r = random.Random(case["lseed"])
    return [_log(r, case["lo"], case["hi"]) for _ in range(case["n"])]


# ---- inputs ------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    kind, dt, train = case["kind"], _DT[case["io"]], case["kind"].endswith("_train")
    leaf = lambda x: None if x is None else x.contiguous().requires_grad_() if train else x  # noqa: E731
    s = {"case": dict(case), "dt": dt}
    if kind.startswith("add_norm"):
        R, D = case["R"], case["D"]
        rdt = None if case["res"] == "none" else torch.float32 if case["res"] == "fp32" else dt
        s["x"] = leaf(rn(R, D).to(dt))  # what a block's last projection gives
        # a residual stream: rows of differing scale, a few wide channels
        s["r"] = None if rdt is None else leaf((rn(R, D) * (0.5 + 2 * torch.rand(R, 1, generator=gen, device=DEV))
                                                + rn(D)).to(rdt))
        s["w"] = leaf((1 + 0.1 * rn(D)).to(dt))
        s["s"] = {"none": None, "number": 0.5, "channel": leaf((0.5 + 0.1 * rn(D)).to(dt))}[case["scale"]]
        if rdt is None:
            s["s"] = None
        if train:
            s["dy"], s["dh"] = rn(R, D).to(dt), None if rdt is None else rn(R, D).to(rdt)
        return s
    H = case["H"]
    if kind.startswith("gate_norm"):
        R, D = case["R"], case["D"]
        s["x"] = leaf((rn(R, H, D) * (0.2 + 3 * torch.rand(R, H, 1, generator=gen, device=DEV))).to(dt))
        s["z"] = leaf(rn(R, H * D + H).to(dt)[:, :H * D].unflatten(1, (H, D)))  # beside the gates in one projection
        s["w"] = leaf((1 + 0.1 * rn(D)).to(dt))
        if train:
            s["dy"] = rn(R, H, D).to(dt)
        return s
    Hk, Dk, Dv = case["Hk"], case["Dk"], case["Dv"]
    if "lseed" in case:
        s["lens"] = _lengths(case)
        s["cu"] = torch.tensor([0] + s["lens"], dtype=torch.int64).cumsum(0).to(torch.int32).to(DEV)
        lead, rows, nseq = (sum(s["lens"]),), case["n"] + 3, case["n"]
    elif kind == "attn_step":
        lead, rows, nseq = (case["B"],), case["B"] + 3, case["B"]
    else:
        lead, rows, nseq = (case["B"], case["T"]), case["B"], case["B"]
    if rows > nseq:  # sessions in scattered slots of a larger pool
        s["slots"] = torch.randperm(rows, generator=gen, device=DEV)[:nseq].to(torch.int32)
    qkv = rn(*lead, 2 * Hk * Dk + H * Dv).to(dt)  # one projection
    s["q"] = leaf(qkv[..., :Hk * Dk].unflatten(-1, (Hk, Dk)))
    s["k"] = leaf(qkv[..., Hk * Dk:2 * Hk * Dk].unflatten(-1, (Hk, Dk)))
    s["v"] = leaf(qkv[..., 2 * Hk * Dk:].unflatten(-1, (H, Dv)))
    if case["gate"] == "head":
        s["g"] = leaf(torch.log1p(-torch.exp2(-5.0 - torch.arange(H, device=DEV) % 8)))
    else:
        step = torch.exp(torch.rand(H, generator=gen, device=DEV) * math.log(100.0) + math.log(1e-3))
        a = 1 + 15 * torch.rand(H, generator=gen, device=DEV)
        s["g"] = leaf(-a * torch.nn.functional.softplus(0.5 * rn(*lead, H) + step + torch.log(-torch.expm1(-step))))
    s["state"] = leaf(rn(rows, H, Dk, Dv))
    s["scale"] = Dk**-0.5
    if train:
        s["do"], s["dstate"] = rn(*lead, H, Dv).to(dt), 0.1 * rn(nseq, H, Dk, Dv)
    return s


# ---- the plain forms -----------------------------------------------------------------------------
_C = 64


def _f(t):
    return None if t is None else t.detach().float()


def _chunks(x, fill=0.0):
    """[B, T, H, ...] as [B, chunks, H, 64, ...]."""
    T = x.shape[1]
    n = -(-T // _C)
    if n * _C > T:
        x = torch.cat((x, torch.full_like(x[:, :1], fill).expand(-1, n * _C - T, *x.shape[2:])), 1)
    return x.unflatten(1, (n, _C)).transpose(2, 3)


def _flat(x, T):
    return x.transpose(2, 3).flatten(1, 2)[:, :T]


def _states(a, x):
    """S_c = a_c S_{c-1} + x_c along dim 1 from S = 0, by doubling; a [B, n, H, 1, 1]."""
    step = 1
    while step < x.shape[1]:
        x = torch.cat((x[:, :step], x[:, step:] + a[:, step:] * x[:, :-step]), 1)
        a = torch.cat((a[:, :step], a[:, step:] * a[:, :-step]), 1)
        step *= 2
    return x


def _share(x, H):
    return x.repeat_interleave(H // x.shape[-2], -2)


def _attn_fwd(q, k, v, g, scale, s0, starts=None):
    """Chunked outputs and all that the gradients take; starts: the chunks at which packed sequences start."""
    G = g.cumsum(3)
    end = G[..., -1:]
    i = torch.arange(_C, device=q.device)
    L = torch.where(i[:, None] >= i, torch.exp((G.unsqueeze(-1) - G.unsqueeze(-2)).clamp(max=0)), 0)
    A = scale * (q @ k.transpose(-1, -2)) * L
    own_ = (k * torch.exp(end - G).unsqueeze(-1)).transpose(-1, -2) @ v
    a = torch.exp(end).unsqueeze(-1)
    x = own_.clone()
    if starts is None:
        x[:, 0] += a[:, 0] * s0
        S = _states(a, x)
        S0 = torch.cat((s0.unsqueeze(1), S[:, :-1]), 1)
    else:
        x[0, starts] += a[0, starts] * s0
        cut = a.clone()
        cut[0, starts] = 0
        S = _states(cut, x)
        S0 = torch.cat((torch.zeros_like(S[:, :1]), S[:, :-1]), 1)
        S0[0, starts] = s0
    o = A @ v + scale * torch.exp(G).unsqueeze(-1) * (q @ S0)
    return o, S, (G, end, L, A, S0, a)


def _attn_plain(s):
    case, dt, scale = s["case"], s["dt"], s["scale"]
    kind, H = case["kind"], case["H"]
    q, k, v, g, s0 = (_f(s[n]) for n in ("q", "k", "v", "g", "state"))
    Hk = q.shape[-2]
    q, k = _share(q, H), _share(k, H)
    if g.dim() == 1:
        g = g.expand(*v.shape[:-1])
    if kind == "attn_step":
        rows = s["slots"].long()
        h = torch.exp(g)[..., None, None] * s0[rows] + k.unsqueeze(-1) * v.unsqueeze(-2)
        s["state"][rows] = h
        return (scale * (q.unsqueeze(-1) * h).sum(-2)).to(dt), s["state"]
    if kind == "attn_packed":  # every sequence padded to whole chunks
        rows, cu = s["slots"].long(), s["cu"].long()
        n = (cu[1:] - cu[:-1] + _C - 1) // _C
        first = torch.cat((n.new_zeros(1), n.cumsum(0)))
        at = torch.arange(q.shape[0], device=q.device)
        seq = torch.searchsorted(cu, at, right=True) - 1
        to = at - cu[seq] + _C * first[seq]
        total = _C * sum(-(-m // _C) for m in s["lens"])
        wide = [x.new_zeros(1, total, *x.shape[1:]).index_copy(1, to, x.unsqueeze(0)) for x in (q, k, v, g)]
        o, S, _ = _attn_fwd(*(_chunks(x) for x in wide), scale, s0[rows], first[:-1])
        s["state"][rows] = S[0, first[1:] - 1]
        return _flat(o, total)[0, to].to(dt), s["state"]
    T = q.shape[1]
    q, k, v, g = (_chunks(x) for x in (q, k, v, g))
    o, S, (G, end, L, A, S0, a) = _attn_fwd(q, k, v, g, scale, s0)
    o, final = _flat(o, T).to(dt), S[:, -1].clone()
    if kind == "attn":
        return o, final
    do, dfin = _chunks(_f(s["do"])), _f(s["dstate"])
    eG, eR = torch.exp(G).unsqueeze(-1), torch.exp(end - G).unsqueeze(-1)
    into = scale * (q * eG).transpose(-1, -2) @ do
    after = torch.cat((into[:, 1:], dfin.unsqueeze(1)), 1)  # the gradient of every chunk's end state
    R = _states(torch.cat((a[:, 1:], torch.zeros_like(a[:, :1])), 1).flip(1), after.flip(1)).flip(1)
    B = scale * (do @ v.transpose(-1, -2)) * L
    dq_in = scale * eG * (do @ S0.transpose(-1, -2))
    dk_in = eR * (v @ R.transpose(-1, -2))
    dq = B @ k + dq_in
    dk = B.transpose(-1, -2) @ q + dk_in
    dv = A.transpose(-1, -2) @ do + eR * (k @ R)
    # log-decays: every pair (writing token before t, reading token at t or behind it), added up without cancelling
    i = torch.arange(_C, device=q.device)
    M = torch.where(i[:, None] > i, (q @ k.transpose(-1, -2)) * B, 0)
    pairs = torch.where(i[:, None] >= i, M.cumsum(-1) - M, 0).sum(-2)
    x, y = (q * dq_in).sum(-1), (k * dk_in).sum(-1)
    dg = pairs + x.flip(-1).cumsum(-1).flip(-1) + (y.cumsum(-1) - y) + (a * S0 * R).sum((-1, -2)).unsqueeze(-1)
    ds0 = a[:, 0] * R[:, 0] + into[:, 0]
    one = lambda x: _flat(x, T).unflatten(2, (Hk, H // Hk)).sum(3).to(dt)  # noqa: E731
    dg = _flat(dg.unsqueeze(-1), T).squeeze(-1)
    return {"o": o, "final": final, "dq": one(dq), "dk": one(dk), "dv": _flat(dv, T).to(dt),
            "dg": dg.sum((0, 1)) if case["gate"] == "head" else dg, "dstate0": ds0}


def _rms(x):
    return torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)


def _norm_plain(s):
    case, dt = s["case"], s["dt"]
    x, w = _f(s["x"]), _f(s["w"])
    train = case["kind"].endswith("_train")
    if case["kind"].startswith("gate"):
        z = _f(s["z"])
        r, sg = _rms(x), torch.sigmoid(z)
        xh, gate = x * r, z * sg
        y = (xh * w * gate).to(dt)
        if not train:
            return y
        dy = _f(s["dy"])
        d = dy * w * gate
        dx = r * (d - xh * (d * xh).mean(-1, keepdim=True))
        return {"y": y, "dx": dx.to(dt), "dz": (dy * xh * w * sg * (1 + z * (1 - sg))).to(dt),
                "dw": (dy * xh * gate).sum((0, 1)).to(dt)}
    res, sc = _f(s["r"]), s["s"]
    sc = _f(sc) if torch.is_tensor(sc) else 1.0 if sc is None else sc
    h = s["x"].detach() if res is None else (res + sc * x).to(s["r"].dtype)  # the stream as it is kept
    hf = h.float()
    r = _rms(hf)
    xh = hf * r
    y = (xh * w).to(dt)
    if not train:
        return y if res is None else (y, h)
    dy = _f(s["dy"])
    d = dy * w
    dh = r * (d - xh * (d * xh).mean(-1, keepdim=True))
    out = {"y": y, "dw": (dy * xh).sum(0).to(dt)}
    if res is None:
        return {**out, "dx": dh.to(dt)}
    dh = dh + _f(s["dh"])
    return {**out, "h": h, "dx": (dh * sc).to(dt), "dr": dh.to(s["r"].dtype),
            "ds": (dh * x).sum(0).to(dt) if torch.is_tensor(s["s"]) else None}


# ---- the framework's calls -----------------------------------------------------------------------
def _grads(outs, ups, names, s, keys):
    have = [(n, s[k]) for n, k in zip(names, keys) if torch.is_tensor(s[k])]
    got = dict(zip([n for n, _ in have], torch.autograd.grad(outs, [x for _, x in have], ups)))
    return {n: got.get(n) for n in names}


def _own(s):
    import triune_amd as fw

    kind = s["case"]["kind"]
    if kind.startswith("add_norm"):
        if s["r"] is None:
            y = fw.rms_norm(s["x"], s["w"], eps=_EPS)
            if kind == "add_norm":
                return y
            return {"y": y.detach(), **_grads((y,), (s["dy"],), ("dw", "dx"), s, ("w", "x"))}
        y, h = fw.add_rms_norm(s["x"], s["r"], s["w"], scale=s["s"], eps=_EPS)
        if kind == "add_norm":
            return y, h
        got = _grads((y, h), (s["dy"], s["dh"]), ("dw", "dx", "dr", "ds"), s, ("w", "x", "r", "s"))
        return {"y": y.detach(), "dw": got.pop("dw"), "h": h.detach(), **got}
    if kind.startswith("gate_norm"):
        y = fw.gated_rms_norm(s["x"], s["z"], s["w"], eps=_EPS)
        if kind == "gate_norm":
            return y
        return {"y": y.detach(), **_grads((y,), (s["dy"],), ("dx", "dz", "dw"), s, ("x", "z", "w"))}
    args = (s["q"], s["k"], s["v"], s["g"])
    if kind == "attn_step":
        return fw.decay_attn_decode_step(*args, s["state"], scale=s["scale"], inplace=True, slots=s["slots"])
    if kind == "attn_packed":
        return fw.decay_attn_varlen(*args, s["cu"], scale=s["scale"], state_pool=s["state"], slots=s["slots"])
    o, final = fw.decay_attn(*args, initial_state=s["state"], scale=s["scale"])
    if kind == "attn":
        return o, final
    return {"o": o.detach(), "final": final.detach(),
            **_grads((o, final), (s["do"], s["dstate"]), ("dq", "dk", "dv", "dg", "dstate0"), s,
                     ("q", "k", "v", "g", "state"))}


def run(state):
    if own:
        return _own(state)
    return (_attn_plain if state["case"]["kind"].startswith("attn") else _norm_plain)(state)


# ---- what a pass cannot do without -----------------------------------------------------------------
def work(case):
    kind, E = case["kind"], _DT[case["io"]].itemsize
    train = kind.endswith("_train")
    if kind.startswith("add_norm"):
        v, par = case["R"] * case["D"], case["D"] * E * (1 + int(case["scale"] == "channel" and case["res"] != "none"))
        r = {"none": 0, "io": E, "fp32": 4}[case["res"]]
        if not train:  # x and r in, y and h out
            return {"bytes": v * (2 * E + 2 * r) + par, "flops": 6 * v}
        return {"bytes": v * (4 * E + 4 * r) + 2 * par, "flops": 20 * v}
    if kind.startswith("gate_norm"):
        v, par = case["R"] * case["H"] * case["D"], case["D"] * E
        if not train:
            return {"bytes": 3 * v * E + par, "flops": 12 * v}
        return {"bytes": 6 * v * E + 2 * par, "flops": 35 * v}
    H, Hk, Dk, Dv = (case[n] for n in ("H", "Hk", "Dk", "Dv"))
    if "lseed" in case:
        tok, nseq = sum(_lengths(case)), case["n"]
    else:
        tok, nseq = case["B"] * case.get("T", 1), case["B"]
    rows, gate = tok * (2 * Hk * Dk + 2 * H * Dv) * E, 4 * (tok * H if case["gate"] == "token" else H)
    state = 2 * nseq * H * Dk * Dv * 4
    if not train:  # q, k, v, g and the states in, o and the states out; a product to write and one to read
        return {"bytes": rows + gate + state, "flops": 5 * tok * H * Dk * Dv}
    return {"bytes": 2 * (rows + gate + state), "flops": 20 * tok * H * Dk * Dv}


# ---- 64-bit results ---------------------------------------------------------------------------------
def _head64(q, k, v, g, scale, h0):
    """One head by the definition's closed form: q, k [T, Dk], v [T, Dv], g [T] -> (o, last state)."""
    G = g.cumsum(0)
    D = (G[:, None] - G[None, :]).tril()
    o = ((scale * (q @ k.T)) * torch.exp(D)).tril() @ v + scale * torch.exp(G)[:, None] * (q @ h0)
    return o, torch.exp(G[-1]) * h0 + (k * torch.exp(G[-1] - G)[:, None]).T @ v


def _attn64(q, k, v, g, scale, h0):
    """[T, heads, *] of one sequence, h0 [H, Dk, Dv]."""
    H, per = v.shape[1], v.shape[1] // q.shape[1]
    got = [_head64(q[:, h // per], k[:, h // per], v[:, h], g[h].expand(v.shape[0]) if g.dim() == 1 else g[:, h], scale,
                   h0[h]) for h in range(H)]
    return torch.stack([o for o, _ in got], 1), torch.stack([f for _, f in got])


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    train = kind.endswith("_train")
    d = {k: v.detach().double().requires_grad_(train) if torch.is_tensor(v) and v.is_floating_point() else v
         for k, v in s.items()}
    up = lambda *names: tuple(s[n].double() for n in names)  # noqa: E731
    if kind.startswith("add_norm"):
        norm = lambda h: h / torch.sqrt((h**2).mean(-1, keepdim=True) + _EPS) * d["w"]  # noqa: E731
        if s["r"] is None:
            y = norm(d["x"])
            if not train:
                return y
            return {"y": y.detach(), **_grads((y,), up("dy"), ("dw", "dx"), d, ("w", "x"))}
        h = d["r"] + d["x"] * (1.0 if s["s"] is None else d["s"])
        kept = h + (h.detach().to(s["r"].dtype).double() - h.detach())  # rounded, with the gradient passing
        y = norm(kept)
        if not train:
            return y, kept
        got = _grads((y, kept), up("dy", "dh"), ("dw", "dx", "dr", "ds"), d, ("w", "x", "r", "s"))
        return {"y": y.detach(), "dw": got.pop("dw"), "h": kept.detach(), **got}
    if kind.startswith("gate_norm"):
        y = d["x"] / torch.sqrt((d["x"]**2).mean(-1, keepdim=True) + _EPS) * d["w"] * d["z"] / (1 + torch.exp(-d["z"]))
        if not train:
            return y
        return {"y": y.detach(), **_grads((y,), up("dy"), ("dx", "dz", "dw"), d, ("x", "z", "w"))}
    args = [d[n] for n in ("q", "k", "v")]
    gates = lambda pick: d["g"] if d["g"].dim() == 1 else pick(d["g"])  # noqa: E731
    if "slots" in s:
        cu = s["cu"].tolist() if "cu" in s else list(range(case["B"] + 1))
        if kind == "attn_packed" and max(s["lens"]) > 16384:
            return None
        o = torch.empty_like(d["v"])
        if kind == "attn_step":
            per, rows = case["H"] // case["Hk"], s["slots"].long()
            q, k = (x.repeat_interleave(per, 1) for x in args[:2])
            h = torch.exp(d["g"])[..., None, None] * d["state"][rows] + torch.einsum("bhk,bhv->bhkv", k, d["v"])
            d["state"][rows] = h
            return s["scale"] * torch.einsum("bhk,bhkv->bhv", q, h), d["state"]
        for i, r in enumerate(s["slots"].tolist()):
            cut = slice(cu[i], cu[i + 1])
            o[cut], d["state"][r] = _attn64(*(x[cut] for x in args), gates(lambda x: x[cut]), s["scale"],
                                            d["state"][r].clone())
        return o, d["state"]
    got = [_attn64(*(x[b] for x in args), gates(lambda x: x[b]), s["scale"], d["state"][b]) for b in range(case["B"])]
    o, final = torch.stack([o for o, _ in got]), torch.stack([f for _, f in got])
    if not train:
        return o, final
    return {"o": o.detach(), "final": final.detach(),
            **_grads((o, final), up("do", "dstate"), ("dq", "dk", "dv", "dg", "dstate0"), d,
                     ("q", "k", "v", "g", "state"))}
