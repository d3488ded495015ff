"""Decay attention on MI355X: linear attention whose state decays by one factor per head and token, for training,
prompts, packed prompts and single tokens.  No reference counterpart: it stands beside GLA, whose decays are per key
dim, as the member with one decay a head, which needs no factor on every element of q and k.

    S_t = e^{g_t} S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t

Layouts: q, k [B, T, Hk, Dk], v [B, T, H, Dv] (packed: [N, heads, dim] or [1, N, heads, dim]) with any strides (the
innermost is made 1 by a copy where it is not), one dtype of float32, bfloat16 and float16; H is a multiple of Hk, and
H / Hk consecutive heads of v share one of q and k.  g: log-decays [B, T, H] in that dtype or float32, or [H]: one
constant per head.  A log-decay above 0 counts as 0 (its gradient is 0 then), -inf forgets.  Dk is at most 128, Dv
at most 16384.  States are float32 [B, H, Dk, Dv].  Sums and states are float32, outputs are rounded once.  Values
are expected to be finite: one that is not reaches the outputs of the other tokens of its block of 32 (gradients of
bfloat16: 64) in the same sequence and head, earlier ones among them, and all later ones; other sequences and heads
it does not reach. Tensors are on one HIP device; there is no CPU path and no forward-mode derivative.
"""

from __future__ import annotations

import torch

from ._lib import call_on, dtype_code, plan_on, ptr, strides
from .ssm import _cu, _needs_grad, _no_grad_path, _one_device, _slots

__all__ = ["decay_attn", "decay_attn_varlen", "decay_attn_decode_step"]

MAX_KEY_DIM, MAX_VALUE_DIM = 128, 16384


def _rows(x):
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _check(q, k, v, g):
    """(H, Hk, Dk, Dv) of a call with token tensors [*lead, heads, dim]."""
    _one_device(q, k, v, g)
    dtype_code(q)
    lead = q.shape[:-2]
    if k.shape != q.shape or v.dim() != q.dim() or v.shape[:-2] != lead:
        raise ValueError(f"k must have q's shape {tuple(q.shape)} and v its leading dims")
    Hk, Dk = q.shape[-2:]
    H, Dv = v.shape[-2:]
    if Hk < 1 or H < 1 or H % Hk:
        raise ValueError(f"{Hk} heads of q and k do not divide {H} heads of v")
    if H >= 1 << 16:
        raise ValueError("fewer than 65536 heads are supported")
    if not 1 <= Dk <= MAX_KEY_DIM or not 1 <= Dv <= MAX_VALUE_DIM:
        raise ValueError(f"head dims {Dk}, {Dv} are not supported (key dims up to {MAX_KEY_DIM}, value dims up to "
                         f"{MAX_VALUE_DIM})")
    if tuple(g.shape) not in ((*lead, H), (H,)):
        raise ValueError(f"g must be {[*lead, H]} or [{H}]")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("q, k and v must share one dtype")
    if g.dtype not in (q.dtype, torch.float32):
        raise TypeError("g must have q's dtype or float32")
    return H, Hk, Dk, Dv


def _head_strides(x, gate=None):
    """Strides up to the heads; of a gate [H] zeros in front of its own."""
    if gate is None:
        return x.stride()[:-1]
    return x.stride() if x.dim() == gate else (*(0,) * (gate - 1), *x.stride())


def _out(out, v):
    if out is None:
        return torch.empty(v.shape, device=v.device, dtype=v.dtype)
    if out.shape != v.shape or out.dtype != v.dtype:
        raise ValueError(f"out must be {tuple(v.shape)} of {v.dtype}")
    _one_device(v, out)
    span, apart = v.shape[-1], v.shape[-1] < 2 or out.stride(-1) == 1
    for s, n in sorted((s, n) for s, n in zip(out.stride()[:-1], v.shape[:-1]) if n > 1):
        apart = apart and s >= span  # past all that the dims of smaller strides reach
        span += (n - 1) * s
    if not apart and out.numel():
        raise ValueError("out needs a unit innermost stride and rows that do not overlap")
    return out


def _initial(s0, like, shape):
    if s0 is None:
        return None
    _one_device(like, s0)
    if tuple(s0.shape) != shape:
        raise ValueError(f"initial_state must be {list(shape)}")
    return s0.to(torch.float32).contiguous()


def _attn(q, k, v, g, scale, s0, out, flags=0):
    """(o, final state, workspace or None) of a dense call with B, T > 0."""
    B, T, H, Dv = v.shape
    Hk, Dk = q.shape[2:]
    q, k, v = _rows(q), _rows(k), _rows(v)
    o = _out(out, v)
    fin = torch.empty(B, H, Dk, Dv, device=q.device, dtype=torch.float32)
    wsb = plan_on(q, "triune_hip_decay_attn_workspace_size", B, T, H, Hk, Dk, Dv, flags)
    ws = torch.empty(wsb, device=q.device, dtype=torch.uint8) if wsb else None
    st = strides(*(_head_strides(x) for x in (q, k, v)), _head_strides(g, 3), _head_strides(o))
    call_on(q, "triune_hip_decay_attn", ptr(q), ptr(k), ptr(v), ptr(g), dtype_code(q), dtype_code(g), st, scale, ptr(s0),
            ptr(o), ptr(fin), B, T, H, Hk, Dk, Dv, flags, ptr(ws), wsb)
    return o, fin, ws


def _no_tokens(q, H, Dv, s0):
    """The final state of a call without tokens or sequences."""
    if s0 is None:
        return torch.zeros(q.shape[0], H, q.shape[-1], Dv, device=q.device, dtype=torch.float32)
    return s0.to(torch.float32).clone()


def _attn_bwd(q, k, v, g, scale, s0, do, dfin, want_s0, flags=0, kept=None):
    B, T, H, Dv = v.shape
    Hk, Dk = q.shape[2:]
    dev, f32 = q.device, torch.float32
    q, k, v = _rows(q), _rows(k), _rows(v)
    do = torch.zeros(B, T, H, Dv, device=dev, dtype=q.dtype) if do is None else _rows(do.to(q.dtype))
    dfin = None if dfin is None else dfin.to(f32).contiguous()
    dq, dk = (torch.empty(B, T, Hk, Dk, device=dev, dtype=q.dtype) for _ in range(2))
    dv = torch.empty(B, T, H, Dv, device=dev, dtype=q.dtype)
    dg = torch.empty(g.shape, device=dev, dtype=g.dtype)
    ds0 = torch.empty(B, H, Dk, Dv, device=dev, dtype=f32) if want_s0 else None
    head = int(g.dim() == 1)
    wsb = plan_on(q, "triune_hip_decay_attn_bwd_workspace_size", B, T, H, Hk, Dk, Dv, dtype_code(q), head, flags)
    wsb -= 0 if kept is None else kept.numel()  # the forward's end states
    ws = torch.empty(wsb, device=dev, dtype=torch.uint8)
    st = strides(*(_head_strides(x) for x in (q, k, v)), _head_strides(g, 3), _head_strides(do))
    call_on(q, "triune_hip_decay_attn_bwd", ptr(q), ptr(k), ptr(v), ptr(g), ptr(do), dtype_code(q), dtype_code(g), st, scale,
            ptr(s0), ptr(dfin), ptr(dq), ptr(dk), ptr(dv), ptr(dg), head, ptr(ds0), B, T, H, Hk, Dk, Dv, flags, ptr(kept),
            0 if kept is None else kept.numel(), ptr(ws), wsb)
    return dq, dk, dv, dg, ds0


class _DecayAttn(torch.autograd.Function):
    """decay_attn with gradients.  The forward keeps the states of its segments (none of short calls); the backward forms
    those of every 64th token (32nd of float32 and float16) from them, as scratch."""

    @staticmethod
    def forward(ctx, q, k, v, g, s0, scale):
        s0f = None if s0 is None else s0.to(torch.float32).contiguous()
        if q.shape[0] == 0 or q.shape[1] == 0:
            o, fin, kept = torch.empty(v.shape, device=v.device, dtype=v.dtype), _no_tokens(q, *v.shape[2:], s0f), None
        else:
            o, fin, kept = _attn(q, k, v, g, scale, s0f, None)
        ctx.save_for_backward(q, k, v, g, s0, kept)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, fin

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, dfin):
        q, k, v, g, s0, kept = ctx.saved_tensors
        if do is None and dfin is None:
            return (None,) * 6
        want = s0 is not None and ctx.needs_input_grad[4]
        if q.shape[0] == 0 or q.shape[1] == 0:  # no tokens: the final state is the initial state
            zero = [torch.zeros_like(t) for t in (q, k, v, g)]
            return (*zero, dfin.to(s0.dtype) if want and dfin is not None else None, None)
        s0f = None if s0 is None else s0.to(torch.float32).contiguous()
        dq, dk, dv, dg, ds0 = _attn_bwd(q, k, v, g, ctx.scale, s0f, do, dfin, want, kept=kept)
        return dq, dk, dv, dg, ds0.to(s0.dtype) if want else None, None


def decay_attn(q, k, v, g, initial_state=None, scale=1.0, out=None):
    """Decay attention over [B, T, heads, dim] prompts.

    q, k: [B, T, Hk, Dk]; v: [B, T, H, Dv]; g: [B, T, H] or [H]; initial_state: [B, H, Dk, Dv] or None (zeros); out:
    optional [B, T, H, Dv] buffer in q's dtype that overlaps no input, for calls without gradients.  Returns (o
    [B, T, H, Dv] in q's dtype, final state float32 [B, H, Dk, Dv]).

    Differentiable in every tensor argument (once): the gradients come from triune_hip_decay_attn_bwd and do not depend
    on timing."""
    if q.dim() != 4:
        raise ValueError("q must be [B, T, heads, dim]")
    H, Hk, Dk, Dv = _check(q, k, v, g)
    B, T = q.shape[:2]
    if _needs_grad(q, k, v, g, initial_state):
        if out is not None:
            raise ValueError("out is for calls without gradients")
        _initial(initial_state, q, (B, H, Dk, Dv))
        return _DecayAttn.apply(q, k, v, g, initial_state, float(scale))
    s0 = _initial(initial_state, q, (B, H, Dk, Dv))
    if B == 0 or T == 0:  # nothing to read: the final state is the initial state
        return _out(out, v), _no_tokens(q, H, Dv, s0)
    return _attn(q, k, v, g, float(scale), s0, out)[:2]


def decay_attn_varlen(q, k, v, g, cu_seqlens, initial_state=None, scale=1.0, out=None, *, state_pool=None, slots=None):
    """decay_attn over packed ragged prompts, without gradients: q, k [N, Hk, Dk] or [1, N, Hk, Dk], v likewise, g [N, H],
    [1, N, H] or [H], cu_seqlens int32 [n + 1] ascending offsets (device or host); initial_state [n, H, Dk, Dv] or
    None.  Returns (o like v, final states float32 [n, H, Dk, Dv]).  Rows of o outside the sequences are not written.

    With state_pool (contiguous float32 [rows, H, Dk, Dv]) and slots (int32 [n], distinct), sequence i starts from
    state_pool[slots[i]] and leaves its final state there, and the second item returned is state_pool; a slot
    outside the pool (-1 for a padded row) starts from zero and keeps nothing."""
    _no_grad_path("decay_attn_varlen", q, k, v, g, initial_state, state_pool)
    lead1 = q.dim() == 4
    if lead1:
        if q.shape[0] != 1:
            raise ValueError("packed varlen tensors have batch size 1")
        if any(t.dim() != 4 or t.shape[0] != 1 for t in (k, v) if t is not None) or (
                out is not None and (out.dim() != 4 or out.shape[0] != 1)) or (g.dim() > 1 and g.shape[0] != 1):
            raise ValueError("packed varlen tensors must all have the leading 1")
        q, k, v, g = q[0], k[0], v[0], g if g.dim() == 1 else g[0]
        out = None if out is None else out[0]
    if q.dim() != 3:
        raise ValueError("q must be [N, heads, dim] or [1, N, heads, dim]")
    H, Hk, Dk, Dv = _check(q, k, v, g)
    _one_device(q, initial_state, out, state_pool)
    total = q.shape[0]
    cu = _cu(cu_seqlens, q.device)
    n = cu.numel() - 1
    if state_pool is not None:
        if initial_state is not None:
            raise ValueError("pass either initial_state or state_pool, not both")
        if slots is None:
            raise ValueError("state_pool needs slots")
        if (state_pool.dtype != torch.float32 or not state_pool.is_contiguous() or state_pool.dim() != 4 or
                tuple(state_pool.shape[1:]) != (H, Dk, Dv)):
            raise ValueError(f"state_pool must be a contiguous float32 tensor of rows {(H, Dk, Dv)}")
        s0 = fin = state_pool
    else:
        if slots is not None:
            raise ValueError("slots needs state_pool")
        s0 = _initial(initial_state, q, (n, H, Dk, Dv))
        fin = torch.empty(n, H, Dk, Dv, device=q.device, dtype=torch.float32)
    sl = _slots(slots, n, q.device)
    o = _out(out, v)
    if total == 0:
        if state_pool is None:
            fin.zero_() if s0 is None else fin.copy_(s0)
    elif n > 0:
        q, k, v = _rows(q), _rows(k), _rows(v)
        wsb = plan_on(q, "triune_hip_decay_attn_varlen_workspace_size", n, total, H, Hk, Dk, Dv, 0)
        ws = torch.empty(wsb, device=q.device, dtype=torch.uint8) if wsb else None
        st = strides(*(_head_strides(x) for x in (q, k, v)), _head_strides(g, 2), _head_strides(o))
        call_on(q, "triune_hip_decay_attn_varlen", ptr(q), ptr(k), ptr(v), ptr(g), dtype_code(q), dtype_code(g), st,
                float(scale), ptr(cu), n, total, ptr(s0), ptr(fin), ptr(sl), fin.shape[0], ptr(o), H, Hk, Dk, Dv, 0,
                ptr(ws), wsb)
    return (o.unsqueeze(0) if lead1 else o), fin


def decay_attn_decode_step(q, k, v, g, state, scale=1.0, out=None, *, inplace=False, slots=None):
    """One token of decay_attn for each of a batch of sequences, without gradients: q, k [B, Hk, Dk] or [B, 1, Hk, Dk], v
    likewise, g [B, H], [B, 1, H] or [H]; state [B, H, Dk, Dv], or a pool [rows, H, Dk, Dv] addressed by int32 slots
    [B] (distinct; a slot outside the pool, -1 for a padded row, reads and writes no state and gets zero outputs).
    Returns (o like v, state): a new state, or with inplace=True the state tensor itself (contiguous float32),
    updated."""
    _no_grad_path("decay_attn_decode_step", q, k, v, g, state)
    token = q.dim() == 4
    if token:
        if any(t.dim() != 4 or t.shape[1] != 1 for t in (q, k, v)) or (
                out is not None and (out.dim() != 4 or out.shape[1] != 1)) or (
                g.dim() != 1 and (g.dim() != 3 or g.shape[1] != 1)):
            raise ValueError("decode step takes one token per sequence (T == 1)")
        q, k, v, g = q[:, 0], k[:, 0], v[:, 0], g if g.dim() == 1 else g[:, 0]
        out = None if out is None else out[:, 0]
    if q.dim() != 3:
        raise ValueError("q must be [B, heads, dim] or [B, 1, heads, dim]")
    H, Hk, Dk, Dv = _check(q, k, v, g)
    _one_device(q, state, out)
    n = q.shape[0]
    if state.dim() != 4 or tuple(state.shape[1:]) != (H, Dk, Dv):
        raise ValueError(f"state must hold rows {(H, Dk, Dv)}")
    if slots is None and state.shape[0] != n:
        raise ValueError(f"state has {state.shape[0]} rows for a batch of {n} (pass slots to address a pool)")
    if inplace:
        if state.dtype != torch.float32 or not state.is_contiguous():
            raise ValueError("inplace decode needs a contiguous float32 state")
        s_in = s_out = state
    else:
        s_in = state.to(torch.float32).contiguous()
        # with slots only the addressed rows are written: the others keep their input values
        s_out = torch.empty_like(s_in) if slots is None else s_in.clone()
    sl = _slots(slots, n, q.device)
    o = _out(out, v)
    if n > 0:
        q, k, v = _rows(q), _rows(k), _rows(v)
        st = strides(*(_head_strides(x) for x in (q, k, v)), _head_strides(g, 2), _head_strides(o))
        call_on(q, "triune_hip_decay_attn_decode_step", ptr(q), ptr(k), ptr(v), ptr(g), dtype_code(q), dtype_code(g), st,
                float(scale), ptr(s_in), ptr(s_out), ptr(sl), s_in.shape[0], ptr(o), n, H, Hk, Dk, Dv)
    return (o.unsqueeze(1) if token else o), s_out
