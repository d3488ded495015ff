"""State space layer operators on MI355X: the selective scan and the short causal convolution in front
of it, for training, prompts, packed prompts and single tokens.  No reference counterpart: they
stand beside the GLA and Gated DeltaNet operators as the diagonal member of the family, where every
(channel, state) has a decay of its own and channels share B and C.

Scan, per channel d with states n:
    dt = softplus(delta + delta_bias);  h <- exp(dt A) h + dt u B;  y = (sum_n C h + D u) silu(z)

Layouts: token tensors [B, T, channels] (packed: [N, channels] or [1, N, channels]) with any strides
(the innermost is made 1 by a copy where it is not), one dtype of float32, bfloat16 and float16;
parameters A, D and delta_bias in float32; scan states float32 [B, channels, N], convolution states
[B, W - 1, channels] in x's dtype (the last W - 1 inputs, oldest first).  Everything that the kernels sum or
carry is float32; outputs are rounded once.  A may be positive and dt below 0 (modes that grow), but one token's
exp(dt A) has to be a float32 number; A of -inf forgets at every step above 0.  Tensors are on one HIP device;
there is no CPU path and no forward-mode derivative.
"""

from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from ._lib import call_on, dtype_code, plan_on, ptr, strides

__all__ = [
    "ssm_scan",
    "ssm_scan_varlen",
    "ssm_decode_step",
    "short_conv",
    "short_conv_varlen",
    "short_conv_decode_step",
]

MAX_STATES = 64


def _kept_every(N):
    """Tokens between the states that the forward keeps for the backward."""
    return 32 if N <= 32 else 16


def _one_device(first, *rest):
    if not first.is_cuda:
        raise ValueError("triune_amd kernels take HIP device tensors (device='cuda'); got a CPU tensor")
    dev = first.get_device()
    for t in rest:
        if t is not None and t.get_device() != dev:
            raise ValueError("all tensors must be on one HIP device")


_MAX_TOKEN_STRIDE = 1 << 22  # the scan's kernels address a tile's rows in 32 bits


def _rows(x, tok=None):
    """x with a unit innermost stride, and a stride of its token dim tok that the kernels take (a copy
    where it has not)."""
    if x.stride(-1) == 1 and (tok is None or x.stride(tok) < _MAX_TOKEN_STRIDE or x.shape[tok] == 1):
        return x
    if tok is not None and x.shape[tok] != 1 and math.prod(x.shape[tok + 1:]) >= _MAX_TOKEN_STRIDE:
        raise ValueError(f"tokens of {tuple(x.shape[tok + 1:])} are too wide: they need below {_MAX_TOKEN_STRIDE} values")
    return x.contiguous()


def _lead(x, tok):
    """The strides up to x's token dim; 0 for a single token's."""
    st = x.stride()[:tok + 1]
    return st if x.shape[tok] != 1 else (*st[:tok], 0)


def _lead_out(y, tok):
    """The same of an output, whose rows are never on top of each other."""
    st = y.stride()[:tok + 1]
    return st if y.shape[tok] != 1 else (*st[:tok], y.shape[-1])


def _needs_grad(*ts) -> bool:
    """Whether a call on these is recorded.  Refuses forward-mode duals: they do not require a gradient, and
    their tangents would be dropped."""
    if forward_ad._current_level >= 0:  # inside dual_level()
        for t in ts:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError("there is no forward-mode derivative: an input carries a tangent")
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


def _no_grad_path(what, *ts):
    if _needs_grad(*ts):
        raise ValueError(f"{what} has no gradient: call it under torch.no_grad()")


def _out(out, shape, dtype, like, tok=None):
    if out is None:
        return torch.empty(shape, device=like.device, dtype=dtype)
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype:
        raise ValueError(f"out must be {tuple(shape)} of {dtype}")
    span, apart = shape[-1], shape[-1] < 2 or out.stride(-1) == 1
    for s, n in sorted((s, n) for s, n in zip(out.stride()[:-1], shape[:-1]) if n > 1):
        apart = apart and s >= span  # past all that the dims of smaller strides reach
        span += (n - 1) * s
    if not apart and out.numel():
        raise ValueError("out needs a unit innermost stride and rows that do not overlap")
    if tok is not None and out.shape[tok] > 1 and out.stride(tok) >= _MAX_TOKEN_STRIDE:
        raise ValueError(f"out's token stride must be below {_MAX_TOKEN_STRIDE}")
    return out


_INTEGERS = (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8)


def _slots(slots, n, dev):
    if slots is None:
        return None
    if slots.numel() != n or slots.dim() != 1:
        raise ValueError(f"slots must hold one index for each of the {n} rows")
    if slots.dtype != torch.int32 or slots.device != dev:
        if slots.dtype not in _INTEGERS:
            raise TypeError(f"slots must be int32 or another of {_INTEGERS}, not {slots.dtype}")
        if slots.dtype == torch.int64:  # past 32 bits is outside every pool, not the row of the low half
            slots = slots.clamp(-1, 2**31 - 1)
        slots = slots.to(device=dev, dtype=torch.int32)
    return slots.contiguous()


def _cu(cu_seqlens, dev):
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1 or cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise ValueError("cu_seqlens must be int32 offsets [n + 1]")
    if cu_seqlens.dtype == torch.int64:  # past 32 bits is behind every row, as for offsets that fit
        cu_seqlens = cu_seqlens.clamp(0, 2**31 - 1)
    return cu_seqlens.to(device=dev, dtype=torch.int32).contiguous()


def _pool(state_pool, slots, initial_state, row_shape, dtype):
    if initial_state is not None:
        raise ValueError("pass either initial_state or state_pool, not both")
    if slots is None:
        raise ValueError("state_pool needs slots")
    if (state_pool.dtype != dtype or not state_pool.is_contiguous() or
            tuple(state_pool.shape[1:]) != row_shape or state_pool.dim() != 3):
        raise ValueError(f"state_pool must be a contiguous {dtype} tensor of rows {row_shape}")


# ---------------------------------------------------------------------------------------
# Selective scan
# ---------------------------------------------------------------------------------------


def _check_scan(u, delta, A, B, C, D, z, delta_bias):
    """(Dm, G, N) of a call with token tensors [*lead, channels]."""
    _one_device(u, delta, A, B, C, D, z, delta_bias)
    dtype_code(u)
    shape, dt = u.shape, u.dtype
    Dm = shape[-1]
    if delta.shape != shape or (z is not None and z.shape != shape):
        raise ValueError(f"delta and z must have u's shape {tuple(shape)}")
    if A.dim() != 2 or A.shape[0] != Dm:
        raise ValueError(f"A must be [{Dm}, N]")
    N = A.shape[1]
    if not 1 <= N <= MAX_STATES or Dm < 1:
        raise ValueError(f"{N} states per channel are not supported (1 to {MAX_STATES})")
    lead, bs = len(shape) - 1, B.shape
    if bs != C.shape or bs[:lead] != shape[:lead] or bs[-1] != N or len(bs) not in (lead + 1, lead + 2):
        raise ValueError(f"B and C must be {[*shape[:-1], N]} or [..., groups, {N}]")
    G = bs[-2] if len(bs) == lead + 2 else 1
    if G < 1 or Dm % G:
        raise ValueError(f"{G} groups do not divide {Dm} channels")
    if delta.dtype != dt or B.dtype != dt or C.dtype != dt or (z is not None and z.dtype != dt):
        raise TypeError("u, delta, z, B and C must share one dtype")
    f32 = torch.float32
    if A.dtype != f32 or (D is not None and D.dtype != f32) or (delta_bias is not None and delta_bias.dtype != f32):
        raise TypeError("A, D and delta_bias must be float32")
    for name, t in (("D", D), ("delta_bias", delta_bias)):
        if t is not None and (t.dim() != 1 or t.shape[0] != Dm):
            raise ValueError(f"{name} must be [{Dm}]")
    return Dm, G, N


def _c(x):
    return None if x is None else x.contiguous()


def _group_strides(x, lead):
    """Strides of B or C in front of its states: (lead ..., group)."""
    return (*_lead(x, lead - 1), x.stride(lead) if x.dim() == lead + 2 else 0)


def _scan(u, delta, A, B, C, D, z, bias, softplus, s0, out, keep, flags=0):
    """(y, final state, kept states or None) of a dense call with B, T > 0."""
    Bn, T, Dm = u.shape
    N = A.shape[1]
    G = B.shape[2] if B.dim() == 4 else 1
    u, delta, B, C = _rows(u, 1), _rows(delta, 1), _rows(B, 1), _rows(C, 1)
    z = None if z is None else _rows(z, 1)
    A, D, bias = A.contiguous(), _c(D), _c(bias)
    if s0 is not None:
        s0 = s0.to(torch.float32).contiguous()
    y = _out(out, u.shape, u.dtype, u, 1)
    fin = torch.empty(Bn, Dm, N, device=u.device, dtype=torch.float32)
    kept = None
    if keep:
        kept = torch.empty(Bn, -(-T // _kept_every(N)), N, Dm, device=u.device, dtype=torch.float32)
    wsb = plan_on(u, "triune_hip_ssm_scan_workspace_size", Bn, T, Dm, G, N, flags)
    ws = torch.empty(wsb, device=u.device, dtype=torch.uint8) if wsb else None
    st = strides(_lead(u, 1), _lead(delta, 1), (0, 0) if z is None else _lead(z, 1), _lead_out(y, 1),
                 _group_strides(B, 2), _group_strides(C, 2))
    call_on(u, "triune_hip_ssm_scan", ptr(u), ptr(delta), ptr(z), ptr(B), ptr(C), ptr(A), ptr(D), ptr(bias),
            dtype_code(u), st, int(softplus), ptr(s0), ptr(y), ptr(fin), ptr(kept), Bn, T, Dm, G, N, flags, ptr(ws),
            wsb)
    return y, fin, kept


def _scan_bwd(u, delta, A, B, C, D, z, bias, softplus, kept, dy, dfin, want_s0, flags=0):
    Bn, T, Dm = u.shape
    N = A.shape[1]
    G = B.shape[2] if B.dim() == 4 else 1
    dev, f32 = u.device, torch.float32
    u, delta, Br, Cr = _rows(u, 1), _rows(delta, 1), _rows(B, 1), _rows(C, 1)
    zr = None if z is None else _rows(z, 1)
    Ac, Dc, bc = A.contiguous(), _c(D), _c(bias)
    dy = torch.zeros(Bn, T, Dm, device=dev, dtype=u.dtype) if dy is None else _rows(dy.to(u.dtype), 1)
    dfin = None if dfin is None else dfin.to(f32).contiguous()
    du, dd = (torch.empty(Bn, T, Dm, device=dev, dtype=u.dtype) for _ in range(2))
    dz = None if z is None else torch.empty_like(du)
    dB, dC = (torch.empty(B.shape, device=dev, dtype=u.dtype) for _ in range(2))
    dA = torch.empty(Dm, N, device=dev, dtype=f32)
    dD = None if D is None else torch.empty(Dm, device=dev, dtype=f32)
    db = None if bias is None else torch.empty(Dm, device=dev, dtype=f32)
    ds0 = torch.empty(Bn, Dm, N, device=dev, dtype=f32) if want_s0 else None
    wsb = plan_on(u, "triune_hip_ssm_bwd_workspace_size", Bn, T, Dm, G, N, flags)
    ws = torch.empty(wsb, device=dev, dtype=torch.uint8)
    st = strides(_lead(u, 1), _lead(delta, 1), (0, 0) if zr is None else _lead(zr, 1), _lead(dy, 1),
                 _group_strides(Br, 2), _group_strides(Cr, 2))
    call_on(u, "triune_hip_ssm_bwd", ptr(u), ptr(delta), ptr(zr), ptr(Br), ptr(Cr), ptr(Ac), ptr(Dc), ptr(bc), ptr(dy),
            dtype_code(u), st, int(softplus), ptr(kept), ptr(dfin), ptr(du), ptr(dd), ptr(dz), ptr(dB), ptr(dC),
            ptr(dA), ptr(dD), ptr(db), ptr(ds0), Bn, T, Dm, G, N, flags, ptr(ws), wsb)
    return du, dd, dA, dB, dC, dD, dz, db, ds0


def _no_tokens(u, N, s0):
    """The final state of a call without tokens or sequences."""
    if s0 is None:
        return torch.zeros(u.shape[0], u.shape[-1], N, device=u.device, dtype=torch.float32)
    return s0.to(torch.float32).clone()


class _SsmScan(torch.autograd.Function):
    """ssm_scan with gradients.  The forward keeps the state of every 32nd token (N / 8 bytes per token
    and channel: 2 beside the 8 of u, delta, z and y in 16 bits at N = 16) as a saved tensor."""

    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, bias, s0, softplus):
        if u.shape[0] == 0 or u.shape[1] == 0:
            y, fin, kept = torch.empty_like(u), _no_tokens(u, A.shape[1], s0), None
        else:
            y, fin, kept = _scan(u, delta, A, B, C, D, z, bias, softplus, s0, None, True)
        ctx.save_for_backward(u, delta, A, B, C, D, z, bias, kept)
        ctx.softplus, ctx.s0_dtype = softplus, None if s0 is None else s0.dtype
        ctx.set_materialize_grads(False)
        return y, fin

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dfin):
        u, delta, A, B, C, D, z, bias, kept = ctx.saved_tensors
        if dy is None and dfin is None:
            return (None,) * 10
        want = ctx.s0_dtype is not None and ctx.needs_input_grad[8]
        if kept is None:  # no tokens: the final state is the initial state
            zero = [None if t is None else torch.zeros_like(t) for t in (u, delta, A, B, C, D, z, bias)]
            return (*zero, dfin.to(ctx.s0_dtype) if want and dfin is not None else None, None)
        du, dd, dA, dB, dC, dD, dz, db, ds0 = _scan_bwd(u, delta, A, B, C, D, z, bias, ctx.softplus, kept, dy, dfin,
                                                        want)
        return du, dd, dA, dB, dC, dD, dz, db, ds0.to(ctx.s0_dtype) if want else None, None


def ssm_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=True, initial_state=None, out=None):
    """Selective state space scan over [B, T, channels] prompts.

    u, delta, z: [B, T, Dm] (z: the gate, or None); A: float32 [Dm, N]; B, C: [B, T, N], or
    [B, T, G, N] where G groups of Dm / G consecutive channels share theirs (G N below 2^22 where T > 1);
    D, delta_bias: float32 [Dm] or None; N at most 64.  dt is softplus(delta + delta_bias), or delta + delta_bias
    without delta_softplus.  initial_state: [B, Dm, N] or None (zeros).  out: optional [B, T, Dm] buffer
    in u's dtype that overlaps no input, for calls without gradients.  Returns (y [B, T, Dm] in u's
    dtype, final state float32 [B, Dm, N]).

    Differentiable in every tensor argument (once): the gradients come from
    triune_hip_ssm_bwd and do not depend on timing."""
    if u.dim() != 3:
        raise ValueError("u must be [B, T, channels]")
    Dm, G, N = _check_scan(u, delta, A, B, C, D, z, delta_bias)
    Bn, T, _ = u.shape
    if initial_state is not None:
        _one_device(u, initial_state)
        if tuple(initial_state.shape) != (Bn, Dm, N):
            raise ValueError(f"initial_state must be [{Bn}, {Dm}, {N}]")
    grad = _needs_grad(u, delta, A, B, C, D, z, delta_bias, initial_state)
    if grad and out is not None:
        raise ValueError("out is for calls without gradients")
    if out is not None:
        _one_device(u, out)
    if grad:
        return _SsmScan.apply(u, delta, A, B, C, D, z, delta_bias, initial_state, bool(delta_softplus))
    if Bn == 0 or T == 0:  # nothing to scan: the final state is the initial state
        return _out(out, u.shape, u.dtype, u), _no_tokens(u, N, initial_state)
    return _scan(u, delta, A, B, C, D, z, delta_bias, delta_softplus, initial_state, out, False)[:2]


def ssm_scan_varlen(u, delta, A, B, C, cu_seqlens, D=None, z=None, delta_bias=None, delta_softplus=True,
                    initial_state=None, out=None, *, state_pool=None, slots=None):
    """ssm_scan over packed ragged prompts, without gradients: u, delta, z [N, Dm] or [1, N, Dm], B, C
    [N, (G,) states] or [1, N, (G,) states], cu_seqlens int32 [n + 1] ascending offsets (device or
    host); initial_state [n, Dm, states] or None.  Returns (y like u, final states float32
    [n, Dm, states]).  Rows of y outside the sequences are not written.

    With state_pool (contiguous float32 [rows, Dm, states]) and slots (int32 [n], distinct),
    sequence i starts from state_pool[slots[i]] and leaves its final state there, and the second
    item returned is state_pool; a slot outside the pool (-1 for a padded row) starts from zero and
    keeps nothing."""
    _no_grad_path("ssm_scan_varlen", u, delta, A, B, C, D, z, delta_bias, initial_state, state_pool)
    lead1 = u.dim() == 3
    if lead1:
        if u.shape[0] != 1:
            raise ValueError("packed varlen tensors have batch size 1")
        if any(t is not None and (t.dim() < 3 or t.shape[0] != 1) for t in (delta, z, B, C, out)):
            raise ValueError("packed varlen tensors must all have the leading 1")
        u, delta, B, C = u[0], delta[0], B[0], C[0]
        z = None if z is None else z[0]
        out = None if out is None else out[0]
    if u.dim() != 2:
        raise ValueError("u must be [N, channels] or [1, N, channels]")
    Dm, G, N = _check_scan(u, delta, A, B, C, D, z, delta_bias)
    _one_device(u, initial_state, out, state_pool)
    total = u.shape[0]
    cu = _cu(cu_seqlens, u.device)
    n = cu.numel() - 1
    if state_pool is not None:
        _pool(state_pool, slots, initial_state, (Dm, N), torch.float32)
        s0 = fin = state_pool
    else:
        if slots is not None:
            raise ValueError("slots needs state_pool")
        if initial_state is not None and tuple(initial_state.shape) != (n, Dm, N):
            raise ValueError(f"initial_state must be [{n}, {Dm}, {N}]")
        s0 = None if initial_state is None else initial_state.to(torch.float32).contiguous()
        fin = torch.empty(n, Dm, N, device=u.device, dtype=torch.float32)
    sl = _slots(slots, n, u.device)
    y = _out(out, u.shape, u.dtype, u, 0)
    if total == 0:
        if state_pool is None:
            fin.zero_() if s0 is None else fin.copy_(s0)
    elif n > 0:
        u, delta, B, C = _rows(u, 0), _rows(delta, 0), _rows(B, 0), _rows(C, 0)
        z = None if z is None else _rows(z, 0)
        A, D, delta_bias = A.contiguous(), _c(D), _c(delta_bias)
        wsb = plan_on(u, "triune_hip_ssm_scan_varlen_workspace_size", n, total, Dm, G, N, 0)
        ws = torch.empty(wsb, device=u.device, dtype=torch.uint8) if wsb else None
        st = strides(_lead(u, 0), _lead(delta, 0), (0,) if z is None else _lead(z, 0), _lead_out(y, 0),
                     _group_strides(B, 1), _group_strides(C, 1))
        call_on(u, "triune_hip_ssm_scan_varlen", ptr(u), ptr(delta), ptr(z), ptr(B), ptr(C), ptr(A), ptr(D),
                ptr(delta_bias), dtype_code(u), st, int(delta_softplus), ptr(cu), n, total, ptr(s0), ptr(fin), ptr(sl),
                fin.shape[0], ptr(y), Dm, G, N, 0, ptr(ws), wsb)
    return (y.unsqueeze(0) if lead1 else y), fin


def _step_states(state, inplace, slots, B, dtype, row_shape):
    """(state in, state out) of a decode step."""
    if state.dim() != 3 or tuple(state.shape[1:]) != row_shape:
        raise ValueError(f"state must hold rows {row_shape}")
    if slots is None and state.shape[0] != B:
        raise ValueError(f"state has {state.shape[0]} rows for a batch of {B} (pass slots to address a pool)")
    if inplace:
        if state.dtype != dtype or not state.is_contiguous():
            raise ValueError(f"inplace decode needs a contiguous {dtype} state")
        return state, state
    s_in = state.to(dtype).contiguous()
    # with slots only the addressed rows are written: the others keep their input values
    return s_in, torch.empty_like(s_in) if slots is None else s_in.clone()


def ssm_decode_step(u, delta, A, B, C, state, D=None, z=None, delta_bias=None, delta_softplus=True, out=None, *,
                    inplace=False, slots=None):
    """One token of ssm_scan for each of a batch of sequences, without gradients: u, delta, z [B, Dm] or
    [B, 1, Dm], B, C [B, (G,) N] or [B, 1, (G,) N]; state [B, Dm, N], or a pool [rows, Dm, N]
    addressed by int32 slots [B] (distinct; a slot outside the pool, -1 for a padded row, reads and
    writes no state and gets zero outputs).  Returns (y like u, state): a new state, or with
    inplace=True the state tensor itself (contiguous float32), updated."""
    _no_grad_path("ssm_decode_step", u, delta, A, B, C, state, D, z, delta_bias)
    token = u.dim() == 3
    if token:
        if any(t is not None and (t.dim() < 3 or t.shape[1] != 1) for t in (u, delta, z, B, C, out)):
            raise ValueError("decode step takes one token per sequence (T == 1)")
        u, delta, B, C = u[:, 0], delta[:, 0], B[:, 0], C[:, 0]
        z = None if z is None else z[:, 0]
        out = None if out is None else out[:, 0]
    if u.dim() != 2:
        raise ValueError("u must be [B, channels] or [B, 1, channels]")
    Dm, G, N = _check_scan(u, delta, A, B, C, D, z, delta_bias)
    _one_device(u, state, out)
    n = u.shape[0]
    s_in, s_out = _step_states(state, inplace, slots, n, torch.float32, (Dm, N))
    sl = _slots(slots, n, u.device)
    y = _out(out, u.shape, u.dtype, u)
    if n > 0:
        u, delta, B, C = _rows(u), _rows(delta), _rows(B), _rows(C)
        z = None if z is None else _rows(z)
        A, D, delta_bias = A.contiguous(), _c(D), _c(delta_bias)
        st = strides(u.stride()[:1], delta.stride()[:1], (0,) if z is None else z.stride()[:1], y.stride()[:1],
                     _group_strides(B, 1), _group_strides(C, 1))
        call_on(u, "triune_hip_ssm_decode_step", ptr(u), ptr(delta), ptr(z), ptr(B), ptr(C), ptr(A), ptr(D),
                ptr(delta_bias), dtype_code(u), st, int(delta_softplus), ptr(s_in), ptr(s_out), ptr(sl),
                s_in.shape[0], ptr(y), n, Dm, G, N)
    return (y.unsqueeze(1) if token else y), s_out


# ---------------------------------------------------------------------------------------
# Short causal convolution
# ---------------------------------------------------------------------------------------


def _check_conv(x, weight, bias, activation):
    """(channels, taps, whether silu follows)."""
    _one_device(x, weight, bias)
    dtype_code(x)
    Dm = x.shape[-1]
    if weight.dim() != 2 or weight.shape[0] != Dm or not 2 <= weight.shape[1] <= 4 or Dm < 1:
        raise ValueError(f"weight must be [{Dm}, W] with 2 to 4 taps")
    if weight.dtype not in (x.dtype, torch.float32):
        raise TypeError("weight must have x's dtype or float32")
    if bias is not None and (tuple(bias.shape) != (Dm,) or bias.dtype != weight.dtype):
        raise ValueError(f"bias must be [{Dm}] of weight's dtype")
    if activation not in ("silu", None):
        raise ValueError("activation must be 'silu' or None")
    return Dm, weight.shape[1], activation == "silu"


def _conv(x, weight, bias, silu, s0, out):
    Bn, T, Dm = x.shape
    W = weight.shape[1]
    x, weight, bias = _rows(x), weight.contiguous(), _c(bias)
    s0 = None if s0 is None else s0.to(x.dtype).contiguous()
    y = _out(out, x.shape, x.dtype, x)
    fin = torch.empty(Bn, W - 1, Dm, device=x.device, dtype=x.dtype)
    call_on(x, "triune_hip_short_conv", ptr(x), ptr(weight), ptr(bias), dtype_code(x), dtype_code(weight),
            strides(x.stride()[:2], y.stride()[:2]), int(silu), ptr(s0), ptr(fin), ptr(y), Bn, T, Dm, W)
    return y, fin


def _no_conv_tokens(x, W, s0):
    """The final state of a call without tokens or sequences."""
    if s0 is None:
        return torch.zeros(x.shape[0], W - 1, x.shape[-1], device=x.device, dtype=x.dtype)
    return s0.to(x.dtype).clone()


class _ShortConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, s0, silu):
        if x.shape[0] == 0 or x.shape[1] == 0:
            y, fin = torch.empty_like(x), _no_conv_tokens(x, weight.shape[1], s0)
        else:
            y, fin = _conv(x, weight, bias, silu, s0, None)
        ctx.save_for_backward(x, weight, bias, s0)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return y, fin

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dfin):
        x, weight, bias, s0 = ctx.saved_tensors
        if dy is None and dfin is None:
            return (None,) * 5
        Bn, T, Dm = x.shape
        W = weight.shape[1]
        if Bn == 0 or T == 0:  # the final state is the initial state
            zero = [None if t is None else torch.zeros_like(t) for t in (x, weight, bias)]
            return (*zero, None if s0 is None or dfin is None else dfin.to(s0.dtype), None)
        dev = x.device
        xr, wc, bc = _rows(x), weight.contiguous(), _c(bias)
        dy = torch.zeros_like(xr) if dy is None else _rows(dy.to(x.dtype))
        dfin = None if dfin is None else dfin.to(x.dtype).contiguous()
        sc = None if s0 is None else s0.to(x.dtype).contiguous()
        dx = torch.empty(Bn, T, Dm, device=dev, dtype=x.dtype)
        dw = torch.empty(Dm, W, device=dev, dtype=weight.dtype) if ctx.needs_input_grad[1] else None
        db = torch.empty(Dm, device=dev, dtype=weight.dtype) if bias is not None and ctx.needs_input_grad[2] else None
        ds0 = torch.empty(Bn, W - 1, Dm, device=dev, dtype=x.dtype) if s0 is not None else None
        wsb = plan_on(x, "triune_hip_short_conv_bwd_workspace_size", Bn, T, Dm, W) if dw is not None or db is not None else 0
        ws = torch.empty(wsb, device=dev, dtype=torch.uint8) if wsb else None
        call_on(x, "triune_hip_short_conv_bwd", ptr(xr), ptr(wc), ptr(bc), ptr(dy), dtype_code(x), dtype_code(weight),
                strides(xr.stride()[:2], dy.stride()[:2]), int(ctx.silu), ptr(sc), ptr(dfin), ptr(dx), ptr(dw), ptr(db),
                ptr(ds0), Bn, T, Dm, W, ptr(ws), wsb)
        return dx, dw, db, None if ds0 is None else ds0.to(s0.dtype), None


def short_conv(x, weight, bias=None, initial_state=None, activation="silu", out=None):
    """Causal depthwise convolution of 2 to 4 taps over [B, T, channels]:
    y_t = silu(bias + sum_j weight[:, j] x_{t - W + 1 + j}), without silu when activation is None.

    weight: [channels, W] and bias: [channels] or None, in x's dtype or float32; initial_state:
    [B, W - 1, channels], the tokens before the first, oldest first, or None (zeros); out: optional
    [B, T, channels] buffer in x's dtype that overlaps no input, for calls without gradients.  Returns (y, final state
    [B, W - 1, channels] in x's dtype).  Differentiable (once) in x, weight, bias and initial_state;
    the gradients do not depend on timing."""
    if x.dim() != 3:
        raise ValueError("x must be [B, T, channels]")
    Dm, W, silu = _check_conv(x, weight, bias, activation)
    Bn, T, _ = x.shape
    if initial_state is not None:
        _one_device(x, initial_state)
        if tuple(initial_state.shape) != (Bn, W - 1, Dm):
            raise ValueError(f"initial_state must be [{Bn}, {W - 1}, {Dm}]")
    grad = _needs_grad(x, weight, bias, initial_state)
    if grad and out is not None:
        raise ValueError("out is for calls without gradients")
    if out is not None:
        _one_device(x, out)
    if grad:
        return _ShortConv.apply(x, weight, bias, initial_state, silu)
    if Bn == 0 or T == 0:
        return _out(out, x.shape, x.dtype, x), _no_conv_tokens(x, W, initial_state)
    return _conv(x, weight, bias, silu, initial_state, out)


def short_conv_varlen(x, weight, cu_seqlens, bias=None, initial_state=None, activation="silu", out=None, *,
                      state_pool=None, slots=None):
    """short_conv over packed ragged prompts x [N, channels] or [1, N, channels], without gradients;
    cu_seqlens, initial_state [n, W - 1, channels], state_pool [rows, W - 1, channels] in x's
    dtype, slots and the returned pair as in ssm_scan_varlen."""
    _no_grad_path("short_conv_varlen", x, weight, bias, initial_state, state_pool)
    lead1 = x.dim() == 3
    if lead1:
        if x.shape[0] != 1 or (out is not None and (out.dim() != 3 or out.shape[0] != 1)):
            raise ValueError("packed varlen tensors have batch size 1")
        x, out = x[0], None if out is None else out[0]
    if x.dim() != 2:
        raise ValueError("x must be [N, channels] or [1, N, channels]")
    Dm, W, silu = _check_conv(x, weight, bias, activation)
    _one_device(x, initial_state, out, state_pool)
    total = x.shape[0]
    cu = _cu(cu_seqlens, x.device)
    n = cu.numel() - 1
    if state_pool is not None:
        _pool(state_pool, slots, initial_state, (W - 1, Dm), x.dtype)
        s0 = fin = state_pool
    else:
        if slots is not None:
            raise ValueError("slots needs state_pool")
        if initial_state is not None and tuple(initial_state.shape) != (n, W - 1, Dm):
            raise ValueError(f"initial_state must be [{n}, {W - 1}, {Dm}]")
        s0 = None if initial_state is None else initial_state.to(x.dtype).contiguous()
        fin = torch.empty(n, W - 1, Dm, device=x.device, dtype=x.dtype)
    sl = _slots(slots, n, x.device)
    y = _out(out, x.shape, x.dtype, x)
    if total == 0:
        if state_pool is None:
            fin.zero_() if s0 is None else fin.copy_(s0)
    elif n > 0:
        x, weight, bias = _rows(x), weight.contiguous(), _c(bias)
        call_on(x, "triune_hip_short_conv_varlen", ptr(x), ptr(weight), ptr(bias), dtype_code(x), dtype_code(weight),
                strides(x.stride()[:1], y.stride()[:1]), int(silu), ptr(cu), n, total, ptr(s0), ptr(fin), ptr(sl),
                fin.shape[0], ptr(y), Dm, W)
    return (y.unsqueeze(0) if lead1 else y), fin


def short_conv_decode_step(x, weight, state, bias=None, activation="silu", out=None, *, inplace=False, slots=None):
    """One token of short_conv for each of a batch of sequences, without gradients: x [B, channels] or
    [B, 1, channels]; state [B, W - 1, channels], or a pool of rows addressed by slots, in x's dtype;
    slots, inplace and the returned pair as in ssm_decode_step."""
    _no_grad_path("short_conv_decode_step", x, weight, state, bias)
    token = x.dim() == 3
    if token:
        if x.shape[1] != 1 or (out is not None and (out.dim() != 3 or out.shape[1] != 1)):
            raise ValueError("decode step takes one token per sequence (T == 1)")
        x, out = x[:, 0], None if out is None else out[:, 0]
    if x.dim() != 2:
        raise ValueError("x must be [B, channels] or [B, 1, channels]")
    Dm, W, silu = _check_conv(x, weight, bias, activation)
    _one_device(x, state, out)
    n = x.shape[0]
    s_in, s_out = _step_states(state, inplace, slots, n, x.dtype, (W - 1, Dm))
    sl = _slots(slots, n, x.device)
    y = _out(out, x.shape, x.dtype, x)
    if n > 0:
        x, weight, bias = _rows(x), weight.contiguous(), _c(bias)
        call_on(x, "triune_hip_short_conv_decode_step", ptr(x), ptr(weight), ptr(bias), dtype_code(x),
                dtype_code(weight), strides(x.stride()[:1], y.stride()[:1]), int(silu), ptr(s_in), ptr(s_out), ptr(sl),
                s_in.shape[0], ptr(y), n, Dm, W)
    return (y.unsqueeze(1) if token else y), s_out
