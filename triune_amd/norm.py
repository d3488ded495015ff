"""Norms on MI355X, forward and backward: layer norm and RMS norm in front of a recurrent layer, the latter with the
residual sum, and the gated RMS norm behind one, over the rows of a training batch or of a decode step's tokens.  No
reference counterpart.

    layer_norm       y = (x - mean) rstd weight + bias,   rstd = 1 / sqrt(mean((x - mean)^2) + eps)
    rms_norm         y = x rstd weight,                   rstd = 1 / sqrt(mean(x^2) + eps)
    add_rms_norm     h = residual + scale x,              y = rms_norm(h)
    gated_rms_norm   y = rms_norm(x) silu(z)

Statistics and sums are float32, outputs are rounded once.  There is no CPU path and no forward-mode
derivative.
"""

from __future__ import annotations

import torch

from ._lib import call_on, dtype_code, plan_on, ptr, strides
from .ssm import _needs_grad, _one_device

__all__ = ["layer_norm", "rms_norm", "add_rms_norm", "gated_rms_norm"]

MAX_WIDTH = 16384


def _flat(x):
    """x as rows [R, D] of one stride (a copy where its layout has none)."""
    x = x.reshape(-1, x.shape[-1])
    return x if x.stride(-1) == 1 else x.contiguous()


def _forward(x, weight, bias, eps, stats):
    rows = _flat(x)
    R, D = rows.shape
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    mean = rstd = None
    if stats:
        mean, rstd = torch.empty(2, R, device=x.device, dtype=torch.float32)
    call_on(x, "triune_hip_layer_norm", ptr(rows), rows.stride(0), ptr(weight), ptr(bias), dtype_code(x),
            0 if weight is None else dtype_code(weight), 0 if bias is None else dtype_code(bias), eps, ptr(y),
            ptr(mean), ptr(rstd), R, D)
    return y, mean, rstd


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = _forward(x, weight, bias, eps, True) if x.numel() else (torch.empty_like(x), None, None)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        if mean is None:  # no rows
            db = None if ctx.bias_dtype is None else torch.zeros(x.shape[-1], device=x.device, dtype=ctx.bias_dtype)
            return torch.zeros_like(x), None if weight is None else torch.zeros_like(weight), db, None
        rows, up = _flat(x), _flat(dy.to(x.dtype))
        R, D = rows.shape
        dx = torch.empty(x.shape, device=x.device, dtype=x.dtype)
        dw = torch.empty_like(weight) if weight is not None and ctx.needs_input_grad[1] else None
        db = None
        if ctx.bias_dtype is not None and ctx.needs_input_grad[2]:
            db = torch.empty(D, device=x.device, dtype=ctx.bias_dtype)
        wsb = plan_on(x, "triune_hip_layer_norm_bwd_workspace_size", R, D) if dw is not None or db is not None else 0
        ws = torch.empty(wsb, device=x.device, dtype=torch.uint8) if wsb else None
        call_on(x, "triune_hip_layer_norm_bwd", ptr(rows), rows.stride(0), ptr(weight), ptr(up), up.stride(0),
                dtype_code(x), 0 if weight is None else dtype_code(weight), 0 if db is None else dtype_code(db),
                ptr(mean), ptr(rstd), ptr(dx), ptr(dw), ptr(db), R, D, ptr(ws), wsb)
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm over the last dim of x (at most 16384 wide, any leading dims and strides); weight and bias:
    [D] in x's dtype or float32, each may be None.  Returns y like x, contiguous.  Differentiable
    (once); the gradients do not depend on timing."""
    _one_device(x, weight, bias)
    dtype_code(x)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"rows of 1 to {MAX_WIDTH} elements are supported")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and tuple(p.shape) != (x.shape[-1],):
            raise ValueError(f"{name} must be [{x.shape[-1]}]")
        if p is not None and p.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{name} must have x's dtype or float32")
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if _needs_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    if x.numel() == 0:
        return torch.empty_like(x)
    return _forward(x, weight, bias, float(eps), False)[0]


# ---------------------------------------------------------------------------------------
# RMS norms
# ---------------------------------------------------------------------------------------


def _inner(x):
    """Rows of one stride: those of the dim in front of the last, of a tensor of three dims or more."""
    return x.shape[-2] if x.dim() >= 3 and x.shape[-2] > 0 else 1


def _pair(x, G):
    """(x, stride of every G-th row, stride of the rows between): a copy where the rows have none."""
    if x.is_contiguous():
        return x, G * x.shape[-1], x.shape[-1]
    if x.stride(-1) != 1 and x.shape[-1] != 1:
        x = x.contiguous()
    lead = [(n, s) for n, s in zip(x.shape[:-1], x.stride()[:-1])]
    inner = lead.pop()[1] if x.dim() >= 3 and lead else None
    outer = [(n, s) for n, s in lead if n != 1]
    for (_, s), (n, t) in zip(outer, outer[1:]):
        if s != n * t:
            return _pair(x.contiguous(), G)
    step = outer[-1][1] if outer else 0
    return x, step, step if inner is None else inner


def _rms_check(x, other, eps, weight, scale=None):
    _one_device(x, other, weight, scale)
    dtype_code(x)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"rows of 1 to {MAX_WIDTH} elements are supported")
    for name, p in (("weight", weight), ("scale", scale)):
        if p is None:
            continue
        if p.dim() != 1 or p.shape[0] != x.shape[-1]:
            raise ValueError(f"{name} must be [{x.shape[-1]}]")
        if p.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{name} must have x's dtype or float32")
    if not eps >= 0:
        raise ValueError("eps must not be negative")


def _code(t):
    return 0 if t is None else dtype_code(t)


def _rms(x, r, weight, scale, alpha, eps, stats):
    """(y, h or None, rstd or None)."""
    G, D = _inner(x), x.shape[-1]
    R = x.numel() // D
    x, x0, x1 = _pair(x, G)
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    h = r0 = r1 = None
    if r is not None:
        r, r0, r1 = _pair(r, G)
        h = torch.empty(x.shape, device=x.device, dtype=r.dtype)
    rstd = torch.empty(R, device=x.device, dtype=torch.float32) if stats else None
    if R:
        call_on(x, "triune_hip_rms_norm", ptr(x), ptr(r), ptr(weight), ptr(scale), dtype_code(x), _code(r), _code(weight),
                _code(scale), strides((x0, x1, r0 or 0, r1 or 0)), alpha, eps, ptr(y), ptr(h), ptr(rstd), R, G, D)
    return y, h, rstd


def _grad_space(x, R, D, want):
    wsb = plan_on(x, "triune_hip_rms_norm_bwd_workspace_size", R, D) if want and R else 0
    return (torch.empty(wsb, device=x.device, dtype=torch.uint8) if wsb else None), wsb


class _RmsNorm(torch.autograd.Function):
    """rms_norm (r None) and add_rms_norm."""

    @staticmethod
    def forward(ctx, x, r, weight, scale, alpha, eps):
        y, h, rstd = _rms(x, r, weight, scale, alpha, eps, True)
        # the sum is kept as the output that it is; x is read again for the gradient of its scale only
        ctx.save_for_backward(x if r is None else h, x if scale is not None else None, weight, scale, rstd)
        ctx.alpha, ctx.plain, ctx.x_dtype = alpha, r is None, x.dtype
        ctx.set_materialize_grads(False)
        return y if r is None else (y, h)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh=None):
        h, x, weight, scale, rstd = ctx.saved_tensors
        if dy is None and dh is None:
            return (None,) * 6
        dev, G, D = h.device, _inner(h), h.shape[-1]
        R = h.numel() // D
        wx, wr, ww, ws_ = ctx.needs_input_grad[:4]
        dx = torch.empty(h.shape, device=dev, dtype=ctx.x_dtype) if wx else None
        dr = torch.empty(h.shape, device=dev, dtype=h.dtype) if wr and not ctx.plain else None
        dw = torch.empty_like(weight) if weight is not None and ww else None
        ds = torch.empty_like(scale) if scale is not None and ws_ else None
        if R == 0:
            return dx, dr, None if dw is None else dw.zero_(), None if ds is None else ds.zero_(), None, None
        dy = torch.zeros(h.shape, device=dev, dtype=ctx.x_dtype) if dy is None else dy.to(ctx.x_dtype)
        h, h0, h1 = _pair(h, G)
        dy, y0, y1 = _pair(dy, G)
        d0 = d1 = x0 = x1 = 0
        if dh is not None:
            dh, d0, d1 = _pair(dh.to(h.dtype), G)
        if x is not None:
            x, x0, x1 = _pair(x, G)
        ws, wsb = _grad_space(h, R, D, dw is not None or ds is not None)
        call_on(h, "triune_hip_rms_norm_bwd", ptr(h), ptr(dy), ptr(dh), ptr(x), ptr(weight), ptr(scale), dtype_code(dy),
                dtype_code(h), _code(weight), _code(scale), strides((h0, h1, y0, y1, d0, d1, x0, x1)), ctx.alpha,
                ptr(rstd), ptr(dx), ptr(dr), ptr(dw), ptr(ds), R, G, D, ptr(ws), wsb)
        return dx, dr, dw, ds, None, None


def rms_norm(x, weight=None, eps=1e-6):
    """RMS norm over the last dim of x (at most 16384 wide, any leading dims and strides); weight: [D] in x's dtype or
    float32, or None.  Returns y like x, contiguous.  Differentiable (once); the gradients do not depend on timing."""
    _rms_check(x, None, eps, weight)
    weight = None if weight is None else weight.contiguous()
    if _needs_grad(x, weight):
        return _RmsNorm.apply(x, None, weight, None, 1.0, float(eps))
    return _rms(x, None, weight, None, 1.0, float(eps), False)[0]


def add_rms_norm(x, residual, weight=None, scale=None, eps=1e-6):
    """The residual sum h = residual + scale x in front of a block and its RMS norm, in one pass.

    x: a block's output, any leading dims and strides, at most 16384 wide; residual: its shape, in x's dtype or float32;
    scale: a number, [D] in x's dtype or float32 (a residual scale for each channel), or None (1); weight: as in
    rms_norm.  Returns (y in x's dtype, h in residual's dtype), contiguous; y is the norm of h as rounded, so that
    rms_norm(h) gives it again.  Differentiable in every tensor argument (once); the gradients do not depend on
    timing."""
    alpha = 1.0
    if scale is not None and not torch.is_tensor(scale):
        scale, alpha = None, float(scale)
    _rms_check(x, residual, eps, weight, scale)
    if residual.shape != x.shape:
        raise ValueError(f"residual must be {list(x.shape)}")
    if residual.dtype not in (x.dtype, torch.float32):
        raise TypeError("residual must have x's dtype or float32")
    weight = None if weight is None else weight.contiguous()
    scale = None if scale is None else scale.contiguous()
    if _needs_grad(x, residual, weight, scale):
        return _RmsNorm.apply(x, residual, weight, scale, alpha, float(eps))
    return _rms(x, residual, weight, scale, alpha, float(eps), False)[:2]


def _gated(x, z, weight, eps, stats):
    G, D = _inner(x), x.shape[-1]
    R = x.numel() // D
    x, x0, x1 = _pair(x, G)
    z, z0, z1 = _pair(z, G)
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    rstd = torch.empty(R, device=x.device, dtype=torch.float32) if stats else None
    if R:
        call_on(x, "triune_hip_gated_rms_norm", ptr(x), ptr(z), ptr(weight), dtype_code(x), _code(weight),
                strides((x0, x1, z0, z1)), eps, ptr(y), ptr(rstd), R, G, D)
    return y, rstd


class _GatedRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, z, weight, eps):
        y, rstd = _gated(x, z, weight, eps, True)
        ctx.save_for_backward(x, z, weight, rstd)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, z, weight, rstd = ctx.saved_tensors
        G, D = _inner(x), x.shape[-1]
        R = x.numel() // D
        wx, wz, ww = ctx.needs_input_grad[:3]
        dx, dz = (torch.empty(x.shape, device=x.device, dtype=x.dtype) if w else None for w in (wx, wz))
        dw = torch.empty_like(weight) if weight is not None and ww else None
        if R == 0:
            return dx, dz, None if dw is None else dw.zero_(), None
        x, x0, x1 = _pair(x, G)
        z, z0, z1 = _pair(z, G)
        dy, y0, y1 = _pair(dy.to(x.dtype), G)
        ws, wsb = _grad_space(x, R, D, dw is not None)
        call_on(x, "triune_hip_gated_rms_norm_bwd", ptr(x), ptr(z), ptr(dy), ptr(weight), dtype_code(x), _code(weight),
                strides((x0, x1, z0, z1, y0, y1)), ptr(rstd), ptr(dx), ptr(dz), ptr(dw), R, G, D, ptr(ws), wsb)
        return dx, dz, dw, None


def gated_rms_norm(x, z, weight=None, eps=1e-6):
    """rms_norm(x, weight) silu(z): the norm behind a recurrent layer with its gate, over the last dim ([..., heads, dim]
    norms each head).  x and z: one shape and dtype, any leading dims and strides, at most 16384 wide; weight: as in
    rms_norm.  Returns y like x, contiguous.  Differentiable (once); the gradients do not depend on timing."""
    _rms_check(x, z, eps, weight)
    if z.shape != x.shape or z.dtype != x.dtype:
        raise ValueError(f"z must be {list(x.shape)} of {x.dtype}")
    weight = None if weight is None else weight.contiguous()
    if _needs_grad(x, z, weight):
        return _GatedRmsNorm.apply(x, z, weight, float(eps))
    return _gated(x, z, weight, float(eps), False)[0]
