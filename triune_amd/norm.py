"""Layer norm on MI355X, forward and backward: the norm in front of a recurrent layer, over the rows of a
training batch or of a decode step's tokens.  No reference counterpart.

    y = (x - mean) rstd weight + bias,   rstd = 1 / sqrt(mean((x - mean)^2) + eps)

Statistics and sums are float32, outputs are rounded once.  There is no CPU path and no forward-mode
derivative.
"""

from __future__ import annotations

import torch

from ._lib import call_on, dtype_code, plan_on, ptr
from .ssm import _needs_grad, _one_device

__all__ = ["layer_norm"]

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
