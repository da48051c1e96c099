"""norm.py — layer norm over the last axis (no counterpart in the reference, which
has the scans alone).

    layer_norm(x, weight, bias, eps=1e-5)   -> y, of x's shape and dtype
    layer_norm_reference(x, weight, bias)   -> y  (plain torch)

The scans return fp32 and the projections around them take 16-bit inputs, so an
fp32 x may leave as another type (``out_dtype``) without a pass of its own.
"""
from __future__ import annotations

import math

import torch

from . import _lib


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, eps, out_dtype, grad):
        dev = _lib.require_device(x, w, b)
        x_ = _lib.prep(x, _lib.common_dtype(x))
        D = x_.shape[-1]
        rows = x_.numel() // D
        w_dtype = torch.float32 if w is None and b is None else (b if w is None else w).dtype
        w_ = None if w is None else _lib.prep(w, w_dtype)
        b_ = None if b is None else _lib.prep(b, w_dtype)
        y = torch.empty(x_.shape, dtype=out_dtype, device=dev)
        mean = rstd = None
        if grad:
            mean, rstd = torch.empty((2, rows), dtype=torch.float32, device=dev)
        with _lib.device_guard(dev):
            _lib.layer_norm_fwd(x_, w_, b_, w_dtype, rows, D, eps, y, mean, rstd)
        if grad:
            ctx.save_for_backward(x_, w_, mean, rstd)
            ctx.w_dtype = w_dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        _lib.refuse_second_derivatives()
        x_, w_, mean, rstd = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        D = x_.shape[-1]
        rows = x_.numel() // D
        dy_ = _lib.prep(dy, dy.dtype)
        dx = torch.empty_like(x_) if need_x else None
        dw = torch.empty((D,), dtype=ctx.w_dtype, device=x_.device) if need_w else None
        db = torch.empty((D,), dtype=ctx.w_dtype, device=x_.device) if need_b else None
        with _lib.device_guard(x_.device):
            _lib.layer_norm_bwd(dy_, x_, w_, ctx.w_dtype, mean, rstd, rows, D, dx, dw, db)
        return dx, dw, db, None, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, out_dtype=None):
    """Layer norm on the GPU (fused forward + backward).

    ``y = (x - mean) / sqrt(var + eps) * weight + bias`` with the mean and the
    (biased) variance of each row, the last axis of x; statistics and sums are
    fp32 whatever the types.

    Args:
        x:         [..., D], D up to 32768.
        weight:    [D] scale, or None (1).
        bias:      [D] shift, or None (0).
        eps:       added to the variance.
        out_dtype: the type of y: x's (default), or for an fp32 x any of the
                   three input types.

    Returns:
        y:         x's shape.  Gradients flow to x, weight and bias (first derivatives only).
    """
    if x.ndim < 1 or x.shape[-1] == 0:
        raise ValueError(f"x must be [..., D] with D > 0, got shape {tuple(x.shape)}")
    shape = x.shape[-1:]
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.shape != shape:
            raise ValueError(f"{name} must be [D] = [{shape[0]}], got {tuple(t.shape)}")
    eps = float(eps)
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    dt = _lib.common_dtype(x)
    out = dt if out_dtype is None else out_dtype
    if out != dt and (out not in _lib.DTYPE_CODE or dt != torch.float32):
        raise ValueError(f"out_dtype must be {dt} (or any input type for a float32 x), got {out_dtype}")
    if weight is not None or bias is not None:
        wdt = _lib.common_dtype(*(t for t in (weight, bias) if t is not None))
        weight = weight if weight is None or weight.dtype == wdt else weight.to(wdt)
        bias = bias if bias is None or bias.dtype == wdt else bias.to(wdt)
    if x.dtype != dt:
        x = x.to(dt)
    ext = _lib.autograd_ext()
    if ext is not None:   # the same forward / backward as one C++ autograd node
        return ext.layer_norm(x, weight, bias, eps, _lib.DTYPE_CODE[out])
    return _LayerNorm.apply(x, weight, bias, eps, out, _lib.records(x, weight, bias))


def layer_norm_reference(x, weight=None, bias=None, eps=1e-5, *, out_dtype=None):
    """Layer norm as plain torch ops, in fp32 or wider.  Differentiable; runs on any device."""
    ct = torch.promote_types(x.dtype, torch.float32)
    h = x.to(ct)
    d = h - h.mean(-1, keepdim=True)
    y = d * torch.rsqrt((d * d).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.to(ct)
    if bias is not None:
        y = y + bias.to(ct)
    return y.to(x.dtype if out_dtype is None else out_dtype)
