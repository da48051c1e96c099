"""Layer norm, cross entropy and distillation and their gradients in 64 bits, written out
from their formulas (torch on any device), for the tests of the GPU kernels.  The
formulas are themselves checked against differences in test_head_api.py."""
from __future__ import annotations

import math

import torch


def layer_norm(x, w, b, eps, dy=None):
    """y, and with dy: (y, dx, dw, db); w, b may be None."""
    x = x.double()
    D = x.shape[-1]
    one, zero = torch.ones(D, dtype=torch.float64, device=x.device), torch.zeros(D, dtype=torch.float64, device=x.device)
    w, b = (one if w is None else w.double()), (zero if b is None else b.double())
    d = x - x.sum(-1, keepdim=True) / D
    r = ((d * d).sum(-1, keepdim=True) / D + eps) ** -0.5
    xh = d * r
    y = xh * w + b
    if dy is None:
        return y
    dy = dy.double()
    g = dy * w
    dx = r * (g - g.sum(-1, keepdim=True) / D - xh * ((g * xh).sum(-1, keepdim=True) / D))
    return y, dx, (dy * xh).reshape(-1, D).sum(0), dy.reshape(-1, D).sum(0)


def _grads(c, dz, h, w):
    dz = c[:, None] * dz
    return dz @ w, dz.T @ h


def _close(loss, count, valid, reduction, dloss):
    """(reduced loss, upstream of each row) of the rows' losses."""
    loss = torch.where(valid, loss, 0)
    if reduction == "none":
        return loss, torch.where(valid, dloss, 0)
    n = max(1, count) if reduction == "mean" else 1
    return loss.sum() / n, torch.where(valid, dloss / n, 0)


def _softmax(z):
    m = z.max(1, keepdim=True).values
    e = torch.exp(z - m)
    s = e.sum(1, keepdim=True)
    return e / s, (m + torch.log(s))[:, 0]


def cross_entropy(hidden, weight, labels, dloss, ignore=-100, zl=0.0, reduction="mean"):
    """(loss, dhidden, dweight)."""
    w, labels, dloss = weight.double(), labels.long(), dloss.double()
    valid = labels != ignore
    h = torch.where(valid[:, None], hidden.double(), 0)
    at = torch.where(valid, labels, 0)
    z = h @ w.T
    q, lse = _softmax(z)
    each = lse - z.gather(1, at[:, None])[:, 0] + zl * lse * lse
    loss, c = _close(each, int(valid.sum()), valid, reduction, dloss)
    dz = q * (1 + 2 * zl * lse)[:, None]
    dz.scatter_add_(1, at[:, None], -torch.ones_like(at, dtype=torch.float64)[:, None])
    return (loss, *_grads(c, dz, h, w))


def distillation(hidden, weight, t_logits, t_ids, dloss, tau=1.0, reduction="mean"):
    """(loss, dhidden, dweight)."""
    w, dloss = weight.double(), dloss.double()
    there = (t_ids >= 0) & (t_logits != -math.inf)
    valid = there.any(1)
    h = torch.where(valid[:, None], hidden.double(), 0)
    at = torch.where(there, t_ids, 0).long()
    t = torch.where(there, t_logits.double() / tau, -math.inf)
    top = torch.where(valid, t.max(1).values, 0)[:, None]
    e = torch.where(there, torch.exp(t - top), 0)
    p = e / torch.where(valid, e.sum(1), 1)[:, None]
    logp = torch.where(there, t - top - torch.log(torch.where(valid, e.sum(1), 1))[:, None], 0)
    z = h @ w.T / tau
    q, lse = _softmax(z)
    each = tau * tau * (p * (logp - (z.gather(1, at) - lse[:, None]))).sum(1)
    loss, c = _close(each, int(valid.sum()), valid, reduction, dloss)
    dz = q.scatter_add(1, at, -p) * tau
    return (loss, *_grads(c, dz, h, w))
