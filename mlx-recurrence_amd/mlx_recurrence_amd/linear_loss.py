"""linear_loss.py — losses over a large vocabulary straight from hidden states (no
counterpart in the reference, which has the scans alone).

    linear_cross_entropy(hidden, weight, labels)                       -> loss
    linear_distillation(hidden, weight, teacher_logits, teacher_ids)   -> loss
    linear_cross_entropy_reference, linear_distillation_reference      (plain torch)

Both take the head's input and its weight in place of the logits ``hidden @
weight.T``, which are formed tile by tile inside the kernels.  Between forward and
backward the logits of few rows, and where that is faster up to 4 GiB of them, stay in
fp32 (``keep_logits=False``: of few rows alone); beyond that the backward, whose gradient of the logits is a piece of half a GiB at
a time, forms them again.  Without gradients none are kept (a few tiles' logits may be
summed from parts, of at most 256 MiB, during the call).
The products run in the inputs' type with fp32 accumulation; the loss is fp32.
"""
from __future__ import annotations

import math

import torch

from . import _lib

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


class _LinearLoss(torch.autograd.Function):
    """hidden [rows, D] and weight [V, D] of one type; `labels` [rows], or teacher
    logits and ids [rows, K]."""

    @staticmethod
    def forward(ctx, hidden, weight, labels, t_logits, t_ids, ignore_index, z_loss, temperature, reduction, grad):
        dev = _lib.require_device(hidden, weight, labels, t_logits, t_ids)
        dt = hidden.dtype
        h_, w_ = _lib.prep(hidden, dt), _lib.prep(weight, dt)
        (rows, D), V = h_.shape, w_.shape[0]
        K = 1 if t_ids is None else t_ids.shape[1]
        loss = torch.empty((rows,) if reduction == 0 else (), dtype=torch.float32, device=dev)
        with _lib.device_guard(dev):
            state, ws = _lib.linear_loss_buffers(rows, D, V, K, dt, dev, grad)
            if t_ids is None:
                _lib.linear_ce_fwd(h_, w_, _lib.prep(labels, torch.int64), ignore_index, z_loss, reduction, loss, state, ws)
            else:
                tdt = _lib.common_dtype(t_logits)
                _lib.linear_kd_fwd(h_, w_, _lib.prep(t_logits, tdt), _lib.prep(t_ids, torch.int64), temperature, reduction,
                                   loss, state, ws)
        ctx.save_for_backward(w_, state)   # the state holds the rows of hidden that count
        ctx.args = (rows, K, z_loss, temperature, reduction)
        return loss

    @staticmethod
    def backward(ctx, dloss):
        _lib.refuse_second_derivatives()
        w_, state = ctx.saved_tensors
        dh = w_.new_empty((ctx.args[0], w_.shape[1])) if ctx.needs_input_grad[0] else None
        dw = torch.empty_like(w_) if ctx.needs_input_grad[1] else None
        with _lib.device_guard(w_.device):
            _lib.linear_loss_bwd(_lib.prep(dloss, torch.float32), w_, *ctx.args, state, dh, dw)
        return (dh, dw) + (None,) * 8


def _check(hidden, weight, reduction):
    if hidden.ndim < 1 or hidden.shape[-1] == 0:
        raise ValueError(f"hidden must be [..., D] with D > 0, got shape {tuple(hidden.shape)}")
    D = hidden.shape[-1]
    if weight.ndim != 2 or weight.shape[1] != D or weight.shape[0] == 0:
        raise ValueError(f"weight must be [V, D] with V > 0 and D = {D}, got {tuple(weight.shape)}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'none', 'mean' or 'sum', got {reduction!r}")


def _check_ids(name, t):
    if t.dtype.is_floating_point or t.dtype.is_complex or t.dtype == torch.bool:
        raise TypeError(f"{name} must be integers, got {t.dtype}")


def _apply(hidden, weight, keep_logits, *args):
    """args: what _LinearLoss takes behind the weight."""
    lead, D = hidden.shape[:-1], hidden.shape[-1]
    dt = _lib.common_dtype(hidden, weight)
    h = hidden if len(lead) == 1 else hidden.reshape(-1, D)
    h, w = h if h.dtype == dt else h.to(dt), weight if weight.dtype == dt else weight.to(dt)
    ext = _lib.autograd_ext()
    # the same forward / backward as one C++ autograd node where it is built
    grad = (1 if keep_logits else 2) if _lib.records(h, w) else 0
    loss = _LinearLoss.apply(h, w, *args, grad) if ext is None else ext.linear_loss(h, w, *args, grad)
    return loss.reshape(lead) if len(lead) != 1 and loss.ndim == 1 else loss


def linear_cross_entropy(hidden, weight, labels, *, ignore_index=-100, z_loss=0.0, reduction="mean", keep_logits=True):
    """Softmax cross entropy of ``hidden @ weight.T`` with `labels` on the GPU (fused
    forward + backward).

    Per row, with ``z = hidden @ weight.T`` and ``lse = logsumexp(z)``::

        loss = lse - z[label] + z_loss * lse**2

    Args:
        hidden:       [..., D] hidden states.
        weight:       [V, D] of the output projection.  Inputs of two types run in the
                      wider one: cast a master weight to the hidden states' type first.
        labels:       [...] integers in [0, V), or `ignore_index`: such a row gives no loss
                      and no gradient, whatever its hidden state holds, and is not
                      counted by the mean.  Any other label makes the row's loss (and
                      every gradient) NaN.
        z_loss:       weight of the squared log-normaliser.
        reduction:    "mean" over the rows that count (0 where there is none), "sum", or
                      "none".
        keep_logits:  whether the forward may leave the logits of more than 256 rows in
                      memory for the backward, in fp32 and up to 4 GiB, where that is
                      faster.  False: the backward forms them again (8192 rows, 65536
                      words, 2560 channels bf16: 8.7 ms in place of 7.45).

    Returns:
        loss:         fp32, a scalar or [...] for "none".  Gradients flow to hidden and weight
                      (first derivatives only).
    """
    _check(hidden, weight, reduction)
    if tuple(labels.shape) != tuple(hidden.shape[:-1]):
        raise ValueError(f"labels must be {list(hidden.shape[:-1])}, got {tuple(labels.shape)}")
    _check_ids("labels", labels)
    if not math.isfinite(float(z_loss)):
        raise ValueError(f"z_loss must be finite, got {z_loss}")
    return _apply(hidden, weight, keep_logits, labels.reshape(-1), None, None, int(ignore_index), float(z_loss), 1.0,
                  _REDUCTIONS[reduction])


def linear_distillation(hidden, weight, teacher_logits, teacher_ids, *, temperature=1.0, reduction="mean",
                        keep_logits=True):
    """Distillation from a teacher's top logits on the GPU (fused forward + backward).

    Per row, with p the softmax of ``teacher_logits / temperature`` over the row's
    entries and q that of ``hidden @ weight.T / temperature`` over the vocabulary::

        loss = temperature**2 * sum_k p[k] * (log p[k] - log q[teacher_ids[k]])

    Args:
        hidden:         [..., D] the student's hidden states.
        weight:         [V, D] of its output projection.
        teacher_logits: [..., K] the teacher's logits, K up to 1024, in any order.
        teacher_ids:    [..., K] their words, integers below V.  An entry with a negative
                        id or a logit of -inf is absent; a row without entries gives no
                        loss and no gradient and is not counted by the mean.  Any other
                        entry's id of V or more makes the row's loss (and every
                        gradient) NaN.
        temperature:    of both softmaxes.
        reduction, keep_logits:  as for linear_cross_entropy.

    Returns:
        loss:           fp32, a scalar or [...] for "none".  Gradients flow to hidden and
                        weight (first derivatives only), none to the teacher.
    """
    _check(hidden, weight, reduction)
    lead = tuple(hidden.shape[:-1])
    if teacher_ids.ndim != hidden.ndim or tuple(teacher_ids.shape[:-1]) != lead or teacher_ids.shape[-1] == 0:
        raise ValueError(f"teacher_ids must be {list(lead)} + [K] with K > 0, got {tuple(teacher_ids.shape)}")
    if tuple(teacher_logits.shape) != tuple(teacher_ids.shape):
        raise ValueError(f"teacher_logits and teacher_ids must match, got {tuple(teacher_logits.shape)} and "
                         f"{tuple(teacher_ids.shape)}")
    _check_ids("teacher_ids", teacher_ids)
    if not (float(temperature) > 0 and math.isfinite(float(temperature))):
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    K = teacher_ids.shape[-1]
    return _apply(hidden, weight, keep_logits, None, teacher_logits.detach().reshape(-1, K), teacher_ids.reshape(-1, K), 0, 0.0,
                  float(temperature), _REDUCTIONS[reduction])


def _reduce(loss, valid, reduction):
    loss = torch.where(valid, loss, 0)
    if reduction == "none":
        return loss
    return loss.sum() / valid.sum().clamp(min=1) if reduction == "mean" else loss.sum()


def _logits(hidden, weight, valid):
    ct = torch.promote_types(torch.promote_types(hidden.dtype, weight.dtype), torch.float32)
    return torch.where(valid[..., None], hidden.to(ct), 0) @ weight.to(ct).T


def linear_cross_entropy_reference(hidden, weight, labels, *, ignore_index=-100, z_loss=0.0, reduction="mean"):
    """linear_cross_entropy as plain torch ops on the whole logits, in fp32 or wider.
    Differentiable; runs on any device."""
    valid = labels != ignore_index
    z = _logits(hidden, weight, valid)
    lse = torch.logsumexp(z, -1)
    picked = z.gather(-1, torch.where(valid, labels, 0).long()[..., None])[..., 0]
    return _reduce(lse - picked + z_loss * lse * lse, valid, reduction)


def linear_distillation_reference(hidden, weight, teacher_logits, teacher_ids, *, temperature=1.0, reduction="mean"):
    """linear_distillation as plain torch ops on the whole logits, in fp32 or wider.
    Differentiable; runs on any device."""
    there = (teacher_ids >= 0) & (teacher_logits != -math.inf)
    valid = there.any(-1)
    z = _logits(hidden, weight, valid) / temperature
    t = torch.where(there, teacher_logits.to(z.dtype), -math.inf)
    t = torch.where(valid[..., None], t, 0)
    logp = torch.log_softmax((t - t.detach().amax(-1, keepdim=True)) / temperature, -1)
    p = logp.exp()
    logq = z.gather(-1, torch.where(there, teacher_ids, 0).long()) - torch.logsumexp(z, -1, keepdim=True)
    loss = (p * (torch.where(p > 0, logp, 0) - logq)).sum(-1)
    return _reduce(temperature ** 2 * loss, valid, reduction)
