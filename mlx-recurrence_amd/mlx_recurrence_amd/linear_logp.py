"""linear_logp.py — the labels' log-probabilities over a large vocabulary straight from hidden
states, and the losses on them (no counterpart in the reference, which has the scans alone).

    linear_log_probs(hidden, weight, labels)                                     -> log-probabilities
    linear_policy_loss(hidden, weight, labels, advantages, old, ref)             -> loss
    linear_preference_loss(hidden, weight, labels, ref)                          -> loss
    linear_log_probs_reference, linear_policy_loss_reference, linear_preference_loss_reference
                                                                                 (plain torch)

They run on the kernels of linear_loss.py: the logits are formed tile by tile, rows that are
ignored cost nothing, and `keep_logits` is as there.  The losses are taken in the launch that
closes a row's softmax, which leaves the backward one value a row.  The products run in the
inputs' type with fp32 accumulation; log-probabilities and losses are fp32, sums over a
sequence and what follows from them 64 bits.  With 16-bit inputs and more than 64 rows the
gradient of the logits is rounded to their type, half a step at most: give fp32 inputs where
that is too much.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .linear_loss import _REDUCTIONS, _check, _check_ids, _reduce

_LOGP, _POLICY, _PREFERENCE = 0, 1, 2


class _LinearLogp(torch.autograd.Function):
    """hidden [rows, D] and weight [V, D] of one type, labels [rows].  kind _POLICY: advantages [rows / per], old and
    ref [rows]; _PREFERENCE: `losses` pairs of sequences of `per` tokens, ref [pairs, 2].  values: the temperature and
    the loss's own numbers."""

    @staticmethod
    def forward(ctx, hidden, weight, labels, advantages, old, ref, kind, losses, per, ignore_index, values, reduction, grad):
        dev = _lib.require_device(hidden, weight, labels, advantages, old, ref)
        dt = hidden.dtype
        h_, w_, l_ = _lib.prep(hidden, dt), _lib.prep(weight, dt), _lib.prep(labels, torch.int64)
        a_, o_, r_ = (None if t is None else _lib.prep(t, torch.float32) for t in (advantages, old, ref))
        (rows, D), V = h_.shape, w_.shape[0]
        loss = torch.empty((losses,) if reduction == 0 else (), dtype=torch.float32, device=dev)
        with _lib.device_guard(dev):
            state, ws = _lib.linear_loss_buffers(rows, D, V, 1, dt, dev, grad)
            if kind == _LOGP:
                _lib.linear_logp_fwd(h_, w_, l_, ignore_index, values[0], loss, state, ws)
            elif kind == _POLICY:
                _lib.linear_policy_fwd(h_, w_, l_, ignore_index, values[0], a_, per, o_, r_, *values[1:], reduction, loss,
                                       state, ws)
            else:
                _lib.linear_preference_fwd(h_, w_, l_, ignore_index, losses, per, r_, *values[1:], reduction, loss, state, ws)
        ctx.save_for_backward(w_, state)   # the state holds the rows of hidden that count
        ctx.args = (rows, values[0], 2 * per if kind == _PREFERENCE and per > 0 else 1, int(kind == _LOGP), reduction)
        return loss

    @staticmethod
    def backward(ctx, dloss):
        _lib.refuse_second_derivatives()
        w_, state = ctx.saved_tensors
        dh = w_.new_empty((ctx.args[0], w_.shape[1])) if ctx.needs_input_grad[0] else None
        dw = torch.empty_like(w_) if ctx.needs_input_grad[1] else None
        with _lib.device_guard(w_.device):
            _lib.linear_logp_bwd(_lib.prep(dloss, torch.float32), w_, *ctx.args, state, dh, dw)
        return (dh, dw) + (None,) * 11


def _check_head(hidden, weight, labels, reduction):
    _check(hidden, weight, reduction)
    if tuple(labels.shape) != tuple(hidden.shape[:-1]):
        raise ValueError(f"labels must be {list(hidden.shape[:-1])}, got {tuple(labels.shape)}")
    _check_ids("labels", labels)


def _check_real(name, t, shapes):
    if not any(tuple(t.shape) == tuple(s) for s in shapes):
        raise ValueError(f"{name} must be {' or '.join(str(list(s)) for s in shapes)}, got {tuple(t.shape)}")
    if not t.dtype.is_floating_point:
        raise TypeError(f"{name} must be floating-point numbers, got {t.dtype}")


def _check_temperature(temperature):
    if not (float(temperature) > 0 and math.isfinite(float(temperature))):
        raise ValueError(f"temperature must be positive and finite, got {temperature}")


def _apply(hidden, weight, labels, keep_logits, advantages, old, ref, kind, losses, per, ignore_index, values, reduction):
    D = hidden.shape[-1]
    dt = _lib.common_dtype(hidden, weight)
    h = hidden if hidden.ndim == 2 else hidden.reshape(-1, D)
    h, w = h if h.dtype == dt else h.to(dt), weight if weight.dtype == dt else weight.to(dt)
    flat = [None if t is None else t.detach().reshape(-1) for t in (advantages, old, ref)]
    ext = _lib.autograd_ext()
    # the same forward / backward as one C++ autograd node where it is built
    grad = (1 if keep_logits else 2) if _lib.records(h, w) else 0
    args = (h, w, labels.reshape(-1), *flat, kind, losses, per, int(ignore_index), [float(v) for v in values], reduction, grad)
    return _LinearLogp.apply(*args) if ext is None else ext.linear_logp(*args)


def linear_log_probs(hidden, weight, labels, *, temperature=1.0, ignore_index=-100, keep_logits=True):
    """Log-probabilities of `labels` under the softmax of ``hidden @ weight.T / temperature`` on the
    GPU (fused forward + backward): what a policy's or a reference's tokens are scored by.

    Args:
        hidden:       [..., D] hidden states.
        weight:       [V, D] of the output projection.  Inputs of two types run in the
                      wider one: cast a master weight to the hidden states' type first.
        labels:       [...] integers in [0, V), or `ignore_index`: such a row gives 0 and no
                      gradient, whatever its hidden state holds.  Any other label makes the
                      row's result (and every gradient) NaN.
        temperature:  of the softmax.
        keep_logits:  as for linear_cross_entropy.

    Returns:
        log_probs:    [...] fp32.  Gradients flow to hidden and weight (first derivatives only).
    """
    _check_head(hidden, weight, labels, "none")
    _check_temperature(temperature)
    rows = labels.numel()
    out = _apply(hidden, weight, labels, keep_logits, None, None, None, _LOGP, rows, 1, ignore_index, (temperature,), 0)
    return out if labels.ndim == 1 else out.reshape(labels.shape)


def _widths(clip):
    low, high = (clip, clip) if isinstance(clip, (int, float)) else clip
    if not (float(low) >= 0 and float(high) >= 0):
        raise ValueError(f"clip must be the width below and above 1, neither negative, got {clip}")
    return float(low), float(high)


def linear_policy_loss(hidden, weight, labels, advantages, old_log_probs=None, ref_log_probs=None, *, clip=(0.2, 0.2),
                       kl_weight=0.0, temperature=1.0, ignore_index=-100, reduction="mean", keep_logits=True):
    """Clipped policy loss with a KL term on sampled tokens, on the GPU (fused forward + backward).

    Per token, with ``logp`` its log-probability (linear_log_probs), ``r = exp(logp - old)`` and
    ``d = ref - logp``::

        loss = -min(r * A, clamp(r, 1 - clip[0], 1 + clip[1]) * A) + kl_weight * (exp(d) - d - 1)

    Args:
        hidden, weight, labels, temperature, ignore_index, keep_logits:  as for linear_log_probs;
                        a token that is ignored (a prompt's, padding) counts for nothing.
        advantages:     [...] one a token, or [..., 1] one for all tokens of the last axis.
        old_log_probs:  [...] of the policy that sampled, or None: this one (r is 1, and its
                        gradient that of logp).
        ref_log_probs:  [...] of the reference; needed, and read, where kl_weight is not 0.
        clip:           the widths below and above 1 within which a ratio is not clipped, or
                        one for both; math.inf does not clip.  A ratio on a border has its
                        gradient.
        kl_weight:      weight of the KL term.
        reduction:      "mean" over the tokens that count (0 where there is none), "sum", or
                        "none".

    Returns:
        loss:           fp32, a scalar or [...] for "none".  Gradients flow to hidden and weight
                        (first derivatives only), none to the advantages and the other policies.
    """
    _check_head(hidden, weight, labels, reduction)
    _check_temperature(temperature)
    lead = labels.shape
    one = (*lead[:-1], 1) if labels.ndim else lead
    _check_real("advantages", advantages, (lead, one) if labels.ndim else (lead,))
    low, high = _widths(clip)
    if not (float(kl_weight) >= 0 and math.isfinite(float(kl_weight))):
        raise ValueError(f"kl_weight must be finite and not negative, got {kl_weight}")
    for name, t in (("old_log_probs", old_log_probs), ("ref_log_probs", ref_log_probs)):
        if t is not None:
            _check_real(name, t, (lead,))
    if kl_weight and ref_log_probs is None:
        raise ValueError("kl_weight needs ref_log_probs")
    rows = labels.numel()
    per = max(1, lead[-1]) if labels.ndim and tuple(advantages.shape) != tuple(lead) else 1
    out = _apply(hidden, weight, labels, keep_logits, advantages, old_log_probs, ref_log_probs if kl_weight else None, _POLICY,
                 rows, per, ignore_index, (temperature, low, high, kl_weight), _REDUCTIONS[reduction])
    return out.reshape(lead) if reduction == "none" and labels.ndim != 1 else out


def linear_preference_loss(hidden, weight, labels, ref_log_probs=None, *, beta=0.1, label_smoothing=0.0, ignore_index=-100,
                           reduction="mean", keep_logits=True):
    """Preference loss on pairs of sequences, on the GPU (fused forward + backward).

    With ``S`` the sum of a sequence's log-probabilities (linear_log_probs) over its tokens that
    count, the preferred sequence of a pair first::

        m = beta * ((S[0] - ref[0]) - (S[1] - ref[1]))
        loss = -(1 - label_smoothing) * log_sigmoid(m) - label_smoothing * log_sigmoid(-m)

    Args:
        hidden:           [..., 2, L, D] hidden states of both sequences of each pair.
        weight, keep_logits:  as for linear_log_probs.
        labels:           [..., 2, L] integers in [0, V), or `ignore_index` (prompts, padding):
                          such a token counts for nothing.  Any other label makes the pair's
                          loss (and every gradient) NaN.
        ref_log_probs:    [..., 2] the reference's sums, or None (0).  Sums of long sequences are best
                          given in float64: what they differ by is not rounded with them.
        beta:             how far the policy may move from the reference: the smaller, the farther.
        label_smoothing:  share of pairs whose order is taken to be wrong, 0 to 0.5.
        reduction:        "mean" over the pairs with a token that counts (0 where there is
                          none), "sum", or "none".

    Returns:
        loss:             fp32, a scalar or [...] for "none".  Gradients flow to hidden and weight
                          (first derivatives only), none to the reference.
    """
    _check_head(hidden, weight, labels, reduction)
    if labels.ndim < 2 or labels.shape[-2] != 2:
        raise ValueError(f"labels must be [..., 2, L], a pair's preferred sequence first, got {tuple(labels.shape)}")
    lead = labels.shape[:-2]
    if ref_log_probs is not None:
        _check_real("ref_log_probs", ref_log_probs, ((*lead, 2),))
    if not (float(beta) > 0 and math.isfinite(float(beta))):
        raise ValueError(f"beta must be positive and finite, got {beta}")
    if not 0 <= float(label_smoothing) <= 0.5:
        raise ValueError(f"label_smoothing must be in [0, 0.5], got {label_smoothing}")
    if ref_log_probs is not None and ref_log_probs.dtype == torch.float64:
        # The loss takes their difference alone.  The sums are in the thousands, and rounded to fp32 each would be
        # off by up to 2.4e-4.
        ref = ref_log_probs.detach()
        ref_log_probs = torch.stack([ref[..., 0] - ref[..., 1], torch.zeros_like(ref[..., 0])], -1)
    out = _apply(hidden, weight, labels, keep_logits, None, None, ref_log_probs, _PREFERENCE, math.prod(lead), labels.shape[-1],
                 ignore_index, (1.0, beta, label_smoothing), _REDUCTIONS[reduction])
    return out.reshape(lead) if reduction == "none" and len(lead) != 1 else out


# ------------------------------------------------------------------ plain forms
def linear_log_probs_reference(hidden, weight, labels, *, temperature=1.0, ignore_index=-100):
    """linear_log_probs as plain torch ops on the whole logits, in fp32 or wider.
    Differentiable; runs on any device."""
    valid = labels != ignore_index
    ct = torch.promote_types(torch.promote_types(hidden.dtype, weight.dtype), torch.float32)
    z = torch.where(valid[..., None], hidden.to(ct), 0) @ weight.to(ct).T / temperature
    picked = torch.log_softmax(z, -1).gather(-1, torch.where(valid, labels, 0).long()[..., None])[..., 0]
    return torch.where(valid, picked, 0)


def linear_policy_loss_reference(hidden, weight, labels, advantages, old_log_probs=None, ref_log_probs=None, *,
                                 clip=(0.2, 0.2), kl_weight=0.0, temperature=1.0, ignore_index=-100, reduction="mean"):
    """linear_policy_loss as plain torch ops on the whole logits, in fp32 or wider.
    Differentiable; runs on any device."""
    low, high = _widths(clip)
    valid = labels != ignore_index
    logp = linear_log_probs_reference(hidden, weight, labels, temperature=temperature, ignore_index=ignore_index)
    A = torch.where(valid, advantages.detach().to(logp.dtype), 0)
    old = logp if old_log_probs is None else old_log_probs.to(logp.dtype)
    moved = logp - torch.where(valid, old, 0).detach()
    r = torch.exp(moved.detach())
    clipped = torch.where(A > 0, r > 1 + high, r < 1 - low)
    flat = clipped | ((A == 0) & ~torch.isnan(r))   # (not inf x 0)
    border = torch.where(A == 0, 1.0, torch.where(A > 0, 1 + high, 1 - low)).to(logp.dtype)
    loss = -torch.where(flat, border, torch.exp(torch.where(flat, 0, moved))) * A
    if kl_weight:
        d = torch.where(valid, ref_log_probs.detach().to(logp.dtype), 0) - logp
        loss = loss + kl_weight * (torch.expm1(d) - d)
    return _reduce(loss, valid, reduction)


def linear_preference_loss_reference(hidden, weight, labels, ref_log_probs=None, *, beta=0.1, label_smoothing=0.0,
                                     ignore_index=-100, reduction="mean"):
    """linear_preference_loss as plain torch ops on the whole logits, sums in 64 bits.
    Differentiable; runs on any device."""
    logp = linear_log_probs_reference(hidden, weight, labels, ignore_index=ignore_index)
    counts = (labels != ignore_index).flatten(-2).any(-1)
    S = logp.double().sum(-1)
    if ref_log_probs is not None:
        S = S - ref_log_probs.detach().double()
    m = beta * torch.where(counts, S[..., 0] - S[..., 1], 0)
    log_sigmoid = torch.nn.functional.logsigmoid
    loss = -(1 - label_smoothing) * log_sigmoid(m)
    if label_smoothing:
        loss = loss - label_smoothing * log_sigmoid(-m)
    return _reduce(loss, counts, reduction).to(logp.dtype)
