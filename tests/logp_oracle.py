"""Log-probabilities, the clipped policy loss and the preference loss with their gradients in 64
bits, written out from their formulas (torch on any device), for the tests of the GPU kernels.
The formulas are themselves checked against differences in test_logp_api.py."""
from __future__ import annotations


import torch


def _head(hidden, weight, labels, tau, ignore):
    """Flat: (h, w, valid, place of each row's label, softmax, log-probabilities)."""
    D = weight.shape[1]
    w, l = weight.detach().double(), labels.reshape(-1).long()
    valid = l != ignore
    h = torch.where(valid[:, None], hidden.detach().reshape(-1, D).double(), 0)
    at = torch.where(valid, l, 0)[:, None]
    z = h @ w.T / tau
    m = z.max(1, keepdim=True).values
    e = torch.exp(z - m)
    s = e.sum(1, keepdim=True)
    logp = torch.where(valid, (z.gather(1, at) - m - torch.log(s))[:, 0], 0)
    return h, w, valid, at, e / s, logp


def _grads(by, q, at, h, w, tau, shape):
    """From the derivative by each row's log-probability.  And how far words that are nearly sure magnify
    errors: a probability's is against 1, what is left of it against 1 - q."""
    left = by * (1 - q.gather(1, at)[:, 0])
    sure = float(torch.nan_to_num(by).norm() / torch.nan_to_num(left).norm().clamp(min=1e-30))
    dz = -q * by[:, None]
    dz.scatter_add_(1, at, by[:, None])
    dz /= tau
    return (dz @ w).reshape(shape), dz.T @ h, max(1.0, sure)


def log_probs(hidden, weight, labels, up, tau=1.0, ignore=-100):
    """(log-probabilities, dhidden, dweight, what sure words magnify errors by)."""
    h, w, valid, at, q, logp = _head(hidden, weight, labels, tau, ignore)
    by = torch.where(valid, up.reshape(-1).double(), 0)
    return (logp.reshape(labels.shape), *_grads(by, q, at, h, w, tau, hidden.shape))


def policy(hidden, weight, labels, advantages, old, ref, up, clip=(0.2, 0.2), kl=0.0, tau=1.0, ignore=-100,
           reduction="mean"):
    """(loss, dhidden, dweight, what sure words magnify errors by)."""
    h, w, valid, at, q, logp = _head(hidden, weight, labels, tau, ignore)
    A = torch.where(valid, advantages.expand(labels.shape).reshape(-1).double(), 0)
    o = logp if old is None else torch.where(valid, old.reshape(-1).double(), 0)
    r = torch.exp(logp - o)
    out = torch.where(A > 0, r > 1 + clip[1], r < 1 - clip[0]) & (A != 0)
    best = torch.where(out, torch.where(A > 0, 1 + clip[1], 1 - clip[0]).double(), r)
    loss, by = -best * A, torch.where(out, 0, -r * A)
    if kl:
        d = torch.where(valid, ref.reshape(-1).double(), 0) - logp
        loss, by = loss + kl * (torch.expm1(d) - d), by - kl * torch.expm1(d)
    loss, by = torch.where(valid, loss, 0), torch.where(valid, by, 0)
    n = max(1, int(valid.sum())) if reduction == "mean" else 1
    by = by * up.reshape(-1).double() / n
    out = loss.reshape(labels.shape) if reduction == "none" else loss.sum() / n
    return (out, *_grads(by, q, at, h, w, tau, hidden.shape))


def preference(hidden, weight, labels, ref, up, beta=0.1, eps=0.0, ignore=-100, reduction="mean"):
    """(loss, dhidden, dweight, what sure words magnify errors by)."""
    h, w, valid, at, q, logp = _head(hidden, weight, labels, 1.0, ignore)
    L = labels.shape[-1]
    counts = valid.reshape(-1, 2 * L).any(1)
    S = logp.reshape(-1, 2, L).sum(2)
    if ref is not None:
        S = S - ref.reshape(-1, 2).double()
    m = beta * (S[:, 0] - S[:, 1])

    def softplus(x):
        return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))

    def sigmoid(x):
        return torch.exp(-softplus(-x))

    loss = torch.where(counts, (1 - eps) * softplus(-m) + eps * softplus(m), 0)
    n = max(1, int(counts.sum())) if reduction == "mean" else 1
    by_m = torch.where(counts, eps * sigmoid(m) - (1 - eps) * sigmoid(-m), 0) * up.reshape(-1).double() / n
    by = beta * torch.stack([by_m, -by_m], 1)[:, :, None].expand(-1, 2, L).reshape(-1)
    by = torch.where(valid, by, 0)
    out = loss.reshape(labels.shape[:-2]) if reduction == "none" else loss.sum() / n
    return (out, *_grads(by, q, at, h, w, 1.0, hidden.shape))


def size_of(hidden, weight, labels, tau=1.0, ignore=-100):
    """The largest |log-probability|: an error of one in 2^n of it moves a ratio by so much times that."""
    logp = _head(hidden, weight, labels, tau, ignore)[-1]
    return float(logp[torch.isfinite(logp)].abs().max()) if logp.numel() else 0.0


