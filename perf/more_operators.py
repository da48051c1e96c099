"""Performance cases of the operators that training from preferences and rewards adds to a language
model's output head: the losses on log-probabilities straight from hidden states, the
log-probabilities themselves, and the clipping of a step's gradients by their norm.

Kinds and their ranges (`draw` spreads cases over them; `listed` holds several of each):

    logp        linear_log_probs, forward alone (a reference or an old policy's pass, scoring), 1 to
                8192 rows of 32 to 5120 channels against a vocabulary of 500 to 131072
    policy      linear_policy_loss of sequences of 1 to 2048 tokens, forward and backward, with a
                reference and without, an advantage a token or a sequence
    preference  linear_preference_loss of 1 to 128 pairs of sequences of 1 to 1024 tokens, forward and
                backward
    clip        clip_grad_norm over 1 to 400 tensors of up to 480 million values, of one type or of two;
                tensors of their own, or pieces of one flat buffer as gradient buckets have them

Hidden states are of unit variance with a part that points at the row's label, so that a row's softmax
has a head and a long tail.  Some tokens are ignored, as prompts and padding are.  The old policy's and
the reference's log-probabilities are the model's own with some noise: a policy moves a little between
the pass that sampled and the step.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ITEM = {"f32": 4, "bf16": 2, "f16": 2}
IGNORE = -100
CLIP = (0.2, 0.28)           # below and above 1
MOST = 8192 * 2560 * 65536   # rows x channels x vocabulary of the largest case
MOST_VALUES = 483_000_000    # of the largest clipped step


def listed():
    return [
        # scoring the new tokens of a serving batch at a sampling temperature: the weight is read once
        dict(name="logp_token", kind="logp", dtype="bf16", B=8, L=1, D=5120, V=65536, ignored=0.0, tau=0.7),
        # the reference's pass over a batch of a 2560-wide model
        dict(name="logp_reference", kind="logp", dtype="bf16", B=16, L=512, D=2560, V=65536, ignored=0.25, tau=1.0),
        # a policy step of a small model, an advantage a sequence, no reference
        dict(name="policy_small", kind="policy", dtype="bf16", B=16, L=96, D=768, V=32000, ignored=0.25, tau=1.0, kl=0.0,
             by_token=False, mean=True),
        # a policy step of a 2560-wide model with a large vocabulary and a KL term
        dict(name="policy_large", kind="policy", dtype="bf16", B=8, L=1024, D=2560, V=65536, ignored=0.1, tau=1.0,
             kl=0.04, by_token=False, mean=True),
        # ragged in every size, an advantage and a loss a token, a sampling temperature
        dict(name="policy_ragged_f16", kind="policy", dtype="f16", B=7, L=143, D=1000, V=20011, ignored=0.3, tau=1.3,
             kl=0.1, by_token=True, mean=False),
        # fp32 training of a small model
        dict(name="policy_f32", kind="policy", dtype="f32", B=8, L=64, D=512, V=16001, ignored=0.1, tau=1.0, kl=0.02,
             by_token=True, mean=True),
        # two pairs of a small model
        dict(name="preference_small", kind="preference", dtype="bf16", B=2, L=128, D=768, V=32000, ignored=0.3, beta=0.1,
             eps=0.0, mean=True),
        # eight pairs of a 2560-wide model with a large vocabulary
        dict(name="preference_large", kind="preference", dtype="bf16", B=8, L=512, D=2560, V=65536, ignored=0.2, beta=0.1,
             eps=0.0, mean=True),
        # ragged in every size, a loss a pair, smoothed labels
        dict(name="preference_ragged_f32", kind="preference", dtype="f32", B=5, L=101, D=500, V=10007, ignored=0.4,
             beta=0.2, eps=0.1, mean=False),
        # a small model of eleven tensors: latency
        dict(name="clip_small", kind="clip", dtype="f32", layers=2, D=256, V=2000, flat=False, mixed=False, clips=True),
        # a 2560-wide model: matrices in bf16, norms and biases in fp32
        dict(name="clip_large", kind="clip", dtype="bf16", layers=12, D=2560, V=65536, flat=False, mixed=True, clips=True),
        # buckets: pieces of odd sizes of one flat buffer, most of them small
        dict(name="clip_bucket", kind="clip", dtype="bf16", tensors=301, values=7_500_001, flat=True, mixed=False, clips=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _odd_or_even(rng, n, step):
    """Half of the sizes are multiples of `step`, as most models' are, half are left as drawn."""
    return max(step, n // step * step) if rng.random() < 0.5 else n


def draw(rng):
    kind = rng.choice(["logp", "policy", "policy", "preference", "preference", "clip"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
    if kind == "clip":
        clips = rng.random() < 0.7
        if rng.random() < 0.5:
            values = _log_int(rng, 1000, 250_000_000)
            return dict(kind=kind, dtype=dtype, tensors=_log_int(rng, 1, min(400, values // 8)), values=values, flat=True,
                        mixed=False, clips=clips)
        D, V = 32 * _log_int(rng, 2, 80), _log_int(rng, 500, 65536)
        layers = max(1, min(_log_int(rng, 1, 14), (MOST_VALUES - V * D) // (4 * D * D)))
        return dict(kind=kind, dtype=dtype, layers=layers, D=D, V=V, flat=False, mixed=rng.random() < 0.4, clips=clips)
    D = _odd_or_even(rng, _log_int(rng, 32, 5120), 64)
    V = _odd_or_even(rng, _log_int(rng, 500, 131072), 64)
    rows = min(8192, 8192 * 65536 // V, MOST // (8 * D * V) if dtype == "f32" else MOST // (D * V))
    c = dict(kind=kind, dtype=dtype, D=D, V=V, ignored=rng.choice([0.0, 0.1, 0.4]))
    if kind == "preference":
        c["L"] = _log_int(rng, 1, max(1, min(1024, rows // 2)))
        c["B"] = _log_int(rng, 1, max(1, min(128, rows // (2 * c["L"]))))
        c.update(beta=rng.choice([0.05, 0.1, 0.2]), eps=rng.choice([0.0, 0.0, 0.1]), mean=rng.random() < 0.7)
        return c
    c["L"] = _log_int(rng, 1, max(1, min(2048, rows)))
    c["B"] = _log_int(rng, 1, max(1, min(1024, rows // c["L"])))
    c["tau"] = rng.choice([0.7, 1.0, 1.0, 1.3])
    if kind == "policy":
        c.update(kl=rng.choice([0.0, 0.02, 0.1]), by_token=rng.random() < 0.5, mean=rng.random() < 0.7)
    return c


# ------------------------------------------------------------------ inputs
def _log_probs_of(h, w, labels, tau):
    """The model's own log-probabilities, a few hundred million logits at a time."""
    w, out = w.float(), []
    step = max(1, (1 << 28) // len(w))
    for a, l in zip(h.split(step), labels.split(step)):
        z = (a.float() @ w.T) / tau
        out.append(z.gather(1, l[:, None])[:, 0] - torch.logsumexp(z, 1))
    return torch.cat(out)


def _head_inputs(case, g):
    dt, D, V = DTYPES[case["dtype"]], case["D"], case["V"]
    lead = (case["B"], 2, case["L"]) if case["kind"] == "preference" else (case["B"], case["L"])
    rows = math.prod(lead)

    def n(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    w = n(V, D) * (2 / math.sqrt(D))
    words = torch.randint(0, V, (rows,), generator=g, device="cuda")
    h = (n(rows, D) + 1.5 * w[words]).to(dt)
    w = w.to(dt)
    ignored = torch.rand(rows, generator=g, device="cuda") < case["ignored"]
    s = dict(hidden=h.view(*lead, D), weight=w, labels=torch.where(ignored, IGNORE, words).view(lead))
    if case["kind"] == "logp":
        return s
    logp = _log_probs_of(h, w, words, case.get("tau", 1.0)).view(lead)
    if case["kind"] == "preference":
        sums = torch.where(ignored.view(lead), 0, logp).double().sum(-1)
        s["ref"] = (sums + 3 * n(*lead[:-1]) - torch.tensor([1.0, 0.0], device="cuda")).float()
        s["dloss"] = torch.ones((), device="cuda") if case["mean"] else (0.5 + torch.rand(lead[:1], generator=g, device="cuda"))
        return s
    # The ratio keeps a thousandth away from both borders of the clipping, where the gradient jumps: on
    # which side a last bit puts a token is not what is measured.
    moved = 0.15 * n(*lead)
    for border in (math.log(1 - CLIP[0]), math.log(1 + CLIP[1])):
        moved = torch.where((moved - border).abs() < 1e-3, border + torch.where(moved < border, -2e-3, 2e-3), moved)
    s["old"] = logp - moved
    s["ref"] = logp - 0.2 * n(*lead) if case["kl"] else None
    # Most of what was sampled did better than the baseline: a mean over tokens that nearly cancel would
    # measure their last bits.
    s["advantages"] = 0.8 + 0.8 * (n(*lead) if case["by_token"] else n(case["B"], 1))
    s["dloss"] = torch.ones((), device="cuda") if case["mean"] else (0.5 + torch.rand(lead, generator=g, device="cuda")) / rows
    return s


def _clip_shapes(case, g):
    if case["flat"]:
        n = case["tensors"]
        cuts = torch.exp(3 * torch.randn(n, generator=g, device="cuda").double())
        sizes = (cuts / cuts.sum() * (case["values"] - n)).long().cpu() + 1
        sizes[-1] += case["values"] - int(sizes.sum())
        return [(int(v),) for v in sizes]
    D, V = case["D"], case["V"]
    layer = [(D, 3 * D), (D, D), (D,), (D,)]
    return [s for _ in range(case["layers"]) for s in layer] + [(V, D), (D,), (D,)]


def _clip_inputs(case, g):
    dt = DTYPES[case["dtype"]]
    shapes = _clip_shapes(case, g)
    total = sum(math.prod(s) for s in shapes)
    max_norm = 0.02 * math.sqrt(total) * (0.3 if case["clips"] else 3.0)   # values of about 0.02

    def grad(shape):
        other = torch.bfloat16 if case["dtype"] == "f32" else torch.float32
        t = 0.02 * torch.randn(shape, generator=g, device="cuda")
        return t.to(other if case["mixed"] and len(shape) == 1 else dt)

    if not case["flat"]:
        grads = [grad(s) for s in shapes]
        return dict(grads=grads, out=[torch.empty_like(t) for t in grads], max_norm=max_norm)
    flat = grad((total,))
    out = torch.empty_like(flat)
    sizes = [s[0] for s in shapes]
    return dict(flat_out=out, grads=list(flat.split(sizes)), out=list(out.split(sizes)), max_norm=max_norm)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 1_000_003 + 31)
    return _clip_inputs(case, g) if case["kind"] == "clip" else _head_inputs(case, g)


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] in ("policy", "preference"):
        s["hidden"].requires_grad_(True)
        s["weight"].requires_grad_(True)
    s["case"] = case
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    kind = s["case"]["kind"]
    if own and kind in ("policy", "preference"):
        return _framework(s)
    with torch.no_grad():
        if own:
            return _framework(s)
        return {"logp": _plain_logp, "policy": _plain_policy, "preference": _plain_preference, "clip": _plain_clip}[kind](s)


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-recurrence_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mlx_recurrence_amd
    return mlx_recurrence_amd


def _framework(s):
    mr, c = _package(), s["case"]
    if c["kind"] == "clip":
        norm = mr.clip_grad_norm(s["grads"], s["max_norm"], out=s["out"])
        return [norm, s["flat_out"]] if c["flat"] else [norm, *s["out"]]
    if c["kind"] == "logp":
        return mr.linear_log_probs(s["hidden"], s["weight"], s["labels"], temperature=c["tau"], ignore_index=IGNORE)
    reduction = "mean" if c["mean"] else "none"
    if c["kind"] == "policy":
        loss = mr.linear_policy_loss(s["hidden"], s["weight"], s["labels"], s["advantages"], s["old"], s["ref"], clip=CLIP,
                                     kl_weight=c["kl"], temperature=c["tau"], ignore_index=IGNORE, reduction=reduction)
    else:
        loss = mr.linear_preference_loss(s["hidden"], s["weight"], s["labels"], s["ref"], beta=c["beta"],
                                         label_smoothing=c["eps"], ignore_index=IGNORE, reduction=reduction)
    return (loss.detach(), *torch.autograd.grad(loss, (s["hidden"], s["weight"]), s["dloss"]))


def _plain_head(s, tau):
    """Hidden states and weight in 32 bits, which tokens count, their words, exp(z - max) with its sum, and
    the words' log-probabilities (0 for the others)."""
    D = s["weight"].shape[1]
    h, w, labels = s["hidden"].reshape(-1, D).float(), s["weight"].float(), s["labels"].reshape(-1)
    valid = labels != IGNORE
    at = torch.where(valid, labels, 0)[:, None]
    z = (h @ w.T) / tau
    m = z.max(1, keepdim=True).values
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True)
    logp = torch.where(valid, (z.gather(1, at) - m - torch.log(total))[:, 0], 0)
    return h, w, valid, at, e, total, logp


def _plain_logp(s):
    return _plain_head(s, s["case"]["tau"])[-1].view(s["labels"].shape)


def _plain_gradients(s, h, w, at, e, total, coef, tau):
    """From coef, the loss's derivative by each token's log-probability."""
    dz = e * (-coef[:, None] / (tau * total))
    dz.scatter_add_(1, at, coef[:, None] / tau)
    return (dz @ w).to(s["hidden"].dtype).view(s["hidden"].shape), (dz.T @ h).to(s["weight"].dtype)


def _plain_policy(s):
    c = s["case"]
    h, w, valid, at, e, total, logp = _plain_head(s, c["tau"])
    A = s["advantages"].expand(s["labels"].shape).reshape(-1)
    lo, hi = 1 - CLIP[0], 1 + CLIP[1]
    r = torch.exp(logp.double() - s["old"].reshape(-1).double())
    clipped = torch.where(A > 0, r > hi, r < lo)
    loss = -torch.minimum(r * A, r.clamp(lo, hi) * A)
    coef = torch.where(clipped, 0, -r * A)
    if c["kl"]:
        d = s["ref"].reshape(-1).double() - logp.double()
        loss = loss + c["kl"] * (torch.expm1(d) - d)
        coef = coef - c["kl"] * torch.expm1(d)
    loss = torch.where(valid, loss, 0)
    count = valid.sum().clamp(min=1) if c["mean"] else 1
    up = s["dloss"] / count if c["mean"] else s["dloss"].reshape(-1)
    coef = torch.where(valid, coef * up, 0).float()
    out = (loss.sum() / count if c["mean"] else loss.view(s["labels"].shape)).float()
    return (out, *_plain_gradients(s, h, w, at, e, total, coef, c["tau"]))


def _plain_preference(s):
    c = s["case"]
    h, w, valid, at, e, total, logp = _plain_head(s, 1.0)
    sums = logp.double().view(s["labels"].shape).sum(-1) - s["ref"].double()
    m = c["beta"] * (sums[:, 0] - sums[:, 1])
    counts = valid.view(c["B"], -1).any(1)

    def softplus(x):
        return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))

    loss = torch.where(counts, (1 - c["eps"]) * softplus(-m) + c["eps"] * softplus(m), 0)
    count = counts.sum().clamp(min=1) if c["mean"] else 1
    by_m = s["dloss"] / count * (c["eps"] / (1 + torch.exp(-m)) - (1 - c["eps"]) / (1 + torch.exp(m)))
    coef = c["beta"] * torch.stack([by_m, -by_m], 1)[:, :, None].expand(s["labels"].shape).reshape(-1)
    out = (loss.sum() / count if c["mean"] else loss).float()
    return (out, *_plain_gradients(s, h, w, at, e, total, torch.where(valid, coef, 0).float(), 1.0))


def _plain_clip(s):
    squares = [g.double().square().sum() for g in s["grads"]]
    norm = torch.stack(squares).sum().sqrt()
    factor = torch.where(norm > s["max_norm"], s["max_norm"] / norm, 1).float()
    out = [(g.float() * factor).to(g.dtype) for g in s["grads"]]
    return [norm.float(), torch.cat(out)] if s["case"]["flat"] else [norm.float(), *out]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    """Bytes: every input read once, every output written once.  Flops: for the losses the products alone,
    the logits forward and both gradients backward; for the clipping three a value."""
    e = ITEM[case["dtype"]]
    if case["kind"] == "clip":
        if case["flat"]:
            values, vectors = case["values"], 0
        else:
            D = case["D"]
            values, vectors = case["layers"] * 4 * D * D + case["V"] * D, (2 * case["layers"] + 2) * D
        other = (2 if e == 4 else 4) if case["mixed"] else e
        return dict(bytes=2 * (values * e + vectors * other), flops=3 * (values + vectors))
    D, V = case["D"], case["V"]
    rows = case["B"] * case["L"] * (2 if case["kind"] == "preference" else 1)
    both = (rows + V) * D * e
    if case["kind"] == "logp":
        return dict(bytes=both + rows * 12, flops=2 * rows * D * V)
    return dict(bytes=2 * both + rows * 24, flops=6 * rows * D * V)


# ------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "clip":
        flat = torch.cat([g.reshape(-1).double() for g in s["grads"]])
        norm = torch.linalg.vector_norm(flat)
        flat *= min(1.0, s["max_norm"] / float(norm))
        return [norm, flat] if case["flat"] else [norm, *(v.view(g.shape) for v, g in
                                                          zip(flat.split([g.numel() for g in s["grads"]]), s["grads"]))]
    grad = case["kind"] != "logp"
    hidden, weight = (s[k].double().requires_grad_(grad) for k in ("hidden", "weight"))
    rows = torch.nonzero(s["labels"].reshape(-1) != IGNORE)[:, 0]
    z = torch.matmul(hidden.flatten(0, -2)[rows], weight.t()) / case.get("tau", 1.0)
    picked = z.gather(1, s["labels"].reshape(-1)[rows][:, None])[:, 0] - torch.logsumexp(z, 1)
    logp = torch.zeros(s["labels"].numel(), dtype=torch.float64, device="cuda").index_put((rows,), picked)
    if not grad:
        return logp.view(s["labels"].shape)
    if case["kind"] == "policy":
        pick = lambda t: t.double().expand(s["labels"].shape).reshape(-1)[rows]  # noqa: E731
        A, ratio = pick(s["advantages"]), torch.exp(picked - pick(s["old"]))
        best = torch.where(A >= 0, torch.clamp(ratio, max=1 + CLIP[1]), torch.clamp(ratio, min=1 - CLIP[0]))
        each = -best * A
        if case["kl"]:
            gap = pick(s["ref"]) - picked
            each = each + case["kl"] * (gap.exp() - 1 - gap)
        loss = torch.zeros_like(logp).index_put((rows,), each).view(s["labels"].shape)
        out = loss.sum() / max(1, len(rows)) if case["mean"] else loss
    else:
        gap = logp.view(s["labels"].shape).sum(2) - s["ref"].double()
        m = case["beta"] * (gap[:, 0] - gap[:, 1])
        log_sigmoid = torch.nn.functional.logsigmoid
        loss = -(1 - case["eps"]) * log_sigmoid(m) - case["eps"] * log_sigmoid(-m)
        there = (s["labels"] != IGNORE).flatten(1).any(1)
        loss = loss * there
        out = loss.sum() / max(1, int(there.sum())) if case["mean"] else loss
    if not rows.numel():
        return (out.detach(), torch.zeros_like(hidden), torch.zeros_like(weight))
    return (out.detach(), *torch.autograd.grad(out, (hidden, weight), s["dloss"].double()))
