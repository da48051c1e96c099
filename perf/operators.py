"""Performance cases of the operators around a language model's output head: the norm in front of
it, the loss on labels and the loss on a teacher's top logits, both straight from hidden states.

Kinds and their ranges (`draw` spreads cases over them; `listed` holds several of each):

    norm      layer_norm, 1 to 32768 rows of 32 to 8192 channels; forward alone (decoding) or forward
              and backward with the weight's and the bias's gradient; fp32 rows may leave as bf16 (a
              scan returns fp32, the next product reads bf16)
    ce        linear_cross_entropy, 1 to 8192 rows of 32 to 5120 channels against a vocabulary of 500
              to 131072; forward alone (scoring) or forward and backward; some rows ignored
    distill   linear_distillation of the same sizes on a teacher's 1 to 128 top logits a row; rows
              with fewer entries, and rows with none

Hidden states are of unit variance with a part that points at the row's label (or at the teacher's
first entry), so that a row's softmax has a head and a long tail.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ITEM = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5
IGNORE = -100
Z_LOSS = 1e-4
MOST = 8192 * 2560 * 65536   # rows x channels x vocabulary of the largest case


def listed():
    return [
        # one decoded token of a wide model: latency
        dict(name="norm_token", kind="norm", dtype="bf16", out="bf16", rows=1, D=5120, grad=False),
        # one training layer of a small model (3 x 512 tokens)
        dict(name="norm_train_small", kind="norm", dtype="bf16", out="bf16", rows=1536, D=768, grad=True),
        # one training layer of a 2560-wide model (8 x 4096 tokens): bytes
        dict(name="norm_train_large", kind="norm", dtype="bf16", out="bf16", rows=32768, D=2560, grad=True),
        # a scan's fp32 output normed into bf16, at sizes that divide nothing
        dict(name="norm_ragged_f32", kind="norm", dtype="f32", out="bf16", rows=4099, D=1001, grad=True),
        # scoring the next token of a serving batch: the weight is read once
        dict(name="ce_score", kind="ce", dtype="bf16", rows=16, D=5120, V=65536, grad=False, ignored=0.0, mean=False,
             z=False),
        # the head of a small model at 3 x 512 tokens, a third of them a prompt that is not trained on
        dict(name="ce_train_small", kind="ce", dtype="bf16", rows=1536, D=768, V=32000, grad=True, ignored=0.33,
             mean=True, z=True),
        # the head of a 2560-wide model with a large vocabulary
        dict(name="ce_train_large", kind="ce", dtype="bf16", rows=8192, D=2560, V=65536, grad=True, ignored=0.02,
             mean=True, z=False),
        # fp32 training of a small model
        dict(name="ce_train_f32", kind="ce", dtype="f32", rows=1536, D=768, V=32000, grad=True, ignored=0.0, mean=True,
             z=False),
        # ragged in every size, a loss for each row
        dict(name="ce_ragged_f16", kind="ce", dtype="f16", rows=1001, D=1000, V=50021, grad=True, ignored=0.1,
             mean=False, z=True),
        # distillation of a 2560-wide student
        dict(name="distill_large", kind="distill", dtype="bf16", rows=4096, D=2560, V=65536, K=64, grad=True,
             absent=0.0, mean=True, tau=2.0),
        # a small student and a short batch
        dict(name="distill_small", kind="distill", dtype="bf16", rows=512, D=768, V=32000, K=16, grad=True, absent=0.1,
             mean=True, tau=1.0),
        # ragged in every size, rows with few entries and with none
        dict(name="distill_ragged", kind="distill", dtype="bf16", rows=777, D=513, V=10007, K=50, grad=True, absent=0.3,
             mean=False, tau=1.5),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _odd_or_even(rng, n, step):
    """Half of the sizes are multiples of `step`, as most models' are, half are left as drawn."""
    return max(step, n // step * step) if rng.random() < 0.5 else n


def draw(rng):
    kind = rng.choice(["norm", "ce", "distill"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
    grad = rng.random() < 0.75
    if kind == "norm":
        D = _odd_or_even(rng, _log_int(rng, 32, 8192), 64)
        rows = min(_log_int(rng, 1, 32768), 32768 * 2560 // D)
        out = rng.choice(["bf16", "f32"]) if dtype == "f32" else dtype
        return dict(kind=kind, dtype=dtype, out=out, rows=rows, D=D, grad=grad)
    D = _odd_or_even(rng, _log_int(rng, 32, 5120), 64)
    V = _odd_or_even(rng, _log_int(rng, 500, 131072), 64)
    rows = min(_log_int(rng, 1, 8192), 8192 * 65536 // V, MOST // (8 * D * V) if dtype == "f32" else MOST // (D * V))
    c = dict(kind=kind, dtype=dtype, rows=max(1, rows), D=D, V=V, grad=grad, mean=rng.random() < 0.6)
    if kind == "ce":
        c.update(ignored=rng.choice([0.0, 0.05, 0.4]), z=rng.random() < 0.4)
    else:
        c.update(K=_log_int(rng, 1, 128), absent=rng.choice([0.0, 0.0, 0.3]), tau=rng.choice([1.0, 1.5, 2.0, 4.0]))
    return c


# ------------------------------------------------------------------ inputs
def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 1_000_003 + 29)
    dt = DTYPES[case["dtype"]]
    rows, D = case["rows"], case["D"]

    def n(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def un(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    if case["kind"] == "norm":
        x = n(rows, D) * torch.exp(0.5 * n(rows, 1)) + 0.5 * n(1, D)
        param = torch.float32 if case["dtype"] == "f32" else dt
        return dict(x=x.to(dt), weight=(1 + 0.1 * n(D)).to(param), bias=(0.1 * n(D)).to(param),
                    dy=n(rows, D).to(DTYPES[case["out"]]))
    V = case["V"]
    w = n(V, D) * (2 / math.sqrt(D))
    s = {}
    if case["kind"] == "ce":
        first = torch.randint(0, V, (rows,), generator=g, device="cuda")
        s["labels"] = torch.where(un(rows) < case["ignored"], IGNORE, first)
    else:
        K = case["K"]
        offsets = torch.randperm(V, generator=g, device="cuda")[:K]
        first = torch.randint(0, V, (rows,), generator=g, device="cuda")
        ids = (first[:, None] + offsets[None] - offsets[0]) % V
        t = torch.sort(6 + 3 * n(rows, K), dim=1, descending=True).values
        short = un(rows) < case["absent"]
        have = torch.where(short, torch.randint(0, K, (rows,), generator=g, device="cuda"), K)
        gone = torch.arange(K, device="cuda")[None] >= have[:, None]
        s["ids"] = ids.masked_fill(gone, -1)
        s["teacher"] = t.masked_fill(gone, -math.inf).to(dt)
    s["hidden"] = (n(rows, D) + 1.5 * w[first]).to(dt)
    s["weight"] = w.to(dt)
    s["dloss"] = torch.ones((), device="cuda") if case["mean"] else un(rows) / rows
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["grad"]:
        for name in ("x", "hidden", "weight", "bias"):
            if name in s:
                s[name].requires_grad_(True)
    s["case"] = case
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        if s["case"]["grad"]:
            return _framework(s)
        with torch.no_grad():
            return _framework(s)
    with torch.no_grad():
        return {"norm": _plain_norm, "ce": _plain_ce, "distill": _plain_distill}[s["case"]["kind"]](s)


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-recurrence_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mlx_recurrence_amd
    return mlx_recurrence_amd


def _framework(s):
    mr, c = _package(), s["case"]
    if c["kind"] == "norm":
        y = mr.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, out_dtype=DTYPES[c["out"]])
        if not c["grad"]:
            return y
        return (y.detach(), *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"]))
    reduction = "mean" if c["mean"] else "none"
    if c["kind"] == "ce":
        loss = mr.linear_cross_entropy(s["hidden"], s["weight"], s["labels"], ignore_index=IGNORE,
                                       z_loss=Z_LOSS if c["z"] else 0.0, reduction=reduction)
    else:
        loss = mr.linear_distillation(s["hidden"], s["weight"], s["teacher"], s["ids"], temperature=c["tau"],
                                      reduction=reduction)
    if not c["grad"]:
        return loss
    return (loss.detach(), *torch.autograd.grad(loss, (s["hidden"], s["weight"]), s["dloss"]))


def _plain_norm(s):
    c = s["case"]
    x, w = s["x"].float(), s["weight"].float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = torch.rsqrt((d * d).mean(1, keepdim=True) + EPS)
    xhat = d * rstd
    y = (xhat * w + s["bias"].float()).to(DTYPES[c["out"]])
    if not c["grad"]:
        return y
    dy = s["dy"].float()
    gx = dy * w
    dx = rstd * (gx - gx.mean(1, keepdim=True) - xhat * (gx * xhat).mean(1, keepdim=True))
    return y, dx.to(s["x"].dtype), (dy * xhat).sum(0).to(s["weight"].dtype), dy.sum(0).to(s["bias"].dtype)


def _gradients(s, dz, h, w):
    return (dz @ w).to(s["hidden"].dtype), (dz.T @ h).to(s["weight"].dtype)


def _plain_ce(s):
    c = s["case"]
    h, w, labels = s["hidden"].float(), s["weight"].float(), s["labels"]
    valid = labels != IGNORE
    at = torch.where(valid, labels, 0)[:, None]
    zl = Z_LOSS if c["z"] else 0.0
    z = h @ w.T
    m = z.max(1, keepdim=True).values
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True)
    lse = m + torch.log(total)
    loss = torch.where(valid, (lse - z.gather(1, at) + zl * lse * lse)[:, 0], 0)
    count = valid.sum().clamp(min=1) if c["mean"] else 1
    out = loss.sum() / count if c["mean"] else loss
    if not c["grad"]:
        return out
    coef = torch.where(valid, s["dloss"] / count, 0)[:, None]
    dz = e * (coef * (1 + 2 * zl * lse) / total)
    dz.scatter_add_(1, at, -coef)
    return (out, *_gradients(s, dz, h, w))


def _plain_distill(s):
    c = s["case"]
    h, w, ids, tau = s["hidden"].float(), s["weight"].float(), s["ids"], c["tau"]
    there = ids >= 0
    valid = there.any(1, keepdim=True)
    at = torch.where(there, ids, 0)
    t = torch.where(there, s["teacher"].float() / tau, -math.inf)
    t = torch.exp(t - torch.where(valid, t.max(1, keepdim=True).values, 0))
    p = t / torch.where(valid, t.sum(1, keepdim=True), 1)
    z = (h @ w.T) / tau
    m = z.max(1, keepdim=True).values
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True)
    logq = z.gather(1, at) - m - torch.log(total)
    loss = tau * tau * torch.where(p > 0, p * (torch.log(torch.where(p > 0, p, 1)) - logq), 0).sum(1)
    count = valid.sum().clamp(min=1) if c["mean"] else 1
    out = loss.sum() / count if c["mean"] else loss
    if not c["grad"]:
        return out
    dloss = s["dloss"] if c["mean"] else s["dloss"][:, None]
    coef = torch.where(valid, tau * dloss / count, 0)
    dz = e * (coef / total)
    dz.scatter_add_(1, at, -coef * p)
    return (out, *_gradients(s, dz, h, w))


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    """Bytes: every input read once, every output written once.  Flops: for the losses the products
    alone, the logits forward and both gradients backward (a second product for the logits, which a
    backward that keeps no logits needs, is not counted); for the norm about 8 a value forward and 12
    backward."""
    e, rows, D = ITEM[case["dtype"]], case["rows"], case["D"]
    if case["kind"] == "norm":
        o = ITEM[case["out"]]
        if not case["grad"]:
            return dict(bytes=rows * D * (e + o) + 2 * D * e, flops=8 * rows * D)
        return dict(bytes=2 * rows * D * (e + o) + 4 * D * e, flops=20 * rows * D)
    V = case["V"]
    per_row = 8 if case["kind"] == "ce" else case["K"] * (8 + e)
    both = (rows + V) * D * e
    if not case["grad"]:
        return dict(bytes=both + rows * per_row + 4 * rows, flops=2 * rows * D * V)
    return dict(bytes=2 * both + rows * per_row + 8 * rows, flops=6 * rows * D * V)


# ------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    s = {k: v.double() if v.is_floating_point() else v for k, v in _inputs(case, seed).items()}
    leaves = [s[k].requires_grad_(True) for k in (("x", "weight", "bias") if case["kind"] == "norm" else
                                                  ("hidden", "weight"))]
    if case["kind"] == "norm":
        x = leaves[0]
        var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
        out, up = (x - mean) / torch.sqrt(var + EPS) * leaves[1] + leaves[2], s["dy"]
    else:
        tau = case.get("tau", 1.0)
        z = torch.matmul(leaves[0], leaves[1].t()) / tau
        lse = torch.logsumexp(z, 1)
        if case["kind"] == "ce":
            rows = torch.nonzero(s["labels"] != IGNORE)[:, 0]
            each = lse[rows] - z[rows, s["labels"][rows]] + (Z_LOSS if case["z"] else 0.0) * lse[rows].square()
            loss = torch.zeros_like(lse).index_put((rows,), each)
        else:
            rows = torch.nonzero((s["ids"] >= 0).any(1))[:, 0]
            logp = torch.log_softmax(torch.where(s["ids"] >= 0, s["teacher"], -math.inf)[rows] / tau, 1)
            logq = z[rows].gather(1, s["ids"][rows].clamp(min=0)) - lse[rows, None]
            each = torch.nn.functional.kl_div(logq, logp, reduction="none", log_target=True)
            each = torch.where(torch.isfinite(logp), each, 0.0).sum(1)
            loss = torch.zeros_like(lse).index_put((rows,), tau * tau * each)
        out, up = (loss.sum() / max(1, len(rows)) if case["mean"] else loss), s["dloss"]
    if not case["grad"]:
        return out.detach()
    return (out.detach(), *torch.autograd.grad(out, leaves, up))
