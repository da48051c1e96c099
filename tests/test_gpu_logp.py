"""Log-probabilities, policy loss and preference loss from hidden states on the GPU against 64-bit
formulas (tests/logp_oracle.py, on the same rounded inputs).

Two measures, |got - want| over want: of the largest elements, and of the 2-norms.
Bounds, from the arithmetic (u = half a unit in the last place of the output's type: 2^-8 bf16,
2^-11 fp16):
  16-bit gradients  the output's rounding and that of the logits' gradient, u each; tokens of one
                    sequence share a factor, so that the latter need not average out: 2-norm at
                    most 2 u, largest element at most 4 u (the sum's terms may exceed it).
  fp32 outputs      e = 2^-22 + 64 * 2^-24 = 4e-6 for log-probabilities (operands to 2^-22, sums of up to
                    2^16 terms), 2e-5 for the largest.  A ratio, and the derivative it gives, are off by
                    the log-probability's absolute error: times 1 + M, M the largest |logp|.  A sum over
                    the 2 L tokens of a pair, times beta, moves a pair's loss and derivative by at most
                    beta 2 L M e, or sqrt(2 L) in place of 2 L for independent errors: times
                    1 + beta sqrt(2 L) M.
                    A row's gradient is c (q - 1) at its word.  log2 q is a difference of two fp32 values of
                    the size of lse (below 33 here), so q is off by up to 2^-23 * 33 = 4e-6 of 1, however
                    small 1 - q is: times |c| / |c (1 - q)| over the rows, the oracle's fourth value.
"""
from __future__ import annotations

import math

import pytest
import torch

import mlx_recurrence_amd as mr
from mlx_recurrence_amd import _lib
from tests import logp_oracle as orc

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = {BF16: 2.0 ** -8, F16: 2.0 ** -11}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def rand(g, *shape):
    return torch.rand(shape, generator=g, device="cuda")


def check(name, got, want, times=1.0):
    assert got.dtype in (F32, BF16, F16) and got.shape == want.shape, name
    g, w = got.detach().double(), want.detach().double()
    assert torch.equal(torch.isnan(g), torch.isnan(w)), f"{name}: NaN elsewhere"
    g, w = torch.nan_to_num(g, nan=0.0), torch.nan_to_num(w, nan=0.0)
    if not w.numel():
        return
    diff = (g - w).abs()
    if got.dtype == F16:   # less than half of the type's least step is no error: the nearest value is that far off
        diff = diff * (diff > 2.0 ** -25)
    big = float(diff.max() / (w.abs().max() + 1e-30)) if float(diff.max()) else 0.0
    rel = float(torch.linalg.norm(diff) / (torch.linalg.norm(w) + 1e-30)) if big else 0.0
    most, norm = (4 * U[got.dtype], 2 * U[got.dtype]) if got.dtype in U else (2e-5 * times, 4e-6 * times)
    assert big <= most and rel <= norm, f"{name}: largest {big:.2e} (<= {most:.1e}), 2-norm {rel:.2e} (<= {norm:.1e})"


def head(lead, D, V, dtype, seed, ignored=0.25, size=2.0):
    """Generator, hidden states, weight, labels and the model's own log-probabilities."""
    g = gen(seed)
    rows = math.prod(lead)
    w = randn(g, V, D) * (size / math.sqrt(D))
    words = torch.randint(0, V, (rows,), generator=g, device="cuda")
    h, w = (randn(g, rows, D) + 0.5 * w[words]).to(dtype), w.to(dtype)
    labels = torch.where(rand(g, rows) < ignored, -100, words).view(lead)
    logp = orc.log_probs(h.view(*lead, D), w, words.view(lead), torch.zeros(lead, device="cuda"))[0]
    return g, h.view(*lead, D), w, labels, logp


def away(moved, clip):
    """Log-ratios moved off the borders of the clipping, where the gradient jumps."""
    for b in (math.log1p(-clip[0]), math.log1p(clip[1])):
        moved = torch.where((moved - b).abs() < 1e-3, b + torch.where(moved < b, -2e-3, 2e-3), moved)
    return moved


def run(fn, h, w, up, *args, **kw):
    h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = fn(h, w, *args, **kw)
    return (loss.detach(), *torch.autograd.grad(loss, (h, w), up))


def check_all(got, want, times=1.0):
    for name, a, e in zip(("loss", "dhidden", "dweight"), got, want):
        check(name, a, e, times if name == "loss" else times * want[3])


SIZES = [((1,), 1, 1), ((1,), 8, 2), ((2,), 7, 3), ((1, 1), 64, 1000), ((3,), 65, 127), ((31, 1), 64, 128), ((4, 8), 40, 129),
         ((3, 11), 72, 255), ((64,), 128, 256), ((5, 13), 200, 257), ((127,), 96, 1000), ((2, 2, 32), 256, 513),
         ((129,), 33, 2000), ((15, 17), 264, 700), ((257,), 257, 1300), ((3, 100), 1000, 5003), ((7, 100), 320, 4096)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lead,D,V", SIZES)
def test_log_probs(lead, D, V, dtype):
    g, h, w, labels, _ = head(lead, D, V, dtype, 31 * D + 7 * V + len(lead))
    up = randn(g, *lead)
    tau = 0.7 if D % 2 else 1.0
    got = run(mr.linear_log_probs, h, w, up, labels, temperature=tau)
    want = orc.log_probs(h, w, labels, up, tau=tau)
    if V == 1:   # log-probability 0 and no gradient, but for roundings
        assert all(float(t.abs().max()) <= 1e-6 for t in got)
        return
    check_all(got, want)
    with torch.no_grad():
        assert torch.equal(mr.linear_log_probs(h, w, labels, temperature=tau), got[0])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lead,D,V", SIZES)
@pytest.mark.parametrize("kl,by_token", [(0.0, False), (0.1, True)])
def test_policy_loss(lead, D, V, dtype, kl, by_token):
    g, h, w, labels, logp = head(lead, D, V, dtype, 37 * D + 11 * V + len(lead) + by_token)
    clip = (0.2, 0.3)
    old = (logp - away(0.3 * randn(g, *lead), clip)).float()
    ref = (logp - 0.3 * randn(g, *lead)).float()
    A = randn(g, *lead) if by_token else randn(g, *lead[:-1], 1)
    up = rand(g, *lead) + 0.1
    got = run(mr.linear_policy_loss, h, w, up, labels, A, old, ref, clip=clip, kl_weight=kl, reduction="none")
    want = orc.policy(h, w, labels, A, old, ref, up, clip=clip, kl=kl, reduction="none")
    M = 1 + orc.size_of(h, w, labels)
    check("loss", got[0], want[0], M)
    if V == 1:
        assert all(float(t.abs().max()) <= 1e-5 for t in got[1:])
        return
    check_all(got, want, M)


PAIRS = [((1,), 1, 1, 2), ((1,), 1, 8, 2), ((2,), 3, 7, 30), ((1,), 40, 64, 1000), ((3,), 5, 65, 127), ((2, 2), 16, 40, 129),
         ((33,), 1, 72, 255), ((4,), 129, 64, 300), ((5,), 127, 200, 257), ((1,), 300, 96, 1000), ((16,), 20, 320, 4096)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lead,L,D,V", PAIRS)
@pytest.mark.parametrize("eps,use_ref", [(0.0, True), (0.1, False)])
def test_preference_loss(lead, L, D, V, dtype, eps, use_ref):
    g, h, w, labels, logp = head((*lead, 2, L), D, V, dtype, 41 * D + 13 * V + L)
    beta = 0.1
    S = torch.where(labels != -100, logp, 0).sum(-1)
    ref = (S + 5 * randn(g, *lead, 2)).float() if use_ref else None
    up = rand(g, *lead) + 0.1
    got = run(mr.linear_preference_loss, h, w, up, labels, ref, beta=beta, label_smoothing=eps, reduction="none")
    want = orc.preference(h, w, labels, ref, up, beta=beta, eps=eps, reduction="none")
    check_all(got, want, 1 + beta * math.sqrt(2 * L) * orc.size_of(h, w, labels))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_reductions_and_label_types(dtype, reduction):
    """An ignored label of its own, int32 labels, 64-bit and 16-bit advantages, one width for both sides."""
    g, h, w, labels, logp = head((3, 20), 48, 333, dtype, 8)
    labels = torch.where(labels == -100, -1, labels)
    old = (logp - away(0.3 * randn(g, 3, 20), (0.25, 0.25))).float()
    A = (randn(g, 3, 20) + 1).to(BF16)
    up = rand(g, 3, 20) if reduction == "none" else torch.tensor(0.7, device="cuda")
    got = run(mr.linear_policy_loss, h, w, up, labels.int(), A, old.double(), clip=0.25, ignore_index=-1, temperature=1,
              reduction=reduction)
    want = orc.policy(h, w, labels, A, old, None, up, clip=(0.25, 0.25), ignore=-1, reduction=reduction)
    check_all(got, want, 4 * (1 + orc.size_of(h, w, labels, ignore=-1)))   # (most advantages are positive: their mean is no fourth of the mean of their sizes)
    g, h, w, labels, logp = head((2, 3, 2, 10), 48, 333, dtype, 9)
    labels[1, 2] = -100   # a pair that counts for nothing
    up = rand(g, 2, 3) if reduction == "none" else torch.tensor(0.7, device="cuda")
    got = run(mr.linear_preference_loss, h, w, up, labels.short(), beta=0.3, reduction=reduction)
    want = orc.preference(h, w, labels, None, up, beta=0.3, reduction=reduction)
    assert got[0].shape == ((2, 3) if reduction == "none" else ())
    check_all(got, want, 1 + 0.3 * math.sqrt(20) * orc.size_of(h, w, labels))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_policy_of_this_step(dtype):
    """Without old log-probabilities the ratio is 1 and its gradient that of logp."""
    g, h, w, labels, logp = head((4, 30), 96, 500, dtype, 3)
    A = randn(g, 4, 1)
    ref = (logp - 0.2 * randn(g, 4, 30)).float()
    up = rand(g, 4, 30)
    got = run(mr.linear_policy_loss, h, w, up, labels, A, None, ref, kl_weight=0.05, reduction="none")
    check_all(got, orc.policy(h, w, labels, A, None, ref, up, kl=0.05, reduction="none"), 1 + orc.size_of(h, w, labels))


def test_borders_and_infinite_widths():
    """A ratio of exactly 1 on a border of width 0 is inside; infinite widths do not clip; no advantage, no loss."""
    g, h, w, labels, _ = head((40,), 64, 300, F32, 5, ignored=0.0)
    with torch.no_grad():
        own = mr.linear_log_probs(h, w, labels)
    A = torch.where(torch.arange(40, device="cuda") % 2 == 0, 1.5, -0.5)
    up = torch.ones(40, device="cuda")
    a = run(mr.linear_policy_loss, h, w, up, labels, A, own, clip=0.0, reduction="none")
    b = run(mr.linear_policy_loss, h, w, up, labels, A, None, clip=0.0, reduction="none")
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(a[0], -A)
    old = own - 3 * randn(g, 40).sign()
    got = run(mr.linear_policy_loss, h, w, up, labels, A, old, clip=math.inf, reduction="none")
    check_all(got, orc.policy(h, w, labels, A, old, None, up, clip=(1e30, 1e30), reduction="none"),
              1 + orc.size_of(h, w, labels))
    far = own - 500   # the ratio is beyond fp32
    got = run(mr.linear_policy_loss, h, w, up, labels, torch.zeros(40, device="cuda"), far, reduction="none")
    assert not any(t.any() for t in got)
    got = run(mr.linear_policy_loss, h, w, up, labels, A.abs(), far, clip=(0.2, 0.4), reduction="none")
    assert torch.equal(got[0], -1.4 * A.abs()) and not got[1].any() and not got[2].any()


def test_far_and_near_references():
    """The KL term of nearly equal and of far apart log-probabilities."""
    g, h, w, labels, _ = head((64,), 64, 300, F32, 6, ignored=0.0)
    with torch.no_grad():
        own = mr.linear_log_probs(h, w, labels)
    d = torch.logspace(-3, 1.2, 64, device="cuda") * torch.where(torch.arange(64, device="cuda") % 2 == 0, 1, -1)
    ref = own + d
    up = torch.ones(64, device="cuda")
    zero = torch.zeros(64, device="cuda")
    got = run(mr.linear_policy_loss, h, w, up, labels, zero, own, ref, kl_weight=1.0, reduction="none")
    want = orc.policy(h, w, labels, zero, own, ref, up, kl=1.0, reduction="none")
    # an absolute error M e of a log-probability moves exp(d) - d - 1 by |exp(d) - 1| times that
    off = (got[0].double() - want[0]).abs()
    e = 2e-5 * (1 + orc.size_of(h, w, labels))
    assert bool((off <= e * torch.expm1(d.double()).abs() + 1e-6 * want[0]).all())
    check_all(got, want, 1 + orc.size_of(h, w, labels))
    with torch.no_grad():
        assert not mr.linear_policy_loss(h, w, labels, zero, own, own, kl_weight=1.0).any()
        assert torch.isinf(mr.linear_policy_loss(h, w, labels, zero, own, own - math.inf, kl_weight=1.0))


def test_sure_and_hopeless_pairs():
    """Margins of hundreds: the loss is the margin or nothing, its derivative beta or nothing."""
    g, h, w, labels, logp = head((2, 2, 30), 64, 300, F32, 7, ignored=0.0)
    S = logp.sum(-1)
    gap = torch.tensor([[900.0, 0.0], [-900.0, 0.0]], device="cuda")
    ref = (S - gap).float()
    up = torch.ones(2, device="cuda")
    got = run(mr.linear_preference_loss, h, w, up, labels, ref, beta=1.0, reduction="none")
    assert float(got[0][0]) == 0.0 and not got[1][0].any()
    want = orc.preference(h, w, labels, ref, up, beta=1.0, reduction="none")
    check_all(got, want, 1 + math.sqrt(60) * orc.size_of(h, w, labels))
    got = run(mr.linear_preference_loss, h, w, up, labels, ref, beta=1.0, label_smoothing=0.5, reduction="none")
    check_all(got, orc.preference(h, w, labels, ref, up, beta=1.0, eps=0.5, reduction="none"),
              1 + math.sqrt(60) * orc.size_of(h, w, labels))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rows_that_do_not_count_are_not_read(dtype):
    g, h, w, labels, logp = head((5, 30), 64, 500, dtype, 3, ignored=0.5)
    labels[2] = -100
    out = labels == -100
    old, ref, A = (logp - 0.1).float(), (logp + 0.1).float(), randn(g, 5, 30)
    one = torch.ones((), device="cuda")
    clean = run(mr.linear_policy_loss, h, w, one, labels, A, old, ref, kl_weight=0.1)
    h2, old2, ref2, A2 = h.clone(), old.clone(), ref.clone(), A.clone()
    for t in (h2, old2, ref2, A2):
        t[out] = math.nan
    again = run(mr.linear_policy_loss, h2, w, one, labels, A2, old2, ref2, kl_weight=0.1)
    assert all(torch.equal(a, b) for a, b in zip(clean, again)) and not again[1][out].any()
    got = run(mr.linear_log_probs, h2, w, torch.ones(5, 30, device="cuda"), labels)
    assert not got[0][out].any() and not got[1][out].any() and torch.isfinite(got[2]).all()
    hp, lp = h2.view(1, 5, 30, 64)[:, :2].contiguous(), labels[:2].view(1, 2, 30)
    got = run(mr.linear_preference_loss, hp, w, one, lp)
    check_all(got, orc.preference(hp, w, lp, None, one), 1 + 0.1 * math.sqrt(60) * orc.size_of(hp, w, lp))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_no_row_counts(dtype):
    h = torch.full((2, 2, 6, 64), math.nan, device="cuda", dtype=dtype)
    w = torch.randn(100, 64, device="cuda").to(dtype)
    labels = torch.full((2, 2, 6), -100, device="cuda")
    A = torch.full((2, 2, 6), math.nan, device="cuda")
    for reduction in ("mean", "sum", "none"):
        lead = (2, 2, 6) if reduction == "none" else ()
        for up in (1.0, math.inf):
            assert not any(t.any() for t in run(mr.linear_policy_loss, h, w, torch.full(lead, up, device="cuda"), labels, A, A, A,
                                                kl_weight=0.1, reduction=reduction))
            pairs = (2,) if reduction == "none" else ()
            assert not any(t.any() for t in run(mr.linear_preference_loss, h, w, torch.full(pairs, up, device="cuda"), labels,
                                                A[..., 0], reduction=reduction))
    assert not any(t.any() for t in run(mr.linear_log_probs, h, w, torch.ones(2, 2, 6, device="cuda"), labels))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_no_rows(dtype):
    w = torch.randn(50, 24, device="cuda").to(dtype)
    none = torch.zeros(0, 7, dtype=torch.int64, device="cuda")
    h = torch.zeros(0, 7, 24, device="cuda", dtype=dtype)
    loss, dh, dw = run(mr.linear_policy_loss, h, w, torch.ones((), device="cuda"), none, torch.zeros(0, 1, device="cuda"))
    assert float(loss) == 0 and dh.shape == h.shape and not dw.any()
    out, dh, dw = run(mr.linear_log_probs, h, w, torch.zeros(0, 7, device="cuda"), none)
    assert out.shape == (0, 7) and dh.shape == h.shape and not dw.any()
    h, none = torch.zeros(3, 2, 0, 24, device="cuda", dtype=dtype), torch.zeros(3, 2, 0, dtype=torch.int64, device="cuda")
    for reduction, shape in (("none", (3,)), ("mean", ()), ("sum", ())):
        loss, dh, dw = run(mr.linear_preference_loss, h, w, torch.ones(shape, device="cuda"), none, reduction=reduction)
        assert loss.shape == shape and not loss.any() and dh.shape == h.shape and not dw.any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_labels_out_of_range_and_values_that_are_not_finite(dtype):
    g, h, w, labels, logp = head((6, 2, 5), 40, 200, dtype, 4, ignored=0.0)
    labels[0, 0, 1], labels[1, 1, 0] = 200, -7
    h[2, 0, 3, 5] = math.nan
    bad = [(0, 0, 1), (1, 1, 0), (2, 0, 3)]
    ones = torch.ones(6, 2, 5, device="cuda")
    out, dh, dw = run(mr.linear_log_probs, h, w, ones, labels)
    nan = torch.zeros(6, 2, 5, dtype=torch.bool, device="cuda")
    for at in bad:
        nan[at] = True
    assert torch.equal(torch.isnan(out), nan) and torch.equal(torch.isnan(dh).all(-1), nan) and torch.isnan(dw).all()
    out, dh, _ = run(mr.linear_policy_loss, h, w, ones, labels, ones, logp.float(), reduction="none")
    assert torch.equal(torch.isnan(out), nan) and torch.equal(torch.isnan(dh).all(-1), nan)
    out, dh, _ = run(mr.linear_preference_loss, h, w, ones[:, 0, 0], labels, reduction="none")
    pairs = torch.arange(6, device="cuda") < 3
    assert torch.equal(torch.isnan(out), pairs) and torch.equal(torch.isnan(dh).flatten(1).all(1), pairs)
    fine = slice(3, 6)
    check("loss", out[fine], orc.preference(h[fine], w, labels[fine], None, ones[fine, 0, 0], reduction="none")[0],
          1 + 0.1 * math.sqrt(10) * orc.size_of(h[fine], w, labels[fine]))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_upstream_gradients_and_advantages_of_many_sizes(dtype):
    """Each row's gradient keeps its bits beside rows whose gradients are a million times larger."""
    g, h, w, labels, logp = head((300,), 64, 500, dtype, 14, ignored=0.0)
    A = randn(g, 300) * torch.logspace(-4, 2, 300, device="cuda")
    up = torch.ones((), device="cuda")
    loss, dh, _ = run(mr.linear_policy_loss, h, w, up, labels, A, None, reduction="sum")
    want = orc.policy(h, w, labels, A, None, None, up, reduction="sum")[1]
    rel = torch.linalg.norm(dh.double() - want, dim=1) / torch.linalg.norm(want, dim=1)
    big = torch.linalg.norm(want, dim=1) > (1e-2 if dtype == F16 else 0)   # below, fp16's own least steps
    assert float(rel[big].max()) <= 2 * U[dtype]


def test_two_layouts_of_one_call():
    """Strided hidden states and weight, a weight of another type, a batch of one token."""
    g, h, w, labels, logp = head((4, 12), 72, 300, F32, 15)
    A = randn(g, 4, 12)
    up = torch.ones((), device="cuda")
    want = run(mr.linear_policy_loss, h, w, up, labels, A, None)
    h2 = h.transpose(0, 1).contiguous().transpose(0, 1)
    w2 = w.T.contiguous().T
    A2 = A.T.contiguous().T
    l2 = labels.T.contiguous().T
    assert all(torch.equal(a, b) for a, b in zip(run(mr.linear_policy_loss, h2, w2, up, l2, A2, None), want))
    hb = h.to(BF16)
    got = run(mr.linear_policy_loss, hb, w, up, labels, A, None)
    assert got[1].dtype == BF16 and got[2].dtype == F32
    check("loss", got[0], orc.policy(hb, w, labels, A, None, None, up)[0], 8 * (1 + orc.size_of(hb, w, labels)))
    token = run(mr.linear_log_probs, h[0, 0], w, torch.ones((), device="cuda"), torch.tensor(5, device="cuda"))
    check("logp", token[0], orc.log_probs(h[0, 0], w, torch.tensor([5], device="cuda"), torch.ones(1, device="cuda"))[0][0])
    assert token[0].shape == () and token[1].shape == (72,)


def test_keep_logits_is_the_same_result():
    for dtype in (F32, BF16):
        g, h, w, labels, logp = head((5, 2, 64), 1030, 700, dtype, 16)
        up = torch.ones((), device="cuda")
        a = run(mr.linear_preference_loss, h, w, up, labels, keep_logits=True)
        b = run(mr.linear_preference_loss, h, w, up, labels, keep_logits=False)
        assert torch.equal(a[0], b[0])
        check_all(b, orc.preference(h, w, labels, None, up), 1 + 0.1 * math.sqrt(128) * orc.size_of(h, w, labels))


def test_only_what_is_wanted_and_once():
    g, h, w, labels, logp = head((40,), 64, 300, F32, 17)
    A = randn(g, 40).requires_grad_(True)
    old = logp.float().requires_grad_(True)
    whole = run(mr.linear_policy_loss, h, w, torch.ones((), device="cuda"), labels, A.detach(), old.detach())
    for which in (0, 1):
        ins = [h, w]
        ins[which] = ins[which].clone().requires_grad_(True)
        loss = mr.linear_policy_loss(*ins, labels, A, old)
        loss.backward()
        assert torch.equal(ins[which].grad, whole[1 + which]) and A.grad is None and old.grad is None
    hh = h.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(mr.linear_log_probs(hh, w, labels).sum(), hh, create_graph=True)


def test_python_binding_gives_the_same(monkeypatch):
    g, h, w, labels, logp = head((3, 2, 20), 96, 700, BF16, 18)
    A, old, ref = randn(g, 3, 2, 1), (logp - 0.1).float(), (logp + 0.1).float()
    up = torch.ones((), device="cuda")
    calls = ((mr.linear_policy_loss, up, (labels, A, old, ref), dict(kl_weight=0.1)),
             (mr.linear_preference_loss, up, (labels, ref.sum(-1)), dict(label_smoothing=0.1)),
             (mr.linear_log_probs, torch.ones(3, 2, 20, device="cuda"), (labels,), dict(temperature=0.5)))
    first = [run(fn, h, w, u, *a, **kw) for fn, u, a, kw in calls]
    monkeypatch.setattr(_lib, "_autograd_mod", None)
    for (fn, u, a, kw), want in zip(calls, first):
        assert all(torch.equal(x, y) for x, y in zip(run(fn, h, w, u, *a, **kw), want))


def test_more_rows_than_one_piece():
    """Two pieces of the vocabulary, several tiles of rows, sequences longer than a workgroup."""
    g, h, w, labels, logp = head((2, 2, 2048), 72, 70000, BF16, 12, ignored=0.1)
    up = torch.ones((), device="cuda")
    ref = (torch.where(labels != -100, logp, 0).sum(-1) + randn(g, 2, 2)).float()
    got = run(mr.linear_preference_loss, h, w, up, labels, ref)
    check_all(got, orc.preference(h, w, labels, ref, up), 1 + 0.1 * math.sqrt(4096) * orc.size_of(h, w, labels))
    A = randn(g, 2, 2, 1) + 2
    old = (logp + 0.05).float()
    got = run(mr.linear_policy_loss, h, w, up, labels, A, old)
    check_all(got, orc.policy(h, w, labels, A, old, None, up), 1 + orc.size_of(h, w, labels))


def test_other_streams_and_replays():
    """On a stream of its own, and as a graph replayed on new inputs between eager calls."""
    g, h, w, labels, logp = head((4, 2, 16), 128, 600, BF16, 19)
    A, old, ref = randn(g, 4, 2, 1), (logp - 0.1).float(), (logp + 0.1).float()
    h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(True)

    def step():
        policy = mr.linear_policy_loss(h, w, labels, A, old, ref, kl_weight=0.1)
        pairs = mr.linear_preference_loss(h, w, labels, ref.sum(-1))
        return (policy.detach(), pairs.detach(), *torch.autograd.grad(policy + pairs, (h, w)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            out = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(out, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for seed in range(3):
        with torch.no_grad():
            h.copy_(randn(gen(seed), 4, 2, 16, 128))
            A.copy_(randn(gen(seed + 9), 4, 2, 1))
        graph.replay()
        got = [t.clone() for t in static]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("pairs,L", [(1, 1), (3, 40), (17, 9), (64, 16), (40, 30), (7, 200)])
def test_pairs_in_one_launch_and_in_two(pairs, L, dtype, reduction):
    """Up to 2048 tokens and more; pairs that count for nothing among them; factors shared by a sequence."""
    g, h, w, labels, logp = head((pairs, 2, L), 72, 300, dtype, 3 * pairs + L, ignored=0.2)
    labels[1::5] = -100
    ref = (torch.where(labels != -100, logp, 0).sum(-1) + 4 * randn(g, pairs, 2)).float()
    up = rand(g, pairs) + 0.1 if reduction == "none" else torch.tensor(0.7, device="cuda")
    got = run(mr.linear_preference_loss, h, w, up, labels, ref, label_smoothing=0.05, reduction=reduction)
    want = orc.preference(h, w, labels, ref, up, eps=0.05, reduction=reduction)
    check_all(got, want, 1 + 0.1 * math.sqrt(2 * L) * orc.size_of(h, w, labels))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("rows", [2047, 2048, 2049, 3000])
def test_rows_found_in_one_launch_and_in_two(rows, dtype, reduction):
    g, h, w, labels, logp = head((rows,), 130, 640, dtype, rows, ignored=0.4)
    labels[-1] = -100 if rows % 2 else 3
    A = randn(g, rows) + 1
    old = (logp - away(0.3 * randn(g, rows), (0.2, 0.2))).float()
    up = rand(g, rows) + 0.1 if reduction == "none" else torch.tensor(0.7, device="cuda")
    got = run(mr.linear_policy_loss, h, w, up, labels, A, old, reduction=reduction)
    check_all(got, orc.policy(h, w, labels, A, old, None, up, reduction=reduction), 1 + orc.size_of(h, w, labels))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("pairs,L,D,V", [(1, 1, 8, 2), (2, 5, 200, 257), (1, 25, 3000, 300), (4, 25, 100, 513), (3, 50, 1000, 5003),
                                         (5, 70, 320, 4096), (25, 60, 200, 641)])
def test_kernels_write_inside_their_buffers(pairs, L, D, V, dtype, monkeypatch):
    """State and workspaces of exactly the stated sizes between guards: nothing is written outside them, and
    what they held before does not matter."""
    buffers = []

    def guarded(n, device):
        whole = torch.full((n + 8192,), 0xA5, dtype=torch.uint8, device=device)
        whole[4096:4096 + n] = 0xFF   # NaN as a float
        buffers.append((whole, n))
        return whole[4096:4096 + n]

    g, h, w, labels, logp = head((pairs, 2, L), D, V, dtype, pairs + D + V, ignored=0.3)
    A, old = randn(g, pairs, 2, 1), logp.float()
    one = torch.ones((), device="cuda")
    each = rand(g, pairs, 2, L)

    def calls():
        return (run(mr.linear_policy_loss, h, w, one, labels, A, old, old, kl_weight=0.1),
                run(mr.linear_policy_loss, h, w, each, labels, A, reduction="none"),
                run(mr.linear_preference_loss, h, w, one, labels),
                run(mr.linear_preference_loss, h, w, each[:, 0, 0], labels, reduction="none"),
                run(mr.linear_log_probs, h, w, each, labels))

    want = calls()
    monkeypatch.setattr(_lib, "autograd_ext", lambda: None)
    monkeypatch.setattr(_lib, "_alloc_ws", guarded)
    for a, b in zip(calls(), want):
        for x, y in zip(a, b):
            assert torch.equal(x, y)
    assert len(buffers) == 15
    for whole, n in buffers:
        assert (whole[:4096] == 0xA5).all() and (whole[4096 + n:] == 0xA5).all()


def test_dweight_made_whole_in_fp32_writes_inside_its_buffers(monkeypatch):
    """460 rows of 512 channels: the workspace holds no parts of dweight, which is made whole on small tiles."""
    buffers = []

    def guarded(n, device):
        whole = torch.full((n + 8192,), 0xA5, dtype=torch.uint8, device=device)
        whole[4096:4096 + n] = 0xFF
        buffers.append((whole, n))
        return whole[4096:4096 + n]

    g, h, w, labels, logp = head((4, 115), 512, 16001, F32, 26, ignored=0.1)
    A, up = randn(g, 4, 1), torch.ones((), device="cuda")
    monkeypatch.setattr(_lib, "autograd_ext", lambda: None)
    monkeypatch.setattr(_lib, "_alloc_ws", guarded)
    got = run(mr.linear_policy_loss, h, w, up, labels, A, logp.float())
    check_all(got, orc.policy(h, w, labels, A, logp.float(), None, up), 1 + orc.size_of(h, w, labels))
    assert len(buffers) == 3
    for whole, n in buffers:
        assert (whole[:4096] == 0xA5).all() and (whole[4096 + n:] == 0xA5).all()


def test_backward_twice_and_two_calls_at_once():
    """A graph kept for a second backward gives the same; calls on two streams share nothing."""
    g, h, w, labels, logp = head((6, 2, 32), 256, 1000, BF16, 21)
    A, old = randn(g, 6, 2, 1), (logp - 0.1).float()
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    loss = mr.linear_policy_loss(h, w, labels, A, old)
    first = torch.autograd.grad(loss, (h, w), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(loss, (h, w))))
    want = mr.linear_preference_loss(h, w, labels)
    want = (want.detach(), *torch.autograd.grad(want, (h, w)))
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                loss = mr.linear_policy_loss(h, w, labels, A, old) if i == 0 else mr.linear_preference_loss(h, w, labels)
                got[i] = (loss.detach(), *torch.autograd.grad(loss, (h, w)))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got[0][1:], first))
    assert all(torch.equal(a, b) for a, b in zip(got[1], want))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("moved", [30.0, 80.0, 87.0])
def test_a_row_far_from_its_old_policy_leaves_the_others(dtype, moved):
    """A ratio of up to e^87 (a negative advantage does not clip it): the other rows' gradients keep their bits."""
    g, h, w, labels, logp = head((64,), 64, 500, dtype, 23, ignored=0.0)
    old = logp.clone()
    old[5] -= moved
    A = torch.full((64,), -1.0, device="cuda")
    up = torch.ones((), device="cuda")
    loss, dh, _ = run(mr.linear_policy_loss, h, w, up, labels, A, old.float(), reduction="sum")
    want = orc.policy(h, w, labels, A, old.float(), None, up, reduction="sum")
    rest = [i for i in range(64) if i != 5]
    check("dhidden", dh[rest], want[1][rest], (1 + orc.size_of(h, w, labels)) * want[3])
    rel = float((dh[5].double() - want[1][5]).norm() / want[1][5].norm())
    assert rel <= (2 * U[dtype] if dtype in U else 1e-3)


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_reference_sums_in_64_bits(reduction, python, monkeypatch):
    """Sums of 2^17, which differ by what fp32 cannot hold beside them."""
    if python:
        monkeypatch.setattr(_lib, "_autograd_mod", None)
        monkeypatch.setattr(_lib, "autograd_ext", lambda: None)
    g, h, w, labels, logp = head((5, 2, 12), 64, 300, F32, 25)
    ref = torch.where(labels != -100, logp, 0).sum(-1) + 2 * randn(g, 5, 2) - 2.0 ** 17
    assert ref.dtype == torch.float64
    up = rand(g, 5) + 0.1 if reduction == "none" else torch.ones((), device="cuda")
    got = run(mr.linear_preference_loss, h, w, up, labels, ref, beta=0.5, reduction=reduction)
    want = orc.preference(h, w, labels, ref, up, beta=0.5, reduction=reduction)
    check_all(got, want, 1 + 0.5 * math.sqrt(24) * orc.size_of(h, w, labels))


# Rows (a fifth ignored), channels, words.  dhidden has 17 x 18 tiles of 256 x 256 for 4400 rows of 4200 channels, 5 x 105 of
# 256 x 64 for 6720 of 1100 in fp32: more than the 256 (512) that run at one time, so that some tiles are made whole and
# the others in parts.  The last of each type keeps more than 256 MiB of logits, in two pieces of the vocabulary or three.
LARGE = [(BF16, 5500, 4200, 1001), (F16, 5500, 4200, 1001), (F32, 8400, 1100, 301),
         (BF16, 5500, 4200, 60000), (F16, 5500, 4200, 60000), (F32, 8400, 1100, 40000)]


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("dtype,rows,D,V", LARGE)
def test_more_tiles_than_run_at_one_time(dtype, rows, D, V, reduction):
    g, h, w, labels, logp = head((rows,), D, V, dtype, rows + V, ignored=0.2)
    A = 1 + 0.5 * randn(g, rows)
    old = (logp - away(0.15 * randn(g, rows), (0.2, 0.2))).float()
    # (a mean's gradients are a few thousandths of a token's: above fp16's least steps by this)
    up = rand(g, rows) + 0.1 if reduction == "none" else torch.tensor(700.0, device="cuda")
    want = orc.policy(h, w, labels, A, old, None, up, reduction=reduction)
    size = 1 + orc.size_of(h, w, labels)
    for keep in (True, False):
        got = run(mr.linear_policy_loss, h, w, up, labels, A, old, reduction=reduction, keep_logits=keep)
        check_all(got, want, size)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,D,V", [(300, 200, 5003), (1500, 768, 16001)])
def test_gradients_of_16_bits_are_rounded_twice_and_no_more(rows, D, V, dtype):
    """Factors spread over many values: the logits' gradient and the output are each off by up to u, half a step at the
    least value of a binade, evenly between -u and u: u / sqrt(3) in the 2-norm at most.  With fp32's errors, sqrt(2 / 3) u."""
    g, h, w, labels, logp = head((rows,), D, V, dtype, rows + D)
    A = torch.exp(0.5 * randn(g, rows))
    old = (logp - away(0.05 * randn(g, rows), (0.2, 0.2))).float()
    up = torch.ones((), device="cuda")
    # (the upstream gradient keeps fp16's least steps far below what is compared)
    got = run(mr.linear_policy_loss, h, w, up * 64, labels, A, old)
    want = orc.policy(h, w, labels, A, old, None, up * 64)
    for name, a, e in zip(("dhidden", "dweight"), got[1:], want[1:3]):
        rel = float((a.double() - e).norm() / e.norm())
        assert rel <= math.sqrt(2 / 3) * U[dtype] * 1.01, f"{name}: {rel:.2e}"


def two_sure_words(T, dtype, seed):
    """Row 5's softmax is on words 7 and 8 alone (the others' probabilities are 0 in fp32), which no other row has as its
    label: what row 5 gives dweight is in those two rows.  (hidden, weight, labels)"""
    g, h, w, labels, _ = head((T,), 64, 500, dtype, seed, ignored=0.0)
    labels = torch.where((labels == 7) | (labels == 8), 9, labels)
    w[:, 0] = 0.0
    w[7:9, 0] = 32.0
    h[:, 0] = 0.0
    h[5] = 0.0
    h[5, 0] = 4.0
    labels[5] = 7
    return g, h, w, labels


@pytest.mark.parametrize("T", [48, 300])
@pytest.mark.parametrize("dtype,moved", [(F32, 30.0), (F32, 80.0), (BF16, 30.0), (BF16, 80.0), (F16, 7.0), (F16, 14.0)])
def test_a_row_far_from_its_old_policy_leaves_the_others_words(dtype, moved, T):
    """A ratio of e^moved in row 5: dhidden's other rows, and the rows of dweight that only the other tokens give
    anything.  In fp16 the upstream gradient keeps row 5's own in the type's range."""
    g, h, w, labels = two_sure_words(T, dtype, 23)
    logp = orc.log_probs(h, w, labels, torch.zeros(T, device="cuda"))[0]
    assert abs(float(logp[5]) + math.log(2)) < 0.01
    old = logp.clone()
    old[5] -= moved
    A = torch.full((T,), -1.0, device="cuda")
    up = torch.tensor(2.0 ** -8 if moved == 14.0 else 1.0, device="cuda")
    loss, dh, dw = run(mr.linear_policy_loss, h, w, up, labels, A, old.float(), reduction="sum")
    want = orc.policy(h, w, labels, A, old.float(), None, up, reduction="sum")
    rows = [i for i in range(T) if i != 5]
    words = [i for i in range(500) if i not in (7, 8)]
    times = (1 + orc.size_of(h, w, labels)) * want[3]
    check("dhidden", dh[rows], want[1][rows], times)
    check("dweight", dw[words], want[2][words], times)
    for a, e in ((dh[5], want[1][5]), (dw[7:9], want[2][7:9])):
        assert float((a.double() - e).norm() / e.norm()) <= (2 * U[dtype] if dtype in U else 1e-3)
