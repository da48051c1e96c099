"""Output head on the GPU over the range of its types: rows, words and upstream gradients of very different
sizes in one call.  Every element is held to its own bound, from the sums that make it (in 64 bits, with
absolute values), so that nothing large hides what is small.

A sum of n products in fp32, in any order, is off by at most (n + 1) u S, with S the sum of the
products' absolute values and u = 2^-24.  From that:
  logits      E_t = (D + 16) u max_v S_tv         (16: the factor log2(e) and the exponentials, a few u each)
  loss        2 E_t + 16 u |lse|                  (a logit, and the lse of logits so far off)
  dhidden     (V + 16) u sum_v |dz||w| + 4 E_t sum_v |c| q |w|          (q is off by the factor exp(2 E_t),
  dweight     (rows + 16) u sum_t |dz||h| + sum_t 4 E_t |c_t| q |h|      less than 1 + 4 E_t below E_t = 1 / 4)
"""
from __future__ import annotations

import math

import pytest
import torch

import mlx_recurrence_amd as mr
from tests import head_oracle as orc

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def run_ce(h, w, labels, up, **kw):
    h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = mr.linear_cross_entropy(h, w, labels, reduction="none", keep_logits=len(h) != 700, **kw)
    return (loss.detach(), *torch.autograd.grad(loss, (h, w), up))


def parts(h, w, labels, up):
    """64-bit q, |dz| and each logit's sum of absolute products."""
    h, w = h.double(), w.double()
    q = torch.softmax(h @ w.T, 1)
    dz = q.clone()
    dz[torch.arange(len(h)), labels] -= 1
    return q, (dz * up.double()[:, None]).abs(), h.abs() @ w.abs().T


def check_fp32(got, h, w, labels, up):
    u = 2.0 ** -24
    want = orc.cross_entropy(h, w, labels, up, reduction="none")
    q, dz, s = parts(h, w, labels, up)
    e = (h.shape[1] + 16) * u * s.max(1).values
    qe = q * torch.where(e < 0.25, 4 * e, math.inf)[:, None] * up.double().abs()[:, None]
    qe = torch.where(q > 0, qe, 0).nan_to_num(posinf=1e300)
    lse = torch.logsumexp(h.double() @ w.double().T, 1)
    bounds = (2 * e + 16 * u * lse.abs(),
              (len(w) + 16) * u * (dz @ w.double().abs()) + qe @ w.double().abs(),
              (len(h) + 16) * u * (dz.T @ h.double().abs()) + qe.T @ h.double().abs())
    for name, a, b, most in zip(("loss", "dhidden", "dweight"), got, want, bounds):
        assert bool(torch.isfinite(a).all()), f"{name}: not finite"
        off = (a.double() - b).abs() / (most + 1e-35)
        worst = float(off.max())
        assert worst <= 1, f"{name}: {worst:.3g} times the bound at {tuple(int(i) for i in (off == worst).nonzero()[0])}"


def head(rows, D, V, seed, dtype=F32):
    g = gen(seed)
    w = randn(g, V, D) * (2 / math.sqrt(D))
    labels = torch.randint(0, V, (rows,), generator=g, device="cuda")
    return (randn(g, rows, D) + 0.5 * w[labels]).to(dtype), w.to(dtype), labels


# On either side of 256 rows; one more size whose logits are formed again (run_ce).
FP32_SIZES = [(200, 256, 2000), (300, 256, 2000), (700, 64, 1500)]


@pytest.mark.parametrize("rows,D,V", FP32_SIZES)
@pytest.mark.parametrize("size", [1.0, 1e8, 1e13])
def test_fp32_one_large_row(rows, D, V, size):
    h, w, labels = head(rows, D, V, 1)
    h[0] *= size
    up = torch.ones(rows, device="cuda")
    check_fp32(run_ce(h, w, labels, up), h, w, labels, up)


@pytest.mark.parametrize("rows,D,V", FP32_SIZES)
@pytest.mark.parametrize("size", [1e4, 1e8, 1e13])
def test_fp32_one_large_word(rows, D, V, size):
    h, w, labels = head(rows, D, V, 2)
    w[5] *= size
    h[:, 0] = 1 / size
    w[5, 1:] = 0   # its logits stay near 1, so every row has something of it
    labels[labels == 5] = 6
    up = torch.ones(rows, device="cuda")
    check_fp32(run_ce(h, w, labels, up), h, w, labels, up)


@pytest.mark.parametrize("rows,D,V", FP32_SIZES)
def test_fp32_channels_of_other_sizes(rows, D, V):
    """Channels large in the states and small in the weight: products near 1 of factors far apart."""
    h, w, labels = head(rows, D, V, 3)
    f = torch.exp2(torch.arange(D, device="cuda") % 7 * 10.0 - 30)
    up = torch.ones(rows, device="cuda")
    check_fp32(run_ce(h * f, w / f, labels, up), h * f, w / f, labels, up)


@pytest.mark.parametrize("rows,D,V", FP32_SIZES)
def test_fp32_rare_words(rows, D, V):
    """Words of probability 1e-3 to 1e-18: their rows of dweight are as exact as any other."""
    h, w, labels = head(rows, D, V, 4)
    h[:, 0] = 4.0
    w[:, 0] = -torch.arange(V, device="cuda") % 100 / 10.0
    labels = labels // 100 * 100
    up = torch.ones(rows, device="cuda")
    check_fp32(run_ce(h, w, labels, up), h, w, labels, up)


@pytest.mark.parametrize("rows,D,V", FP32_SIZES)
def test_fp32_upstreams_of_other_sizes(rows, D, V):
    h, w, labels = head(rows, D, V, 5)
    up = torch.logspace(0, -20, rows, device="cuda")
    check_fp32(run_ce(h, w, labels, up), h, w, labels, up)


@pytest.mark.parametrize("rows", [120, 300])
@pytest.mark.parametrize("scale_h,scale_w", [(1e-24, 1e24), (1e25, 1e-25), (1.0, 1e-30), (1e-30, 1.0)])
def test_fp32_extreme_scales(rows, scale_h, scale_w):
    h, w, labels = head(rows, 100, 600, 6)
    h, w = h * scale_h, w * scale_w
    up = torch.ones(rows, device="cuda")
    check_fp32(run_ce(h, w, labels, up), h, w, labels, up)


# fp16 outputs, row by row in the 2-norm.  u = 2^-11 (half a unit in the last place), 2^-25 half of fp16's least step:
#   dhidden  u |dh_t| + u sum_v |dz_tv| |w_v| + 2^-25 sqrt(D)         its rounding, that of dz, and what fp16 cannot hold
#   dweight  u |dw_v| + 2 u sum_t |dz_tv| |h_t| + 2^-25 sqrt(D)       and that of a state times its row's power of two
# and an eighth on top for the sums in fp32.
def check_f16(got, h, w, dz, want):
    u, (h, w) = 2.0 ** -11, (h.double(), w.double())
    least = 2.0 ** -25 * math.sqrt(h.shape[1])
    for name, a, b, terms in (("dhidden", got[1], want[1], dz @ w.norm(dim=1)), ("dweight", got[2], want[2], 2 * (dz.T @ h.norm(dim=1)))):
        assert bool(torch.isfinite(a).all()), f"{name}: not finite"
        off = (a.double() - b).norm(dim=1) / (1.125 * u * (b.norm(dim=1) + terms) + least)
        assert float(off.max()) <= 1, f"{name}: {float(off.max()):.3g} times the bound in row {int(off.argmax())}"


@pytest.mark.parametrize("rows,D,V", [(40, 64, 2000), (300, 64, 2000), (700, 200, 3000)])
def test_fp16_upstreams_of_other_sizes(rows, D, V):
    """Upstream gradients from 5e3 to 5e-5: the gradients of the smallest are still fp16's normal values."""
    g = gen(7)
    w = (2 * randn(g, V, D)).to(F16)
    h = (0.05 * randn(g, rows, D)).to(F16)
    labels = torch.randint(0, V, (rows,), generator=g, device="cuda")
    up = torch.logspace(math.log10(5e3), math.log10(5e-5), rows, device="cuda")
    _, dz, _ = parts(h, w, labels, up)
    check_f16(run_ce(h, w, labels, up), h, w, dz, orc.cross_entropy(h, w, labels, up, reduction="none"))


@pytest.mark.parametrize("rows,D,V", [(40, 64, 1000), (300, 64, 1000)])
def test_fp16_words_of_rows_with_a_small_upstream(rows, D, V):
    """Rows of a large upstream that are sure of their word leave the gradients of the others' words alone."""
    g = gen(8)
    w = randn(g, V, D).to(F16)
    labels = torch.randint(0, V, (rows,), generator=g, device="cuda")
    h = randn(g, rows, D)
    h[::2] = 4 * w[labels[::2]].float()
    h = h.to(F16)
    up = torch.where(torch.arange(rows, device="cuda") % 2 == 0, 5e3, 1e-4)
    _, dz, _ = parts(h, w, labels, up)
    assert float(dz[::2].max()) < 1e-6 * float(dz[1::2].max())
    check_f16(run_ce(h, w, labels, up), h, w, dz, orc.cross_entropy(h, w, labels, up, reduction="none"))


@pytest.mark.parametrize("rows", [40, 300])
def test_fp16_distillation_upstreams_of_other_sizes(rows):
    g = gen(9)
    w, h = (2 * randn(g, 1500, 72)).to(F16), (0.05 * randn(g, rows, 72)).to(F16)
    t = 2 * randn(g, rows, 6)
    ids = torch.stack([torch.randperm(1500, generator=g, device="cuda")[:6] for _ in range(rows)])
    up = torch.logspace(math.log10(2e3), math.log10(5e-5), rows, device="cuda")
    up[3] = 0
    hl, wl = h.requires_grad_(True), w.requires_grad_(True)
    loss = mr.linear_distillation(hl, wl, t, ids, temperature=2.0, reduction="none")
    got = (loss, *torch.autograd.grad(loss, (hl, wl), up))
    h, w = h.detach(), w.detach()
    dz = 2 * up.double()[:, None] * (torch.softmax(h.double() @ w.double().T / 2, 1)
                                     .scatter_add(1, ids, -torch.softmax(t.double() / 2, 1)))
    check_f16(got, h, w, dz.abs(), orc.distillation(h, w, t, ids, up, tau=2.0, reduction="none"))


def run_kd(h, w, t, ids, tau):
    h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = mr.linear_distillation(h, w, t, ids, temperature=tau, reduction="none")
    return (loss.detach(), *torch.autograd.grad(loss, (h, w), torch.ones_like(loss)))


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_absent_entries_may_have_any_id(dtype):
    """A logit of -inf is no entry whatever its id, a negative id none whatever its logit."""
    h, w, first = head(70, 40, 300, 10, dtype)
    ids = first[:, None].repeat(1, 5)
    ids[:, 1:] = (ids[:, 1:] + torch.arange(1, 5, device="cuda")) % 300
    t = randn(gen(11), 70, 5)
    t[::2, 3:], t[4] = -math.inf, -math.inf
    gone = t == -math.inf
    want = run_kd(h, w, t, ids.masked_fill(gone, -1), 1.5)
    assert bool(torch.isfinite(want[0]).all()) and float(want[0][4]) == 0
    for bad in (300, 1 << 20, 1 << 40, -(1 << 40)):
        assert same(run_kd(h, w, t, ids.masked_fill(gone, bad), 1.5), want), bad
    assert same(run_kd(h, w, t.masked_fill(gone, math.nan), ids.masked_fill(gone, -5), 1.5), want)
    assert bool(torch.isnan(run_kd(h, w, t, torch.where(gone, ids, 300), 1.5)[0][0]))   # an entry that is there


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tau", [0.25, 1.0, 4.0])
def test_teacher_logits_of_the_largest_and_lowest_values(dtype, tau):
    """The type's lowest value is an entry like any other, also divided by a temperature below 1: equal logits,
    whatever they are, are an even split, and one far below another has weight 0."""
    h, w, first = head(20, 40, 300, 12)
    ids = torch.stack([first, (first + 7) % 300, (first + 50) % 300], 1)
    t = torch.zeros(20, 3, device="cuda", dtype=dtype)
    want = run_kd(h, w, t, ids, tau)
    for value in (torch.finfo(dtype).min, torch.finfo(dtype).max, 1000.0):
        assert same(run_kd(h, w, torch.full_like(t, value), ids, tau), want), value
    one = t.clone()
    one[:, 2] = -math.inf
    for low in (torch.finfo(dtype).min, -6e4):
        two = one.clone()
        two[:, 2] = low
        assert same(run_kd(h, w, two, ids, tau), run_kd(h, w, one, ids, tau)), low
    one[:, 0], t[:, 0] = torch.finfo(dtype).max, torch.finfo(dtype).max
    t[:, 1:], one[:, 1:] = torch.finfo(dtype).min, -math.inf
    assert same(run_kd(h, w, t, ids, tau), run_kd(h, w, one, ids, tau))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("rows", [40, 300])
def test_no_row_counts_whatever_the_upstream(rows, reduction, dtype):
    """A sum over no row, divided by their number: the upstream gradient is not finite, the gradients are 0."""
    h, w, labels = head(rows, 40, 300, 13, dtype)
    none = torch.full((rows, 2), -1, device="cuda")
    for value in (math.inf, math.nan):
        for f in (lambda a, b: mr.linear_cross_entropy(a, b, torch.full_like(labels, -100), reduction=reduction),
                  lambda a, b: mr.linear_distillation(a, b, torch.zeros(rows, 2, device="cuda"), none, reduction=reduction)):
            leaves = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
            loss = f(*leaves)
            for grad in torch.autograd.grad(loss, leaves, torch.full_like(loss, value)):
                assert not grad.any()
