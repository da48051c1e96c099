"""Output head on the GPU in 16 bits, row by row: a row that is off is not hidden by the others.

u is half a unit in the last place (2^-8 bf16, 2^-11 fp16).  A value rounded to nearest is off by at most u of itself
and, over many values, by u / sqrt(3) in the mean square.
  Losses: the output's rounding, and that of the logits' gradient dz before the products (a term's error is its own).
  With S_t^2 = sum_v dz_tv^2 |w_v|^2 for a row of dhidden and sum_t dz_tv^2 |h_t|^2 for one of dweight:
    a row         at most u (|row| + S)         (a single term may be most of S: no mean)
    the tensor    1.1 u / sqrt(3) sqrt(sum |row|^2 + S^2), 1.1 for the fp32 sums and what is no mean yet
  fp16 besides holds nothing below 2^-25 (half its least step) of an element.
  Layer norm: element by element u of the value and, from sums in fp32 of up to 2^15 terms made as trees, 2^-18 of the
  absolute values that it is made of; dweight's and dbias's sums 2^-17 (a hundred steps of 2^-24 at most).
"""
from __future__ import annotations

import math

import pytest
import torch

import mlx_recurrence_amd as mr
from mlx_recurrence_amd import _lib
from tests import head_oracle as orc
from tests.test_gpu_head import gen, head_inputs, randn, run_ce, run_kd, teacher

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}


def check_rows(name, got, want, terms2, least):
    u = U[got.dtype]
    off2 = (got.double() - want).square().sum(1)
    row, s = want.norm(dim=1), terms2.sqrt()
    worst = (off2.sqrt() / (u * (row + s) + least)).max()
    assert float(worst) <= 1, f"{name}: a row {float(worst):.3g} times its bound"
    whole, most = float(off2.sum().sqrt()), 1.1 * u / math.sqrt(3) * math.sqrt(float((row.square() + terms2).sum()))
    assert whole <= most + least * math.sqrt(len(got)), f"{name}: {whole / most:.3g} times its bound"


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("reduction", ["sum", "none"])
@pytest.mark.parametrize("rows,D,V", [(50, 128, 900), (100, 128, 900), (300, 256, 2000), (1000, 511, 5003), (2500, 96, 700)])
def test_losses(rows, D, V, dtype, reduction):
    g, h, w, labels = head_inputs(rows, D, V, dtype, rows + D + V)
    up = torch.rand(rows, generator=g, device="cuda") + 0.1 if reduction == "none" else torch.tensor(0.7, device="cuda")
    t, ids = teacher(g, rows, 5, V, labels)
    c, q = up.double().expand(rows)[:, None], torch.softmax(h.double() @ w.double().T, 1)
    dz = c * q.scatter_add(1, labels[:, None], -torch.ones(rows, 1, dtype=torch.float64, device="cuda"))
    tau = 2.0
    there = ids >= 0
    p = torch.softmax(torch.where(there, t.double() / tau, -math.inf), 1)   # every row has its first entry or none
    valid = there.any(1)
    p = torch.where(valid[:, None], p, 0)
    dz_kd = tau * c * torch.softmax(h.double() @ w.double().T / tau, 1).scatter_add(1, ids.clamp(min=0), -p)
    dz_kd = torch.where(valid[:, None], dz_kd, 0)
    least = 2.0 ** -25 * math.sqrt(D) if dtype == F16 else 1e-30
    for got, want, z in ((run_ce(h, w, labels, up, reduction=reduction), orc.cross_entropy(h, w, labels, up, reduction=reduction), dz),
                         (run_kd(h, w, t, ids, up, temperature=tau, reduction=reduction),
                          orc.distillation(h, w, t, ids, up, tau=tau, reduction=reduction), dz_kd)):
        z2 = z.square()
        check_rows("dhidden", got[1], want[1], z2 @ w.double().square().sum(1), least)
        check_rows("dweight", got[2], want[2], z2.T @ h.double().square().sum(1), least)


# Rows of one to three waves' pieces, of a workgroup's forms (2561 channels and more; 1537 of fp32) and so many that each
# workgroup of the backward, of which there are at most 512, takes several.
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,D", [(20000, 96), (6000, 1000), (5000, 2560), (2100, 1537), (2100, 2561), (1500, 4104), (1300, 5120),
                                    (1100, 8193), (1030, 16384), (1030, 32767)])
def test_layer_norm(rows, D, dtype):
    g = gen(rows + D)
    x = (randn(g, rows, D) * torch.exp(randn(g, rows, 1)) + randn(g, rows, 1)).to(dtype).requires_grad_(True)
    w = (1 + 0.3 * randn(g, D)).to(dtype).requires_grad_(True)
    b = randn(g, D).to(dtype).requires_grad_(True)
    dy = randn(g, rows, D).to(dtype)
    y = mr.layer_norm(x, w, b)
    got = (y, *torch.autograd.grad(y, (x, w, b), dy))
    x, w, b = x.detach(), w.detach(), b.detach()
    u, least = U[dtype], 2.0 ** -25 if dtype == F16 else 0.0
    sums = [torch.zeros(D, dtype=torch.float64, device="cuda") for _ in range(4)]   # dw, db and their absolute values
    for i in range(0, rows, 2000):
        part = slice(i, i + 2000)
        wy, wx, ww, wb = orc.layer_norm(x[part], w, b, 1e-5, dy[part])
        xd, gd = x[part].double(), dy[part].double()
        mean = xd.mean(1, keepdim=True)
        r = ((xd - mean).square().mean(1, keepdim=True) + 1e-5) ** -0.5
        size = (xd.abs() + mean.abs()) * r        # of what x hat is the difference of
        gw = (gd * w.double()).abs()
        for name, a, e, terms in (("y", got[0][part], wy, size * w.double().abs() + b.double().abs()),
                                  ("dx", got[1][part], wx, r * (gw + gw.mean(1, keepdim=True)
                                                                + size * (gw * size).mean(1, keepdim=True)))):
            off = ((a.double() - e).abs() / (u * e.abs() + 2.0 ** -18 * terms + least)).max()
            assert float(off) <= 1, f"{name}: an element {float(off):.3g} times its bound"
        for s, v in zip(sums, (ww, wb, (gd.abs() * size).sum(0), gd.abs().sum(0))):
            s += v
    for name, a, e, terms in (("dw", got[2], sums[0], sums[2]), ("db", got[3], sums[1], sums[3])):
        off = ((a.double() - e).abs() / (u * e.abs() + 2.0 ** -17 * terms + least)).max()
        assert float(off) <= 1, f"{name}: an element {float(off):.3g} times its bound"


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,D", [(1, 8), (300, 1000), (5000, 64), (40, 2000), (9, 2561), (1100, 5000), (7, 20000)])
def test_layer_norm_writes_inside_its_workspace(rows, D, dtype, monkeypatch):
    """A workspace of exactly the stated size between guards, filled with NaN: the same gradients, the guards whole."""
    buffers = []

    def guarded(n, device):
        whole = torch.full((n + 8192,), 0xA5, dtype=torch.uint8, device=device)
        whole[4096:4096 + n] = 0xFF
        buffers.append((whole, n))
        return whole[4096:4096 + n]

    g = gen(rows * D)
    leaves = [randn(g, *s).to(dtype).requires_grad_(True) for s in ((rows, D), (D,), (D,))]
    dy = randn(g, rows, D).to(dtype)
    want = torch.autograd.grad(mr.layer_norm(*leaves), leaves, dy)
    monkeypatch.setattr(_lib, "autograd_ext", lambda: None)
    monkeypatch.setattr(_lib, "_alloc_ws", guarded)
    for a, e in zip(torch.autograd.grad(mr.layer_norm(*leaves), leaves, dy), want):
        assert torch.equal(a, e)
    assert len(buffers) == 1
    whole, n = buffers[0]
    assert (whole[:4096] == 0xA5).all() and (whole[4096 + n:] == 0xA5).all()
