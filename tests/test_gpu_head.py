"""Output head on the GPU: layer norm, cross entropy and distillation from hidden states
against 64-bit formulas (tests/head_oracle.py, on the same rounded inputs).

Two measures, |got - want| over want: of the largest elements, and of the 2-norms.
Bounds, from the arithmetic (u = half a unit in the last place of the output's type, which
holds 8 or 11 bits: 2^-8 bf16, 2^-11 fp16):
  16-bit outputs   the output's rounding and, for dhidden and dweight, that of the logits'
                   gradient, once each, the latter averaged over a sum: 2-norm at most
                   sqrt(2) u, largest element at most 4 u (the sum's terms may exceed it).
  fp32 outputs     operands to 2^-22, sums of up to 2^16 terms in fp32 (rms error growing
                   with the square root of the number of accumulation steps, n / 16):
                   2-norm at most 2^-22 + 64 * 2^-24 = 4e-6, largest element 2e-5.
"""
from __future__ import annotations

import math

import pytest
import torch

import mlx_recurrence_amd as mr
from mlx_recurrence_amd import _lib
from tests import head_oracle as orc

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = {BF16: 2.0 ** -8, F16: 2.0 ** -11}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def check(name, got, want):
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
    most, norm = (4 * U[got.dtype], 1.5 * U[got.dtype]) if got.dtype in U else (2e-5, 4e-6)
    assert big <= most and rel <= norm, f"{name}: largest {big:.2e} (<= {most:.1e}), 2-norm {rel:.2e} (<= {norm:.1e})"


# ------------------------------------------------------------------ layer norm
NORM = [(1, 1), (1, 5120), (2, 7), (3, 8), (5, 64), (4, 65), (9, 512), (7, 513), (129, 768), (33, 1001), (600, 1024),
        (17, 1032), (1030, 2048), (6, 2049), (40, 2560), (3, 8192), (5, 8200), (2, 16385), (2, 32768), (3000, 33)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,D", NORM)
def test_layer_norm(rows, D, dtype):
    g = gen(rows * 7919 + D)
    x = (randn(g, rows, D) * torch.exp(randn(g, rows, 1)) + 3 * randn(g, rows, 1)).to(dtype).requires_grad_(True)
    w = (1 + 0.3 * randn(g, D)).to(dtype).requires_grad_(True)
    b = randn(g, D).to(dtype).requires_grad_(True)
    dy = randn(g, rows, D).to(dtype)
    y = mr.layer_norm(x, w, b)
    got = (y, *torch.autograd.grad(y, (x, w, b), dy))
    want = orc.layer_norm(x.detach(), w.detach(), b.detach(), 1e-5, dy)
    for name, a, e in zip(("y", "dx", "dw", "db"), got, want):
        if D == 1 and name == "dx":
            assert float(a.abs().max()) <= 1e-2   # 0 but for rounding, which 1 / sqrt(eps) = 316 magnifies
        else:
            check(name, a, e)
    with torch.no_grad():
        assert torch.equal(mr.layer_norm(x, w, b), y)


@pytest.mark.parametrize("out", [F32, BF16, F16])
@pytest.mark.parametrize("wd,bd", [(F32, F32), (BF16, F32), (F16, F16), (None, F32), (BF16, None), (None, None)])
def test_layer_norm_types(out, wd, bd):
    g = gen(3)
    x = randn(g, 4, 5, 200).requires_grad_(True)
    w = None if wd is None else (1 + randn(g, 200)).to(wd).requires_grad_(True)
    b = None if bd is None else randn(g, 200).to(bd).requires_grad_(True)
    dy = randn(g, 4, 5, 200).to(out)
    y = mr.layer_norm(x, w, b, eps=1e-3, out_dtype=out)
    leaves = [t for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    wy, wx, ww, wb = orc.layer_norm(x.detach(), w, b, 1e-3, dy)
    assert y.dtype == out
    check("y", y, wy)
    want = [wx] + ([] if w is None else [ww]) + ([] if b is None else [wb])
    for t, a, e in zip(leaves, grads, want):
        assert a.dtype == t.dtype
        check("grad", a, e)


def test_layer_norm_strides_streams_and_edges():
    g = gen(5)
    base = randn(g, 40, 300)
    w, b = randn(g, 300), randn(g, 300)
    want = orc.layer_norm(base.T.contiguous(), w[:40], b[:40], 1e-5)
    check("transposed", mr.layer_norm(base.T, w[:40], b[:40]), want)
    flat = randn(g, 1 + 3 * 20)
    check("offset by one", mr.layer_norm(flat[1:].view(3, 20), w[1:21], b[3:23]),
          orc.layer_norm(flat[1:].view(3, 20), w[1:21], b[3:23], 1e-5))
    x = randn(g, 6, 300).requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = mr.layer_norm(x, w, b)
        (dx,) = torch.autograd.grad(y, x, torch.ones((), device="cuda").expand(6, 300))
    torch.cuda.current_stream().wait_stream(side)
    wy, wdx, _, _ = orc.layer_norm(x.detach(), w, b, 1e-5, torch.ones(6, 300, device="cuda"))
    check("y", y, wy)
    check("dx", dx, wdx)
    empty = torch.zeros(0, 300, device="cuda", requires_grad=True)
    ww = w.clone().requires_grad_(True)
    y = mr.layer_norm(empty, ww, b)
    de, dw = torch.autograd.grad(y, (empty, ww), torch.zeros(0, 300, device="cuda"))
    assert de.shape == (0, 300) and not dw.any()
    x = randn(g, 4, 100)
    x[1, 3], x[2, 5] = math.nan, math.inf
    y = mr.layer_norm(x)
    assert torch.isnan(y[1]).all() and torch.isnan(y[2, 5]) and torch.isfinite(y[0]).all() and torch.isfinite(y[3]).all()
    const = torch.full((2, 64), 7.5, device="cuda")
    assert not mr.layer_norm(const).any()


def test_layer_norm_only_what_is_wanted():
    g = gen(6)
    x, w, b, dy = randn(g, 50, 96), randn(g, 96), randn(g, 96), randn(g, 50, 96)
    wx, ww, wb = orc.layer_norm(x, w, b, 1e-5, dy)[1:]
    for which, want in ((0, wx), (1, ww), (2, wb)):
        ins = [x, w, b]
        ins[which] = ins[which].clone().requires_grad_(True)
        y = mr.layer_norm(*ins)
        y.backward(dy)
        check("grad", ins[which].grad, want)


def test_layer_norm_past_2_31_elements():
    rows, D = 65700, 32768
    x = torch.empty(rows, D, dtype=BF16, device="cuda")
    x[-3:] = randn(gen(1), 3, D).to(BF16)
    x[:-3] = 0
    y = mr.layer_norm(x)
    check("last rows", y[-3:], orc.layer_norm(x[-3:], None, None, 1e-5))
    assert not y[:100].any()


# ------------------------------------------------------------------ losses
def head_inputs(rows, D, V, dtype, seed, size=2.0):
    g = gen(seed)
    w = randn(g, V, D) * (size / math.sqrt(D))
    first = torch.randint(0, V, (rows,), generator=g, device="cuda")
    h = randn(g, rows, D) + 0.5 * w[first]
    return g, h.to(dtype), w.to(dtype), first


def teacher(g, rows, K, V, first, absent=0.3):
    ids = (first[:, None] + torch.randint(0, V, (rows, K), generator=g, device="cuda")) % V
    ids[:, 0] = first
    t = 2 * randn(g, rows, K)
    gone = torch.rand((rows, K), generator=g, device="cuda") < absent
    return t, ids.masked_fill(gone, -1)


def run_ce(h, w, labels, up, **kw):
    h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = mr.linear_cross_entropy(h, w, labels, **kw)
    return (loss.detach(), *torch.autograd.grad(loss, (h, w), up))


def run_kd(h, w, t, ids, up, **kw):
    h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = mr.linear_distillation(h, w, t, ids, **kw)
    return (loss.detach(), *torch.autograd.grad(loss, (h, w), up))


def check_all(got, want):
    for name, a, e in zip(("loss", "dhidden", "dweight"), got, want):
        check(name, a, e)


SIZES = [(1, 1, 1), (1, 8, 2), (2, 7, 3), (1, 64, 1000), (3, 65, 127), (31, 64, 128), (32, 40, 129), (33, 72, 255),
         (64, 128, 256), (65, 200, 257), (127, 96, 1000), (128, 256, 513), (129, 33, 2000), (255, 264, 700), (256, 512, 777),
         (257, 257, 1300), (300, 1000, 5003), (700, 320, 4096)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,D,V", SIZES)
def test_cross_entropy(rows, D, V, dtype):
    g, h, w, labels = head_inputs(rows, D, V, dtype, rows + 31 * D + 7 * V)
    labels = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.25, -100, labels)
    up = torch.rand(rows, generator=g, device="cuda") + 0.1
    check_all(run_ce(h, w, labels, up, z_loss=1e-3, reduction="none"),
              orc.cross_entropy(h, w, labels, up, zl=1e-3, reduction="none"))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,D,V", SIZES)
@pytest.mark.parametrize("K,tau", [(1, 1.0), (5, 2.0)])
def test_distillation(rows, D, V, dtype, K, tau):
    g, h, w, first = head_inputs(rows, D, V, dtype, rows + 37 * D + 11 * V + K)
    t, ids = teacher(g, rows, K, V, first)
    up = torch.rand(rows, generator=g, device="cuda") + 0.1
    got, want = (run_kd(h, w, t, ids, up, temperature=tau, reduction="none"),
                 orc.distillation(h, w, t, ids, up, tau=tau, reduction="none"))
    if V == 1:   # q = sum p = 1: the loss is sum p log p and every gradient 0, but for the rounding of p to 2^-24 each
        check("loss", got[0], want[0])
        for a, factor in zip(got[1:], (w, h)):
            assert float(a.abs().max()) <= K * 2.0 ** -24 * 2 * tau * float(up.max() * factor.abs().max())
        return
    check_all(got, want)


@pytest.mark.parametrize("K", [2, 63, 64, 65, 200, 1024])
def test_distillation_entries(K):
    """Entries in any order, the same word twice, many entries of one tile."""
    g, h, w, first = head_inputs(70, 96, 700, BF16, K)
    t, ids = teacher(g, 70, K, 700, first, absent=0.2)
    ids[3] = torch.arange(K, device="cuda") % 5
    ids[4, :] = 699
    t[5, ::2] = -math.inf
    up = torch.rand(70, generator=g, device="cuda")
    check_all(run_kd(h, w, t.to(BF16), ids, up, temperature=1.5, reduction="none"),
              orc.distillation(h, w, t.to(BF16), ids, up, tau=1.5, reduction="none"))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_reductions_shapes_and_label_types(dtype, reduction):
    g, h, w, labels = head_inputs(60, 48, 333, dtype, 8)
    labels[::7] = -1
    h3, l3 = h.view(3, 20, 48), labels.view(3, 20).int()
    up = torch.rand(3, 20, generator=g, device="cuda") if reduction == "none" else torch.tensor(0.7, device="cuda")
    loss, dh, dw = run_ce(h3, w, l3, up, ignore_index=-1, reduction=reduction)
    want = orc.cross_entropy(h, w, labels, up.reshape(-1) if reduction == "none" else up, ignore=-1, reduction=reduction)
    assert loss.shape == ((3, 20) if reduction == "none" else ()) and loss.dtype == F32 and dh.shape == h3.shape
    check_all((loss.reshape(want[0].shape), dh.view(60, 48), dw), want)
    t, ids = teacher(g, 60, 4, 333, labels.clamp(min=0))
    loss, dh, dw = run_kd(h3, w, t.view(3, 20, 4), ids.view(3, 20, 4), up, temperature=3.0, reduction=reduction)
    want = orc.distillation(h, w, t, ids, up.reshape(-1) if reduction == "none" else up, tau=3.0, reduction=reduction)
    check_all((loss.reshape(want[0].shape), dh.view(60, 48), dw), want)


def test_more_rows_and_words_than_a_piece():
    """Two pieces of the vocabulary, several tiles of rows, against 64 bits."""
    rows, D, V = 8192, 72, 40000
    g, h, w, labels = head_inputs(rows, D, V, BF16, 12)
    labels[torch.rand(rows, generator=g, device="cuda") < 0.1] = -100
    labels[-1] = V - 1
    up = torch.tensor(1.0, device="cuda")
    check_all(run_ce(h, w, labels, up), orc.cross_entropy(h, w, labels, up))
    t, ids = teacher(g, rows, 20, V, labels.clamp(min=0))
    check_all(run_kd(h, w, t, ids, up, temperature=2.0), orc.distillation(h, w, t, ids, up, tau=2.0))


def test_fp32_pieces():
    rows, D, V = 4500, 40, 33000
    g, h, w, labels = head_inputs(rows, D, V, F32, 13)
    up = torch.tensor(1.0, device="cuda")
    check_all(run_ce(h, w, labels, up), orc.cross_entropy(h, w, labels, up))


# few tiles of many channels: the logits' sums are made in parts; words that are no whole segment of 2048
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,D,V", [(1, 5000, 300), (5, 3000, 700), (40, 2048, 5003), (200, 4096, 640), (300, 2050, 2100)])
def test_sums_in_parts(rows, D, V, dtype):
    g, h, w, labels = head_inputs(rows, D, V, dtype, rows + D + V)
    labels[2::5] = -100
    up = torch.rand(rows, generator=g, device="cuda") + 0.1
    got = run_ce(h, w, labels, up, z_loss=1e-3, reduction="none")
    check_all(got, orc.cross_entropy(h, w, labels, up, zl=1e-3, reduction="none"))
    with torch.no_grad():   # without a backward the logits are not kept, the loss is the same
        assert torch.equal(mr.linear_cross_entropy(h, w, labels, z_loss=1e-3, reduction="none"), got[0])
    t, ids = teacher(g, rows, 70, V, labels.clamp(min=0))
    ids[-1] = torch.arange(70, device="cuda") % 3 + V - 3
    check_all(run_kd(h, w, t, ids, up, temperature=2.0, reduction="none"),
              orc.distillation(h, w, t, ids, up, tau=2.0, reduction="none"))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,D,V", [(1500, 65, 300), (3001, 200, 640), (5000, 1100, 129)])
def test_dweight_in_parts(rows, D, V, dtype):
    """Few words and many rows: dweight's sums over the rows that count, whose number only the device knows."""
    g, h, w, labels = head_inputs(rows, D, V, dtype, rows + D + V)
    for ignored in (0.0, 0.95, 1.0):
        l2 = torch.where(torch.rand(rows, generator=g, device="cuda") < ignored, -100, labels)
        up = torch.rand(rows, generator=g, device="cuda") + 0.1
        got = run_ce(h, w, l2, up, reduction="none")
        check_all(got, orc.cross_entropy(h, w, l2, up, reduction="none"))
    assert not got[2].any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_sums_in_parts_of_what_is_not_finite(dtype):
    _, h, w, labels = head_inputs(20, 3000, 300, dtype, 6)
    h[3, 5], h[9, 1] = math.nan, math.inf
    labels[12] = 300
    loss, dh, dw = run_ce(h, w, labels, torch.ones(20, device="cuda"), reduction="none")
    for r in (3, 9, 12):
        assert not torch.isfinite(loss[r]) and torch.isnan(dh[r]).any()
    assert torch.isnan(dw).any()
    fine = [r for r in range(20) if r not in (3, 9, 12)]
    want = orc.cross_entropy(h[fine], w, labels[fine], torch.ones(17, device="cuda"), reduction="none")
    check("loss", loss[fine], want[0])
    check("dhidden", dh[fine], want[1])


@pytest.mark.parametrize("rows,D,V,dtype", [(8192, 1030, 33000, BF16), (4500, 360, 33000, F32)])
def test_kept_logits_of_two_pieces(rows, D, V, dtype):
    """Logits that the forward leaves, read by the backward in two pieces of the vocabulary."""
    g, h, w, labels = head_inputs(rows, D, V, dtype, 15)
    labels[::9] = -100
    up = torch.tensor(1.0, device="cuda")
    check_all(run_ce(h, w, labels, up, z_loss=1e-3), orc.cross_entropy(h, w, labels, up, zl=1e-3))


def test_rows_that_do_not_count_are_not_read():
    for dtype in (F32, BF16, F16):
        g, h, w, labels = head_inputs(150, 64, 500, dtype, 3)
        out = torch.rand(150, generator=g, device="cuda") < 0.5
        labels[out] = -100
        clean = run_ce(h, w, labels, torch.ones((), device="cuda"))
        h2 = h.clone()
        h2[out] = math.nan
        h2[out.nonzero()[0, 0]] = math.inf
        dirty = run_ce(h2, w, labels, torch.ones((), device="cuda"))
        for a, b in zip(clean, dirty):
            assert torch.equal(a, b)
        assert not dirty[1][out].any()
        t, ids = teacher(g, 150, 6, 500, labels.clamp(min=0), absent=0.0)
        ids[out] = -1
        t[out] = math.nan
        for a, b in zip(run_kd(h, w, t, ids, torch.ones((), device="cuda")),
                        run_kd(h2, w, t, ids, torch.ones((), device="cuda"))):
            assert torch.equal(a, b)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_no_row_counts(reduction):
    for dtype in (F32, BF16, F16):
        _, h, w, labels = head_inputs(40, 33, 200, dtype, 4)
        up = torch.ones(40 if reduction == "none" else (), device="cuda")
        none = torch.full((40, 3), -1, device="cuda")
        for got in (run_ce(h, w, torch.full_like(labels, -100), up, reduction=reduction),
                    run_kd(h, w, torch.zeros(40, 3, device="cuda"), none, up, reduction=reduction),
                    run_kd(h, w, torch.full((40, 3), -math.inf, device="cuda"), none + 2, up, reduction=reduction)):
            for a in got:
                assert not a.any() and torch.isfinite(a).all()
        got = run_ce(h[:0], w, labels[:0], up[:0] if reduction == "none" else up, reduction=reduction)
        assert got[0].shape == ((0,) if reduction == "none" else ()) and got[1].shape == (0, 33)
        assert not got[0].any() and not got[2].any()


def test_invalid_ids_give_nan():
    for dtype in (F32, BF16, F16):
        _, h, w, labels = head_inputs(20, 64, 300, dtype, 5)
        up = torch.ones(20, device="cuda")
        for bad in (300, 1 << 40, -7):
            l2 = labels.clone()
            l2[4] = bad
            loss, dh, dw = run_ce(h, w, l2, up, reduction="none")
            assert torch.isnan(loss[4]) and torch.isfinite(loss[torch.arange(20) != 4]).all()
            assert torch.isnan(dh[4]).all() and torch.isfinite(dh[:4]).all() and torch.isfinite(dh[5:]).all()
            assert torch.isnan(dw).all()
        ids = labels[:, None].repeat(1, 3)
        ids[7, 1] = 300
        loss, dh, dw = run_kd(h, w, torch.zeros(20, 3, device="cuda"), ids, up, reduction="none")
        assert torch.isnan(loss[7]) and torch.isfinite(loss[torch.arange(20) != 7]).all()
        assert torch.isnan(dh[7]).all() and torch.isfinite(dh[:7]).all() and torch.isnan(dw).all()


def test_non_finite_states_stay_in_their_row():
    for dtype in (F32, BF16, F16):
        _, h, w, labels = head_inputs(20, 64, 300, dtype, 6)
        h[3, 5], h[9, 1] = math.nan, math.inf
        loss, dh, _ = run_ce(h, w, labels, torch.ones(20, device="cuda"), reduction="none")
        for r in (3, 9):
            assert not torch.isfinite(loss[r]) and torch.isnan(dh[r]).any()
        fine = [r for r in range(20) if r not in (3, 9)]
        want = orc.cross_entropy(h[fine], w, labels[fine], torch.ones(18, device="cuda"), reduction="none")
        check("loss", loss[fine], want[0])
        check("dhidden", dh[fine], want[1])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_large_logits(dtype):
    """Logits of thousands: a softmax of one word, or of none near the label."""
    g, h, w, labels = head_inputs(100, 128, 900, dtype, 7, size=300.0)
    up = torch.rand(100, generator=g, device="cuda")
    check_all(run_ce(h, w, labels, up, reduction="none"), orc.cross_entropy(h, w, labels, up, reduction="none"))


@pytest.mark.parametrize("rows", [120, 300])   # on the fp32 MFMA, in two fp16 planes
@pytest.mark.parametrize("scale_h,scale_w", [(1e-18, 1e6), (1e12, 1e-13), (3e-3, 5e2)])
def test_fp32_range(scale_h, scale_w, rows):
    """fp32 inputs whose sizes no 16-bit float holds, and rows a million times smaller than others."""
    g, h, w, labels = head_inputs(rows, 100, 600, F32, 9)
    h, w = h * scale_h, w * scale_w
    h[::5] *= 1e-6
    up = torch.rand(rows, generator=g, device="cuda")
    check_all(run_ce(h, w, labels, up, reduction="none"), orc.cross_entropy(h, w, labels, up, reduction="none"))


def test_small_gradients_keep_their_bits():
    """An upstream of 1e-7 a row: fp16 gradients of probabilities near 1e-4 are far below fp16's range inside."""
    _, h, w, labels = head_inputs(200, 64, 9000, F16, 10, size=0.1)
    w32 = w.float()
    up = torch.full((200,), 1e-7, device="cuda")
    loss, dh, _ = run_ce(h.float(), w32, labels, up, reduction="none")
    want = orc.cross_entropy(h, w, labels, up, reduction="none")
    check("dhidden", dh, want[1])
    up = torch.full((200,), 16.0, device="cuda")
    check_all(run_ce(h, w, labels, up, reduction="none"), orc.cross_entropy(h, w, labels, up, reduction="none"))


def test_mixed_types_strides_and_streams():
    g, h, w, labels = head_inputs(90, 80, 400, F32, 11)
    up = torch.ones((), device="cuda")
    hb = h.to(BF16)
    got = run_ce(hb, w, labels, up)                # runs in fp32
    assert got[1].dtype == BF16 and got[2].dtype == F32
    check_all(got, orc.cross_entropy(hb, w, labels, up))
    wide = torch.cat([w, w], 1).to(BF16)
    ht = hb.T.contiguous().T                       # strides (1, rows)
    want = orc.cross_entropy(hb, w.to(BF16), labels, up)
    check_all(run_ce(ht, wide[:, 80:], labels, up), want)
    flat = torch.empty(1 + 90 * 80, dtype=BF16, device="cuda")
    flat[1:] = hb.reshape(-1)
    check_all(run_ce(flat[1:].view(90, 80), w.to(BF16), labels.repeat_interleave(2)[::2], up), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_ce(hb, w.to(BF16), labels, up)
    torch.cuda.current_stream().wait_stream(side)
    check_all(got, want)
    hd = h.double().requires_grad_(True)
    loss = mr.linear_cross_entropy(hd, w, labels)
    (dh,) = torch.autograd.grad(loss, hd)
    assert dh.dtype == torch.float64
    check("dhidden", dh.float(), orc.cross_entropy(h, w, labels, up)[1])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_repeatable_and_only_what_is_wanted(dtype):
    g, h, w, labels = head_inputs(520, 136, 3000, dtype, 14)
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    loss = mr.linear_cross_entropy(h, w, labels, z_loss=1e-4)
    dh, dw = torch.autograd.grad(loss, (h, w), retain_graph=True)
    again = torch.autograd.grad(loss, (h, w))
    assert torch.equal(dh, again[0]) and torch.equal(dw, again[1])
    with torch.no_grad():
        assert torch.equal(mr.linear_cross_entropy(h, w, labels, z_loss=1e-4), loss)
    only_h = torch.autograd.grad(mr.linear_cross_entropy(h, w.detach(), labels, z_loss=1e-4), h)[0]
    only_w = torch.autograd.grad(mr.linear_cross_entropy(h.detach(), w, labels, z_loss=1e-4), w)[0]
    assert torch.equal(only_h, dh) and torch.equal(only_w, dw)


def test_gradient_along_a_direction():
    """Differences of the loss itself, in fp32: step 1e-2, third-order term and the loss's own
    rounding (1e-6 of it over the step) leave about 1e-3 of the slope."""
    g, h, w, labels = head_inputs(64, 96, 800, F32, 15)
    t, ids = teacher(g, 64, 8, 800, labels, absent=0.1)
    up = torch.ones((), device="cuda")
    for run, f in ((lambda: run_ce(h, w, labels, up, z_loss=1e-2),
                    lambda a, b: mr.linear_cross_entropy(a, b, labels, z_loss=1e-2)),
                   (lambda: run_kd(h, w, t, ids, up, temperature=2.0),
                    lambda a, b: mr.linear_distillation(a, b, t, ids, temperature=2.0))):
        _, dh, dw = run()
        for grad, step in ((dh, lambda e: f(h + e * dh / dh.norm(), w)), (dw, lambda e: f(h, w + e * dw / dw.norm()))):
            slope = float(step(1e-2).double() - step(-1e-2).double()) / 2e-2
            assert abs(slope - float(grad.norm())) < 2e-3 * float(grad.norm()) + 1e-4


def test_weight_past_2_31_elements():
    rows, D, V = 3, 8200, 262400
    w = torch.empty(V, D, dtype=BF16, device="cuda").normal_(generator=gen(2)) * 0.01
    h = randn(gen(3), rows, D).to(BF16)
    labels = torch.tensor([V - 1, 0, V - 2], device="cuda")
    loss, dh, dw = run_ce(h, w, labels, torch.ones((), device="cuda"))
    z = torch.cat([h.double() @ c.double().T for c in w.split(16384)], 1)
    lse = torch.logsumexp(z, 1)
    check("loss", loss, (lse - z.gather(1, labels[:, None])[:, 0]).mean())
    dz = torch.exp(z - lse[:, None]) / rows
    dz[torch.arange(3), labels] -= 1 / rows
    check("dhidden", dh, sum(dz[:, i:i + 16384] @ w[i:i + 16384].double() for i in range(0, V, 16384)))
    check("dweight's end", dw[-40:], dz[:, -40:].T @ h.double())
    check("dweight's start", dw[:40], dz[:, :40].T @ h.double())


def test_async_status_is_clean():
    _lib.async_status()


def test_python_and_cpp_bindings_agree(monkeypatch):
    """The C++ autograd nodes and the Python Functions make the same calls: the same bits."""
    assert _lib.autograd_ext() is not None

    def everything():
        g = gen(21)
        x, w, b = (t.requires_grad_(True) for t in (randn(g, 30, 100), randn(g, 100), randn(g, 100)))
        y = mr.layer_norm(x, w, b, out_dtype=BF16)
        out = [y, *torch.autograd.grad(y, (x, w, b), torch.ones_like(y))]
        y = mr.layer_norm(x, None, b.detach())
        out += [y, *torch.autograd.grad(y, (x,), torch.ones_like(y))]
        g, h, w, labels = head_inputs(50, 64, 700, BF16, 22)
        t, ids = teacher(g, 50, 7, 700, labels)
        one = torch.ones((), device="cuda")
        out += run_ce(h, w, labels, one, z_loss=1e-3) + run_kd(h, w, t, ids, one, temperature=2.0, reduction="sum")
        with torch.no_grad():
            out += [mr.layer_norm(x), mr.linear_cross_entropy(h, w, labels, reduction="none")]
        return out

    cpp = everything()
    monkeypatch.setattr(_lib, "autograd_ext", lambda: None)
    for a, b in zip(cpp, everything()):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_example_learns():
    """The example's model (norm, scan, norm, both losses together) learns the chain it is trained on."""
    import importlib.util
    import pathlib
    path = pathlib.Path(__file__).resolve().parents[1] / "examples" / "train_head.py"
    spec = importlib.util.spec_from_file_location("train_head", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    history = example.train(steps=30, vocab=300, width=64, batch=8, length=64, report=lambda line: print(line, flush=True))
    first, last = history[0], history[-1]
    assert all(math.isfinite(v) for pair in history for v in pair)
    assert last[0] < 0.8 * first[0] and last[1] < 0.8 * first[1]


def test_graph_replays():
    """A step of the losses and the norm, captured in a HIP graph: every replay gives the eager bits."""
    g, h, w, labels = head_inputs(300, 72, 1000, BF16, 31)
    labels[::6] = -100
    t, ids = teacher(g, 300, 9, 1000, labels.clamp(min=0))
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    scale = torch.ones(72, dtype=BF16, device="cuda").requires_grad_(True)
    one = torch.ones((), device="cuda")

    def step():
        n = mr.layer_norm(h, scale)
        ce, kd = mr.linear_cross_entropy(n, w, labels), mr.linear_distillation(n, w, t, ids, temperature=2.0)
        return (ce, kd, *torch.autograd.grad((ce, kd), (h, w, scale), (one, one)))

    eager = [a.detach().clone() for a in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        for a in out:
            a.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(out, eager):
            assert torch.equal(a, e)
        for a, e in zip(step(), eager):
            assert torch.equal(a, e)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,D,V", [(1, 8, 2), (20, 200, 257), (50, 3000, 300), (200, 100, 513), (300, 1000, 5003),
                                      (700, 320, 4096), (3001, 200, 641)])
def test_kernels_write_inside_their_buffers(rows, D, V, dtype, monkeypatch):
    """State and workspaces of exactly the stated sizes between guards: nothing is written outside them, and
    what they held before does not matter."""
    buffers = []

    def guarded(n, device):
        whole = torch.full((n + 8192,), 0xA5, dtype=torch.uint8, device=device)
        whole[4096:4096 + n] = 0xFF   # NaN as a float
        buffers.append((whole, n))
        return whole[4096:4096 + n]

    g, h, w, labels = head_inputs(rows, D, V, dtype, rows + D + V)
    labels[1::3] = -100
    t, ids = teacher(g, rows, 9, V, labels.clamp(min=0))
    up = torch.rand(rows, generator=g, device="cuda") + 0.1
    want = (run_ce(h, w, labels, up, reduction="none"), run_kd(h, w, t, ids, up, reduction="none"))
    monkeypatch.setattr(_lib, "autograd_ext", lambda: None)
    monkeypatch.setattr(_lib, "_alloc_ws", guarded)
    got = (run_ce(h, w, labels, up, reduction="none"), run_kd(h, w, t, ids, up, reduction="none"))
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            assert torch.equal(x, y)
    assert len(buffers) == 6
    for whole, n in buffers:
        assert (whole[:4096] == 0xA5).all() and (whole[4096 + n:] == 0xA5).all()
