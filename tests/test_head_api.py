"""Output head on the CPU: the plain forms against 64-bit formulas, those formulas against
differences, the refusals of the public functions, and the C ABI's argument checks and
workspace sizes (no kernel runs)."""
import ctypes
import math

import pytest
import torch

import mlx_recurrence_amd as mr
from mlx_recurrence_amd import _lib
from tests import head_oracle as orc

F64 = torch.float64


def _rand(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=F64)


def _differences(f, x, d, eps=1e-5):
    return float((f(x + eps * d) - f(x - eps * d)) / (2 * eps))


# In 64 bits a central difference of step 1e-5 is off by about eps^2 f''' and 1e-16 f / eps: 1e-10.
DIFF = 1e-7


def test_layer_norm_formula_against_differences():
    x, w, b, dy = _rand(5, 7), _rand(7, seed=1), _rand(7, seed=2), _rand(5, 7, seed=3)
    _, dx, dw, db = orc.layer_norm(x, w, b, 1e-5, dy)
    for t, g, f in ((x, dx, lambda v: (orc.layer_norm(v, w, b, 1e-5) * dy).sum()),
                    (w, dw, lambda v: (orc.layer_norm(x, v, b, 1e-5) * dy).sum()),
                    (b, db, lambda v: (orc.layer_norm(x, w, v, 1e-5) * dy).sum())):
        d = _rand(*t.shape, seed=9)
        assert abs(_differences(f, t, d) - float((g * d).sum())) < DIFF


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("kind", ["ce", "kd"])
def test_loss_formulas_against_differences(kind, reduction):
    h, w = _rand(6, 5), _rand(11, 5, seed=1)
    up = _rand(6, seed=2) if reduction == "none" else torch.tensor(1.7, dtype=F64)
    if kind == "ce":
        labels = torch.tensor([3, -100, 10, 0, 3, -100])
        run = lambda a, b: orc.cross_entropy(a, b, labels, up, zl=0.01, reduction=reduction)  # noqa: E731
    else:
        t = _rand(6, 3, seed=4)
        ids = torch.tensor([[1, 2, 3], [-1, -1, -1], [10, -1, 4], [0, 0, 5], [7, 8, 9], [-1, 2, -1]])
        run = lambda a, b: orc.distillation(a, b, t, ids, up, tau=1.5, reduction=reduction)  # noqa: E731
    _, dh, dw = run(h, w)
    value = lambda a, b: (run(a, b)[0] * up).sum()  # noqa: E731
    d = _rand(6, 5, seed=5)
    assert abs(_differences(lambda v: value(v, w), h, d) - float((dh * d).sum())) < DIFF
    d = _rand(11, 5, seed=6)
    assert abs(_differences(lambda v: value(h, v), w, d) - float((dw * d).sum())) < DIFF


def test_plain_forms_are_the_formulas():
    """The public plain forms (autograd) in 64 bits against the written-out gradients."""
    x, w, b, dy = (_rand(4, 9), _rand(9, seed=1), _rand(9, seed=2), _rand(4, 9, seed=3))
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = mr.layer_norm_reference(*leaves)
    got = (y, *torch.autograd.grad(y, leaves, dy))
    for a, e in zip(got, orc.layer_norm(x, w, b, 1e-5, dy)):
        assert torch.allclose(a, e, rtol=0, atol=1e-12)
    h, w = _rand(6, 5), _rand(11, 5, seed=1)
    labels = torch.tensor([3, -100, 10, 0, 3, -100])
    t = _rand(6, 3, seed=4)
    t[4, 1] = -math.inf
    ids = torch.tensor([[1, 2, 3], [-1, -1, -1], [10, -1, 4], [0, 0, 5], [7, 8, 9], [-1, 2, -1]])
    h[1] = math.nan   # a row that counts for nothing
    for reduction in ("mean", "sum", "none"):
        up = _rand(6, seed=2) if reduction == "none" else torch.tensor(1.7, dtype=F64)
        for fn, want in ((lambda a, c: mr.linear_cross_entropy_reference(a, c, labels, z_loss=0.01, reduction=reduction),
                          orc.cross_entropy(h, w, labels, up, zl=0.01, reduction=reduction)),
                         (lambda a, c: mr.linear_distillation_reference(a, c, t, ids, temperature=1.5, reduction=reduction),
                          orc.distillation(h, w, t, ids, up, tau=1.5, reduction=reduction))):
            leaves = [v.clone().requires_grad_(True) for v in (h, w)]
            loss = fn(*leaves)
            for a, e in zip((loss, *torch.autograd.grad(loss, leaves, up)), want):
                assert torch.allclose(a, e, rtol=0, atol=1e-12)


# ------------------------------------------------------------------ refusals
def test_layer_norm_refusals():
    x, w = torch.zeros(3, 8), torch.zeros(8)
    with pytest.raises(ValueError, match=r"weight must be \[D\] = \[8\]"):
        mr.layer_norm(x, torch.zeros(7))
    with pytest.raises(ValueError, match=r"bias must be \[D\] = \[8\]"):
        mr.layer_norm(x, w, torch.zeros(1, 8))
    with pytest.raises(ValueError, match="D > 0"):
        mr.layer_norm(torch.zeros(3, 0))
    with pytest.raises(ValueError, match="D > 0"):
        mr.layer_norm(torch.zeros(()))
    with pytest.raises(ValueError, match="eps"):
        mr.layer_norm(x, w, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        mr.layer_norm(x, w, eps=math.nan)
    with pytest.raises(ValueError, match="out_dtype"):
        mr.layer_norm(x.bfloat16(), w, out_dtype=torch.float32)
    with pytest.raises(ValueError, match="out_dtype"):
        mr.layer_norm(x, w, out_dtype=torch.float64)
    with pytest.raises(TypeError, match="unsupported input dtype"):
        mr.layer_norm(x.long())
    with pytest.raises(RuntimeError, match="run on a ROCm GPU"):
        mr.layer_norm(x, w)


def test_cross_entropy_refusals():
    h, w, l = torch.zeros(3, 8), torch.zeros(10, 8), torch.zeros(3, dtype=torch.int64)
    for bad in (torch.zeros(10, 7), torch.zeros(8), torch.zeros(0, 8)):
        with pytest.raises(ValueError, match="weight must be"):
            mr.linear_cross_entropy(h, bad, l)
    with pytest.raises(ValueError, match="labels must be"):
        mr.linear_cross_entropy(h, w, l[:2])
    with pytest.raises(TypeError, match="labels must be integers"):
        mr.linear_cross_entropy(h, w, l.float())
    with pytest.raises(TypeError, match="labels must be integers"):
        mr.linear_cross_entropy(h, w, l.bool())
    with pytest.raises(ValueError, match="reduction"):
        mr.linear_cross_entropy(h, w, l, reduction="batch")
    with pytest.raises(ValueError, match="z_loss"):
        mr.linear_cross_entropy(h, w, l, z_loss=math.inf)
    with pytest.raises(ValueError, match="hidden must be"):
        mr.linear_cross_entropy(torch.zeros(3, 0), torch.zeros(10, 0), l)
    with pytest.raises(RuntimeError, match="run on a ROCm GPU"):
        mr.linear_cross_entropy(h, w, l)


def test_distillation_refusals():
    h, w = torch.zeros(3, 8), torch.zeros(10, 8)
    t, i = torch.zeros(3, 4), torch.zeros(3, 4, dtype=torch.int64)
    with pytest.raises(ValueError, match="teacher_ids must be"):
        mr.linear_distillation(h, w, t[:2], i[:2])
    with pytest.raises(ValueError, match="teacher_ids must be"):
        mr.linear_distillation(h, w, t[:, :0], i[:, :0])
    with pytest.raises(ValueError, match="must match"):
        mr.linear_distillation(h, w, t[:, :2], i)
    with pytest.raises(TypeError, match="teacher_ids must be integers"):
        mr.linear_distillation(h, w, t, t)
    for tau in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            mr.linear_distillation(h, w, t, i, temperature=tau)
    with pytest.raises(RuntimeError, match="run on a ROCm GPU"):
        mr.linear_distillation(h, w, t, i)


def test_c_abi_refusals():
    """Argument errors are found before any work is enqueued (the pointers are never read)."""
    lib, p, odd = _lib.load(), ctypes.c_void_p(16), ctypes.c_void_p(24)
    big = 1 << 40
    ln = lambda **k: lib.rr_layer_norm_fwd(*{**dict(x=p, xd=1, w=p, b=p, wd=1, rows=4, D=8, eps=1e-5, y=p, yd=1, m=p, r=p,  # noqa: E731,E501
                                                    s=None), **k}.values())
    assert ln(D=0) == _lib.RR_EINVAL and ln(rows=-1) == _lib.RR_EINVAL and ln(xd=5) == _lib.RR_EINVAL
    assert ln(yd=0) == _lib.RR_EINVAL and b"y has x's dtype" in lib.rr_last_error()
    assert ln(eps=-1.0) == _lib.RR_EINVAL and ln(x=None) == _lib.RR_EINVAL and ln(m=None) == _lib.RR_EINVAL
    assert ln(D=32769) == _lib.RR_EUNSUPPORTED and b"32768 channels" in lib.rr_last_error()
    assert ln(rows=0, x=None) == _lib.RR_OK
    need = lib.rr_layer_norm_bwd_workspace_bytes(4, 8)
    assert need > 0
    lnb = lambda **k: lib.rr_layer_norm_bwd(*{**dict(dy=p, yd=1, x=p, xd=1, w=p, wd=1, m=p, r=p, rows=4, D=8, dx=p, dw=p,  # noqa: E731,E501
                                                     db=p, ws=p, n=need, s=None), **k}.values())
    assert lnb(dy=None) == _lib.RR_EINVAL and lnb(m=None) == _lib.RR_EINVAL
    assert lnb(n=need - 1) == _lib.RR_EWORKSPACE and lnb(ws=odd) == _lib.RR_EWORKSPACE
    ce = lambda **k: lib.rr_linear_ce_fwd(*{**dict(h=p, w=p, dt=1, rows=4, D=8, V=10, l=p, ig=-100, z=0.0, red=1, loss=p,  # noqa: E731,E501
                                                   st=p, sn=big, ws=p, wn=big, s=None), **k}.values())
    for bad in (dict(rows=-1), dict(D=0), dict(V=0), dict(dt=9), dict(red=3), dict(h=None), dict(w=None), dict(l=None),
                dict(loss=None), dict(st=None), dict(ws=None), dict(h=odd), dict(w=odd)):
        assert ce(**bad) == _lib.RR_EINVAL, bad
    for bad in (dict(sn=lib.rr_linear_loss_state_bytes(4, 8, 10, 1, 1, 0) - 1), dict(st=odd), dict(ws=odd),
                dict(wn=lib.rr_linear_loss_workspace_bytes(4, 8, 10, 1, 0) - 1)):
        assert ce(**bad) == _lib.RR_EWORKSPACE, bad
    for bad in (dict(V=(1 << 24) + 1), dict(D=65537), dict(rows=1 << 24)):
        assert ce(**bad) == _lib.RR_EUNSUPPORTED, bad
    kd = lambda **k: lib.rr_linear_kd_fwd(*{**dict(h=p, w=p, dt=1, rows=4, D=8, V=10, tl=p, td=0, ti=p, K=3, tau=1.0, red=1,  # noqa: E731,E501
                                                   loss=p, st=p, sn=big, ws=p, wn=big, s=None), **k}.values())
    for bad in (dict(td=4), dict(tau=0.0), dict(tau=math.inf), dict(tau=math.nan), dict(tl=None), dict(ti=None)):
        assert kd(**bad) == _lib.RR_EINVAL, bad
    for bad in (dict(K=0), dict(K=1025)):
        assert kd(**bad) == _lib.RR_EUNSUPPORTED, bad
    bw = lambda **k: lib.rr_linear_loss_bwd(*{**dict(dl=p, w=p, dt=1, rows=4, D=8, V=10, K=3, z=0.0, tau=1.0, red=1,  # noqa: E731,E501
                                                     st=p, sn=big, dh=p, dw=p, ws=p, wn=big, s=None), **k}.values())
    for bad in (dict(dl=None), dict(w=None), dict(st=None), dict(tau=-1.0), dict(red=-1)):
        assert bw(**bad) == _lib.RR_EINVAL, bad
    assert bw(wn=lib.rr_linear_loss_workspace_bytes(4, 8, 10, 1, 1) - 1) == _lib.RR_EWORKSPACE
    # the state of a forward without a backward does not do for one
    assert bw(sn=lib.rr_linear_loss_state_bytes(4, 8, 10, 3, 1, 1) - 1) == _lib.RR_EWORKSPACE
    assert bw(sn=lib.rr_linear_loss_state_bytes(4, 8, 10, 3, 1, 0)) == _lib.RR_EWORKSPACE
    assert bw(dh=None, dw=None) == _lib.RR_OK


@pytest.mark.parametrize("rows,D,V,dtype", [(8192, 2560, 65536, 1), (32768, 2560, 131072, 1), (1536, 768, 32000, 0),
                                            (1, 5120, 131072, 1), (100_000, 64, 32000, 2)])
def test_many_logits_are_not_held(rows, D, V, dtype):
    """The backward's workspace holds a piece of the logits' gradient, not all of it: beside the
    gradients' parts at most about 512 MiB, or 2048 columns of every row.
    The state holds the logits of up to 256 rows, of more where they take
    4 GiB at most."""
    lib, planes = _lib.load(), 2 if dtype == 0 else 1
    rows_up = (rows + 255) // 256 * 256
    pieces = max(512 << 20, 2048 * rows_up * 2 * planes) + (256 * rows_up * 2 * planes)
    copies = planes * 2 * (rows + (V if dtype == 0 else 0)) * (D + 63) // 64 * 64
    parts = 64 * rows_up * ((D + 255) // 256 * 256) * 4
    assert lib.rr_linear_loss_workspace_bytes(rows, D, V, dtype, 1) <= pieces + parts + (1 << 20)
    assert lib.rr_linear_loss_workspace_bytes(rows, D, V, dtype, 0) <= 8 * rows_up * (V + 255) // 32 + (1 << 20)
    state = [lib.rr_linear_loss_state_bytes(rows, D, V, 4, dtype, grad) for grad in (0, 1)]
    assert state[0] <= copies + rows * (4 * 4 + 3 * 4 * 4) + (1 << 20)   # K = 4 entries a row
    logits = rows * ((V + 255) // 256 * 256) * 4
    held = rows <= 256 or logits <= 4 << 30
    assert state[1] - state[0] in ((0, logits) if held else (0,))
    assert state[1] - state[0] == logits or rows > 256
