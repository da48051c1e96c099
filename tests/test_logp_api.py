"""Losses on log-probabilities on the CPU: the 64-bit formulas against differences, the public plain
forms against the formulas, the refusals of the public functions, and the C ABI's argument checks (no
kernel runs)."""
import ctypes
import math
import os
import subprocess
import sys

import pytest
import torch

import mlx_recurrence_amd as mr
from mlx_recurrence_amd import _lib
from tests import logp_oracle as orc
from tests.test_host_sanitize import ROOT, SAN_LIB, _asan_runtime

F64 = torch.float64
# In 64 bits a central difference of step 1e-5 is off by about eps^2 f''' and 1e-16 f / eps: 1e-10.
DIFF = 1e-7


def _rand(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=F64)


def _differences(f, x, d, eps=1e-5):
    return float((f(x + eps * d) - f(x - eps * d)) / (2 * eps))


def _inputs():
    h, w = _rand(3, 2, 4, 5), _rand(11, 5, seed=1)
    labels = torch.randint(0, 11, (3, 2, 4), generator=torch.Generator().manual_seed(2))
    labels[0, 0, 1], labels[1, 1, 3] = -100, -100
    labels[2] = -100
    old = orc.log_probs(h, w, labels, torch.zeros(3, 2, 4, dtype=F64))[0] - 0.4 * _rand(3, 2, 4, seed=3)
    return h, w, labels, old, old + 0.2 * _rand(3, 2, 4, seed=4), _rand(3, 2, 4, seed=5)


def _calls(reduction):
    h, w, labels, old, ref, A = _inputs()
    up = _rand(3, 2, 4, seed=6) if reduction == "none" else torch.tensor(1.7, dtype=F64)
    pairs = _rand(3, seed=7) if reduction == "none" else up
    sums = 10 * _rand(3, 2, seed=8)
    calls = [(lambda a, b: orc.policy(a, b, labels, A, old, ref, up, kl=0.3, tau=1.3, reduction=reduction),
              lambda a, b: mr.linear_policy_loss_reference(a, b, labels, A, old, ref, kl_weight=0.3, temperature=1.3,
                                                           reduction=reduction), up),
             (lambda a, b: orc.policy(a, b, labels, A[..., :1], old, None, up, clip=(0.1, 0.5), reduction=reduction),
              lambda a, b: mr.linear_policy_loss_reference(a, b, labels, A[..., :1], old, clip=(0.1, 0.5), reduction=reduction),
              up),
             (lambda a, b: orc.preference(a, b, labels, sums, pairs, beta=0.3, eps=0.2, reduction=reduction),
              lambda a, b: mr.linear_preference_loss_reference(a, b, labels, sums, beta=0.3, label_smoothing=0.2,
                                                               reduction=reduction), pairs),
             (lambda a, b: orc.preference(a, b, labels, None, pairs, beta=0.7, reduction=reduction),
              lambda a, b: mr.linear_preference_loss_reference(a, b, labels, beta=0.7, reduction=reduction), pairs)]
    if reduction == "none":
        calls.append((lambda a, b: orc.log_probs(a, b, labels, up, tau=0.6),
                      lambda a, b: mr.linear_log_probs_reference(a, b, labels, temperature=0.6), up))
    return h, w, calls


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_formulas_against_differences(reduction):
    h, w, calls = _calls(reduction)
    for run, _, up in calls:
        _, dh, dw, _ = run(h, w)
        value = lambda a, b: (run(a, b)[0] * up).sum()  # noqa: E731
        d = _rand(*h.shape, seed=9)
        assert abs(_differences(lambda v: value(v, w), h, d) - float((dh * d).sum())) < DIFF
        d = _rand(*w.shape, seed=10)
        assert abs(_differences(lambda v: value(h, v), w, d) - float((dw * d).sum())) < DIFF


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_plain_forms_are_the_formulas(reduction):
    h, w, calls = _calls(reduction)
    h = h.clone()
    h[2, 1, 0] = math.nan   # a row that counts for nothing
    for formula, plain, up in calls:
        leaves = [t.clone().requires_grad_(True) for t in (h, w)]
        out = plain(*leaves)
        for a, e in zip((out, *torch.autograd.grad(out, leaves, up)), formula(h, w)):
            assert a.shape == e.shape and torch.allclose(a, e, rtol=0, atol=1e-12)


def test_plain_policy_of_this_step_and_beyond_the_range():
    h, w, labels, old, _, A = _inputs()
    leaves = [t.float().requires_grad_(True) for t in (h, w)]
    loss = mr.linear_policy_loss_reference(*leaves, labels, A.float(), None, reduction="none")
    valid = labels != -100
    assert torch.allclose(loss, torch.where(valid, -A, 0).float()) and torch.autograd.grad(loss.sum(), leaves)[0].any()
    far = (old - 500).float()
    for adv in (A.abs().float(), torch.zeros(3, 2, 4)):
        loss = mr.linear_policy_loss_reference(*leaves, labels, adv, far, reduction="none")
        assert torch.allclose(loss, torch.where(valid, -1.2 * adv, 0))
        assert not any(t.any() for t in torch.autograd.grad(loss.sum(), leaves))


# ------------------------------------------------------------------ refusals
def _zeros(*shape):
    return torch.zeros(shape)


def test_refusals_of_all_three():
    h, w, l, A = _zeros(3, 2, 4, 8), _zeros(10, 8), torch.zeros(3, 2, 4, dtype=torch.int64), _zeros(3, 2, 4)
    for fn, more in ((mr.linear_log_probs, ()), (mr.linear_policy_loss, (A,)), (mr.linear_preference_loss, ())):
        for bad in (_zeros(10, 7), _zeros(8), _zeros(0, 8)):
            with pytest.raises(ValueError, match="weight must be"):
                fn(h, bad, l, *more)
        with pytest.raises(ValueError, match="labels must be"):
            fn(h, w, l[:2], *more)
        with pytest.raises(TypeError, match="labels must be integers"):
            fn(h, w, l.float(), *more)
        with pytest.raises(ValueError, match="hidden must be"):
            fn(_zeros(3, 2, 4, 0), _zeros(10, 0), l, *more)
        with pytest.raises(RuntimeError, match="run on a ROCm GPU"):
            fn(h, w, l, *more)
        if fn is not mr.linear_log_probs:
            with pytest.raises(ValueError, match="reduction"):
                fn(h, w, l, *more, reduction="batch")
        if fn is not mr.linear_preference_loss:
            for tau in (0.0, -1.0, math.inf, math.nan):
                with pytest.raises(ValueError, match="temperature"):
                    fn(h, w, l, *more, temperature=tau)


def test_policy_refusals():
    h, w, l, A = _zeros(3, 4, 8), _zeros(10, 8), torch.zeros(3, 4, dtype=torch.int64), _zeros(3, 4)
    for bad in (_zeros(3), _zeros(4), _zeros(1, 4), _zeros(3, 2), _zeros(12)):
        with pytest.raises(ValueError, match=r"advantages must be \[3, 4\] or \[3, 1\]"):
            mr.linear_policy_loss(h, w, l, bad)
    with pytest.raises(TypeError, match="advantages must be floating-point"):
        mr.linear_policy_loss(h, w, l, l)
    with pytest.raises(ValueError, match="old_log_probs must be"):
        mr.linear_policy_loss(h, w, l, A, A[:, :1])
    with pytest.raises(ValueError, match="ref_log_probs must be"):
        mr.linear_policy_loss(h, w, l, A, A, A[0])
    with pytest.raises(ValueError, match="kl_weight needs ref_log_probs"):
        mr.linear_policy_loss(h, w, l, A, A, kl_weight=0.1)
    for kl in (-0.1, math.nan, math.inf):
        with pytest.raises(ValueError, match="kl_weight must be"):
            mr.linear_policy_loss(h, w, l, A, A, A, kl_weight=kl)
    for clip in (-0.1, (0.2, -0.1), (math.nan, 0.1), math.nan):
        with pytest.raises(ValueError, match="clip must be"):
            mr.linear_policy_loss(h, w, l, A, A, clip=clip)


def test_preference_refusals():
    h, w, l = _zeros(3, 2, 4, 8), _zeros(10, 8), torch.zeros(3, 2, 4, dtype=torch.int64)
    with pytest.raises(ValueError, match=r"labels must be \[..., 2, L\]"):
        mr.linear_preference_loss(h.transpose(0, 1), w, l.transpose(0, 1))
    with pytest.raises(ValueError, match=r"labels must be \[..., 2, L\]"):
        mr.linear_preference_loss(h[0, 0], w, l[0, 0])
    for bad in (_zeros(3), _zeros(3, 2, 4), _zeros(2, 3)):
        with pytest.raises(ValueError, match=r"ref_log_probs must be \[3, 2\]"):
            mr.linear_preference_loss(h, w, l, bad)
    with pytest.raises(TypeError, match="ref_log_probs must be floating-point"):
        mr.linear_preference_loss(h, w, l, l[..., 0])
    for beta in (0.0, -0.1, math.inf, math.nan):
        with pytest.raises(ValueError, match="beta"):
            mr.linear_preference_loss(h, w, l, beta=beta)
    for eps in (-0.1, 0.6, math.nan):
        with pytest.raises(ValueError, match="label_smoothing"):
            mr.linear_preference_loss(h, w, l, label_smoothing=eps)


def test_preference_keeps_what_sums_in_64_bits_differ_by(monkeypatch):
    """Rounded to fp32, sums of 2^17 and more are off by up to 2^-7 each."""
    h, w, l = _zeros(3, 2, 4, 8), _zeros(10, 8), torch.zeros(3, 2, 4, dtype=torch.int64)
    given = []
    monkeypatch.setattr(mr.linear_logp, "_apply", lambda *a: given.append(a[6]) or _zeros(3))
    ref = 3 * _rand(3, 2, seed=1)
    want = ref[:, 0] - ref[:, 1]
    for offset in (0.0, -3000.0, -200_000.0):
        sums = ref + offset   # exact but for 2^-36
        mr.linear_preference_loss(h, w, l, sums)
        got = given[-1].float().double()   # as the kernel takes it: rounded, then subtracted in 64 bits
        assert ((got[:, 0] - got[:, 1] - want).abs() <= 2.0 ** -24 * want.abs() + 2.0 ** -34).all()
    for sums in (ref.float(), ref.bfloat16()):
        mr.linear_preference_loss(h, w, l, sums)
        assert given[-1] is sums
    mr.linear_preference_loss(h, w, l)
    assert given[-1] is None


def test_c_abi_refusals():
    """Argument errors are found before any work is enqueued (the pointers are never read)."""
    lib, p, odd = _lib.load(), ctypes.c_void_p(16), ctypes.c_void_p(24)
    big = 1 << 40
    head = dict(h=p, w=p, dt=1, rows=8, D=8, V=10, l=p, ig=-100)
    tail = dict(st=p, sn=big, ws=p, wn=big, s=None)
    lp = lambda **k: lib.rr_linear_logp_fwd(*{**head, "tau": 1.0, "out": p, **tail, **k}.values())  # noqa: E731
    po = lambda **k: lib.rr_linear_policy_fwd(*{**head, "tau": 1.0, "a": p, "per": 1, "old": p, "ref": p, "lo": 0.2,  # noqa: E731
                                                "hi": 0.2, "kl": 0.1, "red": 1, "out": p, **tail, **k}.values())
    pair = dict(h=p, w=p, dt=1, pairs=2, L=2, D=8, V=10, l=p, ig=-100, ref=p, beta=0.1, eps=0.0, red=1, out=p, **tail)
    pr = lambda **k: lib.rr_linear_preference_fwd(*{**pair, **k}.values())  # noqa: E731
    state, ws = (lib.rr_linear_loss_state_bytes(8, 8, 10, 1, 1, 0), lib.rr_linear_loss_workspace_bytes(8, 8, 10, 1, 0))
    for fn in (lp, po, pr):
        for bad in (dict(D=0), dict(V=0), dict(dt=9), dict(h=None), dict(w=None), dict(l=None), dict(out=None), dict(st=None),
                    dict(ws=None), dict(h=odd), dict(w=odd)):
            assert fn(**bad) == _lib.RR_EINVAL, bad
        for bad in (dict(sn=state - 1), dict(st=odd), dict(ws=odd), dict(wn=ws - 1)):
            assert fn(**bad) == _lib.RR_EWORKSPACE, bad
        for bad in (dict(V=(1 << 24) + 1), dict(D=65537)):
            assert fn(**bad) == _lib.RR_EUNSUPPORTED, bad
    for fn in (lp, po):
        assert fn(rows=-1) == _lib.RR_EINVAL and fn(rows=1 << 24) == _lib.RR_EUNSUPPORTED
        for tau in (0.0, -1.0, math.inf, math.nan):
            assert fn(tau=tau) == _lib.RR_EINVAL
    for bad in (dict(a=None), dict(ref=None), dict(per=0), dict(lo=-0.1), dict(hi=math.nan), dict(kl=-1.0), dict(kl=math.inf),
                dict(red=3)):
        assert po(**bad) == _lib.RR_EINVAL, bad
    for bad in (dict(pairs=-1), dict(L=-1), dict(beta=0.0), dict(beta=math.inf), dict(eps=0.6), dict(eps=-0.1), dict(red=-1)):
        assert pr(**bad) == _lib.RR_EINVAL, bad
    for bad in (dict(pairs=1 << 62), dict(L=1 << 62), dict(pairs=1 << 22, L=1 << 22), dict(pairs=1 << 20, L=8)):
        assert pr(**bad) == _lib.RR_EUNSUPPORTED, bad
    bw = lambda **k: lib.rr_linear_logp_bwd(*{**dict(dl=p, w=p, dt=1, rows=8, D=8, V=10, tau=1.0, group=1, itself=0, red=1,  # noqa: E731,E501
                                                     st=p, sn=big, dh=p, dw=p, ws=p, wn=big, s=None), **k}.values())
    for bad in (dict(dl=None), dict(w=None), dict(st=None), dict(tau=-1.0), dict(red=-1), dict(group=0), dict(group=1 << 40),
                dict(itself=1), dict(itself=1, red=0, group=2)):
        assert bw(**bad) == _lib.RR_EINVAL, bad
    assert bw(wn=lib.rr_linear_loss_workspace_bytes(8, 8, 10, 1, 2) - 1) == _lib.RR_EWORKSPACE
    assert bw(sn=state) == _lib.RR_EWORKSPACE   # that of a forward without a backward
    assert bw(dh=None, dw=None) == _lib.RR_OK


@pytest.mark.skipif(not SAN_LIB.exists(), reason="host-sanitizer build absent "
                    "(python mlx-recurrence_amd/build.py --host-sanitize)")
def test_host_code_under_asan_and_ubsan():
    env = dict(os.environ)
    env.update(LD_PRELOAD=str(_asan_runtime()), MLX_RECURRENCE_AMD_LIB=str(SAN_LIB),
               ASAN_OPTIONS="detect_leaks=0:abort_on_error=1", UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1")
    res = subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider", "tests/test_logp_api.py", "-k",
                          "abi or refus"], cwd=ROOT, env=env, capture_output=True, text=True, timeout=600)
    tail = (res.stdout + res.stderr)[-3000:]
    assert res.returncode == 0, tail
    assert "AddressSanitizer" not in tail and "runtime error" not in tail, tail
    assert " passed" in tail


@pytest.mark.parametrize("rows,D,V,dtype", [(8192, 2560, 65536, 1), (32768, 2560, 131072, 1), (1536, 768, 32000, 0),
                                            (1, 5120, 131072, 1), (100_000, 64, 32000, 2), (512, 65536, 2048, 1), (40, 64, 500, 2)])
def test_backward_workspace_holds_a_piece_of_the_gradient(rows, D, V, dtype):
    """A piece of the logits' gradient (512 MiB, or 2048 words of every row where those are more), dhidden's sums once and
    at most 128 MiB of parts, at most 256 MiB of dweight's, fp16: a copy of the hidden states."""
    lib, mib = _lib.load(), 1 << 20
    size, planes = (4, 1) if dtype == 0 else (2, 2 if rows <= 64 else 1)
    up = lambda a, b: (a + b - 1) // b * b  # noqa: E731
    rows_up = 32 if rows <= 32 else up(rows, 256)
    piece = max(512 * mib, 2048 * rows_up * size * planes)
    sums = rows_up * up(D, 256) * 4 + (128 + 256) * mib
    copy = rows * up(D, 64) * 2 if dtype == 2 else 0
    assert 0 < lib.rr_linear_loss_workspace_bytes(rows, D, V, dtype, 2) <= piece + sums + copy + rows_up * 16 + 4096


@pytest.mark.parametrize("rows,D,V", [(512, 512, 16001), (460, 512, 16001), (700, 768, 8000)])
def test_backward_workspace_of_fp32_has_no_parts_of_dweight_where_it_is_made_whole(rows, D, V):
    """The gradient of all logits, dhidden's sums, two tiles of 256 x 64 a slot of its 512, and two floats a row."""
    up = lambda a, b: (a + b - 1) // b * b  # noqa: E731
    rows_up = up(rows, 256)
    most = rows_up * up(V, 256) * 4 + rows_up * up(D, 256) * 4 + 1024 * 256 * 64 * 4 + rows_up * 8 + 4096
    assert 0 < _lib.load().rr_linear_loss_workspace_bytes(rows, D, V, 0, 2) <= most
