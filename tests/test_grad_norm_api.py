"""The norm of gradients and their clipping on the CPU: the plain forms, the refusals of the public
functions, and the C ABI's argument checks (no kernel runs)."""
import contextlib
import ctypes
import math
import os
import subprocess
import sys

import pytest
import torch

import mlx_recurrence_amd as mr
from mlx_recurrence_amd import _lib
from mlx_recurrence_amd.grad_norm import _dense
from tests.test_host_sanitize import ROOT, SAN_LIB, _asan_runtime


def test_plain_forms():
    g = [torch.tensor([3.0, 0.0]), torch.tensor([[4.0]]), None, torch.zeros(0)]
    assert float(mr.global_grad_norm_reference(g)) == 5.0
    norm, out = mr.clip_grad_norm_reference(g, 2.5)
    assert float(norm) == 5.0 and torch.equal(out[0], torch.tensor([1.5, 0.0])) and float(out[1]) == 2.0 and len(out) == 3
    for most in (5.0, 7.0, math.inf):
        assert all(torch.equal(a, b) for a, b in zip(mr.clip_grad_norm_reference(g, most)[1], mr.grad_norm._tensors(g)))
    for bad in (math.inf, math.nan):
        norm, out = mr.clip_grad_norm_reference([torch.tensor([bad, 1.0])], 0.5)
        assert not math.isfinite(float(norm)) and float(out[0][1]) == 1.0
    assert not mr.clip_grad_norm_reference([torch.tensor([3.0])], 0.0)[1][0].any()


def test_what_lies_without_gaps():
    t = torch.zeros(4, 6, 5)
    assert _dense(t) and _dense(t.transpose(0, 2)) and _dense(t[:2]) and _dense(t[:, :1, :1][:1]) and _dense(t.permute(1, 2, 0))
    assert not _dense(t[:, :3]) and not _dense(t[..., ::2]) and not _dense(t[:1, :1].expand(4, 6, 5))
    for v in (t, t.transpose(0, 2), t[:, :3], t[..., ::2], t[:0], t[:1], t[:1, :1].expand(4, 6, 5)):
        assert _dense(v) == torch.ops.aten.is_non_overlapping_and_dense(v)


@pytest.mark.parametrize("python", [False, True])
def test_refusals(python, monkeypatch):
    if python:
        monkeypatch.setattr(_lib, "_autograd_mod", None)
    t = torch.zeros(4)
    for call in (mr.global_grad_norm, lambda g: mr.clip_grad_norm(g, 1.0)):
        for none in ([], [None, None], ()):
            with pytest.raises(ValueError, match="no gradients"):
                call(none)
        for one in ([t], t, [None, t]):
            with pytest.raises(RuntimeError, match="run on a ROCm GPU"):
                call(one)
        with pytest.raises((TypeError, RuntimeError)):
            call([t.to_sparse()])
    for most in (-1.0, math.nan, -math.inf):
        with pytest.raises(ValueError, match="max_norm must not be negative"):
            mr.clip_grad_norm([t], most)
    with pytest.raises(ValueError, match="out must have a tensor for each gradient"):
        mr.clip_grad_norm([t], 1.0, out=[t, t])
    with pytest.raises(ValueError, match="out must have a tensor of each gradient's shape"):
        mr.clip_grad_norm([t], 1.0, out=[None])


def test_outputs_of_another_layout_share_no_memory(monkeypatch):
    """Outputs that are copied to are checked too, together with those written directly (the library replaced
    by the plain form)."""
    monkeypatch.setattr(_lib, "_autograd_mod", None)
    monkeypatch.setattr(_lib, "autograd_ext", lambda: None)
    monkeypatch.setattr(_lib, "require_device", lambda *t: t[0].device)
    monkeypatch.setattr(_lib, "device_guard", lambda dev: contextlib.nullcontext())

    def plain(grads, out, max_norm, norm):
        n, scaled = mr.clip_grad_norm_reference(grads, max_norm)
        norm.copy_(n)
        for o, v in zip(out, scaled):
            o.copy_(v)

    monkeypatch.setattr(_lib, "grad_norm", plain)
    a, b, o = torch.ones(4, 4), torch.full((4, 4), 2.0).T, torch.zeros(8, 4)
    assert a.stride() != b.stride()
    for grads, out in (([a, b], [o[:4], o[:4]]), ([a, b], [o[:4], o[1:5]]), ([b, a], [o[1:5], o[:4]]), ([b, b], [o[:4], o[2:6]]),
                       ([a, b[:2]], [o[:4], o[:4:2]]), ([b[:2], b[:2]], [o[:4:2], o[:4:2]])):
        with pytest.raises(ValueError, match="share memory"):
            mr.clip_grad_norm(grads, 1.0, out=out)
    assert not o.any()
    mr.clip_grad_norm([a, b, b[:1]], 1.0, out=[o[:4], o[4:], torch.zeros(1, 4)])   # one behind the other
    f = 1 / math.sqrt(16 + 4 * 16 + 16)
    assert torch.allclose(o[:4], a * f) and torch.allclose(o[4:], b * f)
    o = torch.zeros(4, 8)
    mr.clip_grad_norm([a, b], 1.0, out=[o[:, :4], o[:, 4:]])   # one in the other's gaps
    f = 1 / math.sqrt(16 + 4 * 16)
    assert torch.allclose(o[:, :4], a * f) and torch.allclose(o[:, 4:], b * f)


def _arrays(tensors):
    n = len(tensors)
    return ((ctypes.c_void_p * n)(*(a for a, _, _ in tensors)), (ctypes.c_int64 * n)(*(c for _, c, _ in tensors)),
            (ctypes.c_int * n)(*(d for _, _, d in tensors)))


def test_c_abi_refusals():
    """Argument errors are found before any work is enqueued (the addresses are never read)."""
    lib, p, odd = _lib.load(), ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 8)
    need = lib.rr_grad_norm_workspace_bytes
    assert need(0) > 0 and need(-1) == 0 and need((1 << 24) + 1) == 0 and need(1) <= need(128) < need(129) < need(10 ** 6)

    def norm(tensors, **k):
        at, numel, types = _arrays(tensors)
        a = dict(count=len(tensors), at=at, numel=numel, types=types, norm=p, ws=p, n=1 << 30, s=None)
        return lib.rr_grad_norm(*{**a, **k}.values())

    def clip(tensors, out=None, **k):
        at, numel, types = _arrays(tensors)
        to = _arrays(tensors if out is None else [(a, c, d) for a, (_, c, d) in zip(out, tensors)])[0]
        a = dict(count=len(tensors), at=at, to=to, numel=numel, types=types, most=1.0, norm=p, ws=p, n=1 << 30, s=None)
        return lib.rr_clip_grad_norm(*{**a, **k}.values())

    good = [(4096, 10, 0), (8192, 7, 1)]
    for fn in (norm, clip):
        for bad in (dict(count=-1), dict(count=(1 << 24) + 1), dict(at=None), dict(numel=None), dict(types=None), dict(norm=None),
                    dict(ws=None)):
            assert fn(good, **bad) == _lib.RR_EINVAL, bad
        for bad in (dict(n=need(2) - 1), dict(ws=odd)):
            assert fn(good, **bad) == _lib.RR_EWORKSPACE, bad
        for bad in ((4096, 10, 3), (4096, -1, 0), (4096, 1 << 60, 0), (0, 10, 0), (4098, 10, 0), (4097, 10, 1)):
            assert fn([good[1], bad]) == _lib.RR_EINVAL, bad
        assert fn([(4096, 1 << 47, 0)]) == _lib.RR_EUNSUPPORTED
    for most in (-1.0, math.nan):
        assert clip(good, most=most) == _lib.RR_EINVAL
    assert clip(good, to=None) == _lib.RR_EINVAL
    shared = b"share memory", b"shares memory"
    for tensors, out in (([(4096, 10, 0), (4096, 10, 0)], None),            # the same twice
                         ([(4096, 10, 0), (4132, 10, 0)], None),            # the last value of one is the first of the other
                         ([(4096, 10, 1), (4114, 10, 1)], None),
                         ([(4096, 10, 0), (8192, 10, 0)], [16384, 16384]),
                         ([(4096, 10, 0), (8192, 10, 0)], [16384, 4132]),   # reaches into what the other reads
                         ([(4096, 10, 0), (8192, 10, 0)], [8192, 4096]),    # the other's
                         ([(4096, 10, 0)], [4100])):                        # itself, shifted
        assert clip(tensors, out) == _lib.RR_EINVAL and any(s in lib.rr_last_error() for s in shared), (tensors, out)
    assert clip([(4096, 10, 0)], [0]) == _lib.RR_EINVAL and clip([(4096, 10, 0)], [4098]) == _lib.RR_EINVAL


@pytest.mark.skipif(not SAN_LIB.exists(), reason="host-sanitizer build absent "
                    "(python mlx-recurrence_amd/build.py --host-sanitize)")
def test_host_code_under_asan_and_ubsan():
    env = dict(os.environ)
    env.update(LD_PRELOAD=str(_asan_runtime()), MLX_RECURRENCE_AMD_LIB=str(SAN_LIB),
               ASAN_OPTIONS="detect_leaks=0:abort_on_error=1", UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1")
    res = subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider", "tests/test_grad_norm_api.py", "-k",
                          "abi"], cwd=ROOT, env=env, capture_output=True, text=True, timeout=600)
    tail = (res.stdout + res.stderr)[-3000:]
    assert res.returncode == 0, tail
    assert "AddressSanitizer" not in tail and "runtime error" not in tail, tail
    assert " passed" in tail
