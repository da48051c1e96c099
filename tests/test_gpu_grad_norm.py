"""The norm of gradients and their clipping on the GPU against 64 bits.

Bounds, from the arithmetic: sums are in 64 bits, so the norm is off by its rounding to fp32, 2^-24 of
it, and the sum's own, n 2^-53 at most (n values: 2^31 here, 2^-22; below 2^27 values 2^-26).  A value is
g f rounded to the output's type once (16 bits: through fp32 first, 2^-24 of it more) with f off by
as little: half a step, 2^-24 fp32, 2^-8 bf16, 2^-11 fp16 of the value, or 2^-25 where fp16 has no
smaller step (2^-150 fp32, 2^-134 bf16)."""
from __future__ import annotations

import math

import pytest
import torch

import mlx_recurrence_amd as mr
from mlx_recurrence_amd import _lib
from tests import logp_oracle as orc

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
LEAST = {F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 2.0 ** -25}
DTYPES = [F32, BF16, F16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def tensors(shapes, dtype, seed=0, size=1.0):
    """dtype None: all three in turn."""
    g = gen(seed)
    return [(size * torch.randn(s, generator=g, device="cuda")).to(DTYPES[i % 3] if dtype is None else dtype)
            for i, s in enumerate(shapes)]


def norm64(grads):
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


def check(norm, got, grads, max_norm):
    """norm and scaled values against the gradients as they were."""
    n = norm64(grads)
    assert norm.dtype == F32 and norm.shape == ()
    if n > torch.finfo(F32).max:   # 1000 values of 1e37: 3.7e38, where fp32 ends at 3.4e38
        assert torch.isinf(norm)
    else:
        assert abs(float(norm) - n) <= (2.0 ** -24 + 2.0 ** -26) * n
    f = max_norm / n if n > max_norm else 1.0
    for a, g in zip(got, grads):
        want = g.double() * f
        off = (a.double() - want).abs()
        assert a.dtype == g.dtype and a.shape == g.shape
        assert bool((off <= want.abs() * (U[a.dtype] + 2.0 ** -23 * (a.dtype != F32) + 2.0 ** -40) + LEAST[a.dtype]).all())


SETS = [[(1,)], [(7,)], [()], [(2048,)], [(2047,), (2049,)], [(0,), (5,), (0, 3)], [(3, 5), (64, 33), (8191,), (1,), (2, 3, 4)],
        [(100_003,)], [(1000, 1001), (17,)], [(i % 97 + 1,) for i in range(128)], [(i * 37 % 501,) for i in range(129)],
        [(i * 91 % 3001 + 1,) for i in range(700)]]


@pytest.mark.parametrize("dtype", [F32, BF16, F16, None])
@pytest.mark.parametrize("shapes", SETS)
def test_norm_and_clipping(shapes, dtype):
    grads = tensors(shapes, dtype, seed=len(shapes))
    before = [g.clone() for g in grads]
    n = norm64(grads)
    most = 0.3 * n
    norm = mr.global_grad_norm(grads)
    assert abs(float(norm) - n) <= (2.0 ** -24 + 2.0 ** -26) * n and all(torch.equal(a, b) for a, b in zip(grads, before))
    out = [torch.full_like(g, 9.0) for g in grads]
    check(mr.clip_grad_norm(grads, most, out=out), out, before, most)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    # above the norm: copied as they are, or not touched
    assert torch.equal(mr.clip_grad_norm(grads, 2 * n + 1, out=out), norm)
    assert all(torch.equal(a, b) for a, b in zip(out, before))
    assert torch.equal(mr.clip_grad_norm(grads, math.inf), norm) and all(torch.equal(a, b) for a, b in zip(grads, before))
    again = [g.clone() for g in grads]
    check(mr.clip_grad_norm(grads, most), grads, before, most)
    mr.clip_grad_norm(again, most)   # the same bits
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    assert torch.equal(mr.clip_grad_norm(grads, 0.0) > 0, norm > 0) and not any(g.any() for g in grads)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,shift", [(0, 0), (1, 1), (3, 0), (0, 5), (7, 2)])
def test_pieces_of_a_buffer(dtype, offset, shift):
    """Views at any element; what lies around them stays as it was."""
    sizes = [1, 2, 9, 300, 2048, 4099, 20_000]
    total = sum(sizes) + 64 * len(sizes)
    flat, to = tensors([(total,), (total,)], dtype, seed=offset)
    at, ins, outs = offset, [], []
    for s in sizes:
        ins.append(flat[at:at + s])
        outs.append(to[at + shift:at + shift + s])
        at += s + 11
    keep, before, mask = to.clone(), [t.clone() for t in ins], torch.ones(total, dtype=torch.bool, device="cuda")
    n = norm64(ins)
    check(mr.clip_grad_norm(ins, 0.5 * n, out=outs), outs, before, 0.5 * n)
    for o in outs:
        mask[o.storage_offset():o.storage_offset() + o.numel()] = False
    assert torch.equal(to[mask], keep[mask])
    keep = flat.clone()
    check(mr.clip_grad_norm(ins, 0.5 * n), ins, before, 0.5 * n)
    mask[:] = True
    for t in ins:
        mask[t.storage_offset():t.storage_offset() + t.numel()] = False
    assert torch.equal(flat[mask], keep[mask])


@pytest.mark.parametrize("python", [False, True])
def test_layouts(python, monkeypatch):
    """Transposed tensors, tensors with gaps, and outputs laid out in another way."""
    if python:
        monkeypatch.setattr(_lib, "_autograd_mod", None)
    base = tensors([(40, 30), (40, 30), (6, 8, 10)], F32, seed=2)

    def views():
        a, b, c = (t.clone() for t in base)
        return [a.T, b[:, 3:20], c[..., ::3]], (a, b, c)

    grads, _ = views()
    before = [g.clone() for g in grads]
    n = norm64(before)
    assert abs(float(mr.global_grad_norm(grads)) - n) <= 2.0 ** -23 * n
    out = [torch.zeros(40, 30, device="cuda").T.contiguous(), torch.zeros(17, 40, device="cuda").T, torch.zeros(6, 8, 8, device="cuda")[..., ::2]]
    check(mr.clip_grad_norm(grads, 0.4 * n, out=out), out, before, 0.4 * n)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    grads, whole = views()
    check(mr.clip_grad_norm(grads, 0.4 * n), grads, before, 0.4 * n)
    assert torch.equal(whole[1][:, :3], base[1][:, :3]) and torch.equal(whole[2][..., 1], base[2][..., 1])
    versions = [t._version for t in grads]
    mr.clip_grad_norm(grads, 0.1)
    assert all(t._version > v for t, v in zip(grads, versions))


@pytest.mark.parametrize("python", [False, True])
def test_refusals(python, monkeypatch):
    if python:
        monkeypatch.setattr(_lib, "_autograd_mod", None)
    a, b = tensors([(10, 10), (10, 10)], F32)
    keep = a.clone()
    for grads, out in (([a, a], None), ([a, a.view(-1)[3:50]], None), ([a, b], [a, a]), ([a, b], [b, a]),
                       ([a[:, ::2], a[:, ::2]], None), ([a], [a.view(-1).roll(0)[:0].expand(10, 0)])):
        with pytest.raises(ValueError, match="share|shape"):
            mr.clip_grad_norm(grads, 1.0, out=out)
    with pytest.raises(ValueError, match="more than once"):
        mr.clip_grad_norm([a[:1].expand(10, 10)], 1.0)
    with pytest.raises(ValueError, match="shape and type"):
        mr.clip_grad_norm([a], 1.0, out=[b.half()])
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        mr.clip_grad_norm([a.double()], 1.0)
    with pytest.raises(TypeError, match="dense"):
        mr.clip_grad_norm([a.to_sparse()], 1.0)
    with pytest.raises(RuntimeError, match="one device|run on a ROCm GPU"):
        mr.clip_grad_norm([a, b.cpu()], 1.0)
    with pytest.raises(ValueError, match="not differentiable"):
        mr.global_grad_norm([a.clone().requires_grad_(True)])
    with torch.no_grad():
        mr.global_grad_norm([a.clone().requires_grad_(True)])
    assert torch.equal(a, keep)
    # shared memory is no matter where nothing is written
    assert abs(float(mr.global_grad_norm([a, a, a[:1].expand(10, 10)])) - norm64([a, a, a[:1].expand(10, 10)])) < 1e-4


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_values_of_the_whole_range(dtype):
    """Squares beyond fp32's range on either side, and a factor below its normal values."""
    for size in (1e-37, 1e-25, 1e25, 1e37):
        grads = tensors([(1000,), (333,)], dtype, seed=4, size=size)
        before = [g.clone() for g in grads]
        check(mr.clip_grad_norm(grads, 0.5 * norm64(before)), grads, before, 0.5 * norm64(before))
    grads = tensors([(4096,)], dtype, seed=5, size=1e38)
    grads[0].clamp_(-3e38, 3e38)
    before = [grads[0].clone()]
    norm = mr.clip_grad_norm(grads, 1e-3)
    assert torch.isinf(norm)   # above fp32's largest value; the values are scaled by the norm itself
    f = 1e-3 / norm64(before)
    off = (grads[0].double() - before[0].double() * f).abs()
    assert bool((off <= (U[dtype] + 2.0 ** -23) * before[0].double().abs() * f + LEAST[dtype]).all()) and grads[0].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_norm_that_is_not_finite_changes_nothing(dtype, bad):
    grads = tensors([(5000,), (33,)], dtype, seed=6)
    grads[1][7] = bad
    before = [g.clone() for g in grads]
    out = [torch.zeros_like(g) for g in grads]
    for norm in (mr.clip_grad_norm(grads, 0.1), mr.clip_grad_norm(grads, 0.1, out=out), mr.global_grad_norm(grads)):
        assert torch.isnan(norm) if math.isnan(bad) else torch.isinf(norm)
    for got in (grads, out):
        assert all(torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)) for a, b in zip(got, before))


def test_none_and_one_tensor():
    a, b = tensors([(100,), (50,)], F32, seed=7)
    n = norm64([a, b])
    assert float(mr.global_grad_norm([None, a, None, b])) == float(mr.global_grad_norm((t for t in (a, b))))
    out = [None, torch.zeros(100, device="cuda"), None, torch.zeros(50, device="cuda")]
    check(mr.clip_grad_norm([None, a, None, b], 0.5 * n, out=out), [out[1], out[3]], [a, b], 0.5 * n)
    keep = a.clone()
    check(mr.clip_grad_norm(a, 0.1), [a], [keep], 0.1)
    empty = torch.zeros(0, 4, device="cuda")
    assert float(mr.global_grad_norm([empty])) == 0 and float(mr.clip_grad_norm([empty], 1.0)) == 0
    zeros = torch.zeros(70, device="cuda", dtype=BF16)
    assert float(mr.clip_grad_norm([zeros], 0.0)) == 0 and not zeros.any()


def test_more_than_2_31_values():
    n = (1 << 31) + 4097
    t = torch.zeros(n, dtype=BF16, device="cuda")
    t[-5:] = 2.0
    t[1] = 4.0
    assert float(mr.clip_grad_norm([t], 3.0)) == 6.0
    assert t[-5:].tolist() == [1.0] * 5 and float(t[1]) == 2.0 and int((t != 0).sum()) == 6


def test_streams_and_replays():
    grads = tensors([(1000,), (64, 65), (7,)] + [(30,)] * 200, None, seed=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mine = [g.clone() for g in grads]
        norm = mr.clip_grad_norm(mine, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    check(norm, mine, grads, 1.0)
    static = [g.clone() for g in grads]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = mr.clip_grad_norm(static, 1.0)
    for seed in range(3):
        new = tensors([tuple(g.shape) for g in grads], None, seed=20 + seed, size=10.0 ** (seed - 2))
        for s, g in zip(static, new):
            s.copy_(g)
        graph.replay()
        eager = [g.clone() for g in new]
        want = mr.clip_grad_norm(eager, 1.0)
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(static, eager))
        check(norm, static, new, 1.0)


def test_a_step_of_the_policy_and_the_pairs():
    """The losses' gradients clipped as a training step does, against the same in 64 bits."""
    g = gen(9)
    w = (torch.randn(300, 64, generator=g, device="cuda") / 4).requires_grad_(True)
    h = torch.randn(3, 2, 10, 64, generator=g, device="cuda").requires_grad_(True)
    labels = torch.randint(0, 300, (3, 2, 10), generator=g, device="cuda")
    labels[..., :3] = -100
    with torch.no_grad():
        ref = mr.linear_log_probs(h, w, labels)
    A = torch.randn(3, 2, 1, generator=g, device="cuda")
    loss = mr.linear_policy_loss(h, w, labels, A, ref, ref, kl_weight=0.1) + \
        mr.linear_preference_loss(h, w, labels, ref.sum(-1))
    loss.backward()
    up = torch.ones((), device="cuda")
    a = orc.policy(h, w, labels, A, ref, ref, up, kl=0.1)
    b = orc.preference(h, w, labels, ref.sum(-1), up)
    dh, dw = a[1] + b[1], a[2] + b[2]
    n = math.sqrt(float(dh.square().sum() + dw.square().sum()))
    norm = mr.clip_grad_norm([h.grad, w.grad], 0.5 * n)
    # fp32 gradients are good to 4e-6 times 1 + |logp| (below 20)
    assert abs(float(norm) / n - 1) < 1e-4
    for got, want in ((h.grad, dh), (w.grad, dw)):
        assert float((got.double() - 0.5 * want).norm() / (0.5 * want).norm()) < 2e-4


@pytest.mark.parametrize("python", [False, True])
def test_empty_tensors_of_another_layout(python, monkeypatch):
    """They have no memory to share, and no values to be there twice."""
    if python:
        monkeypatch.setattr(_lib, "_autograd_mod", None)
    def zeros(*shape):
        return torch.zeros(shape, device="cuda")
    grads = [zeros(0, 3), zeros(0, 3), torch.full((4,), 2.0, device="cuda"), zeros(0, 3)]
    out = [zeros(3, 0).T, zeros(3, 0).T, zeros(4), zeros(0, 1).expand(0, 3)]
    assert float(mr.clip_grad_norm(grads, 1.0, out=out)) == 4.0 and torch.equal(out[2], torch.full((4,), 0.5, device="cuda"))
    assert float(mr.clip_grad_norm([zeros(0, 1).expand(0, 3), zeros(3, 0).T], 1.0)) == 0.0


@pytest.mark.parametrize("python", [False, True])
def test_out_that_needs_a_gradient(python, monkeypatch):
    """What is written has no place in a graph: its gradient would be that of the values before."""
    if python:
        monkeypatch.setattr(_lib, "_autograd_mod", None)
    g, leaf = torch.full((5,), 3.0, device="cuda"), torch.zeros(5, device="cuda", requires_grad=True)
    for o in (leaf, leaf * 2, (leaf * 2)[:]):
        with pytest.raises(ValueError, match="out must not need a gradient"):
            mr.clip_grad_norm([g], 1.0, out=[o])
    assert not leaf.detach().any()
    with torch.no_grad():
        mr.clip_grad_norm([g], math.inf, out=[leaf])
    assert torch.equal(leaf.detach(), g)


@pytest.mark.parametrize("python", [False, True])
def test_inference_mode(python, monkeypatch):
    if python:
        monkeypatch.setattr(_lib, "_autograd_mod", None)
    with torch.inference_mode():
        t = torch.full((100,), 3.0, device="cuda")
        assert float(mr.clip_grad_norm([t], 15.0)) == 30.0 and t.tolist() == [1.5] * 100
    assert float(mr.global_grad_norm([t])) == 15.0
    with pytest.raises(ValueError, match="inference mode"):
        mr.clip_grad_norm([t], 1.0)
    assert t.tolist() == [1.5] * 100
    a = torch.full((100,), 3.0, device="cuda")
    assert float(mr.clip_grad_norm([t], 1.0, out=[a])) == 15.0 and abs(float(a.norm()) - 1) < 1e-6


def test_python_binding_gives_the_same(monkeypatch):
    grads = tensors([(1000,), (64, 65), (7,)] + [(30,)] * 200, None, seed=12)
    first, second = ([g.clone() for g in grads] for _ in range(2))
    a = mr.clip_grad_norm(first, 1.0)
    monkeypatch.setattr(_lib, "_autograd_mod", None)
    assert torch.equal(a, mr.clip_grad_norm(second, 1.0)) and all(torch.equal(x, y) for x, y in zip(first, second))
    assert torch.equal(a, mr.global_grad_norm(grads))


def test_workspace_is_written_inside(monkeypatch):
    buffers = []

    def guarded(n, device):
        whole = torch.full((n + 8192,), 0xA5, dtype=torch.uint8, device=device)
        whole[4096:4096 + n] = 0xFF
        buffers.append((whole, n))
        return whole[4096:4096 + n]

    monkeypatch.setattr(_lib, "_autograd_mod", None)
    monkeypatch.setattr(_lib, "_alloc_ws", guarded)
    for shapes in ([(1,)], [(i * 91 % 3001 + 1,) for i in range(700)], [(20_000_000,), (5,), (3_000_001,)]):
        grads = tensors(shapes, BF16, seed=13)
        before = [g.clone() for g in grads]
        check(mr.clip_grad_norm(grads, 0.5 * norm64(before)), grads, before, 0.5 * norm64(before))
    for whole, n in buffers:
        assert (whole[:4096] == 0xA5).all() and (whole[4096 + n:] == 0xA5).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_more_than_the_cache(dtype):
    """Sizes whose first part is read past the cache, and whose second reading is."""
    n = 90_000_001 if dtype == F32 else 180_000_001
    g = gen(14)
    grads = [torch.randn(n, generator=g, device="cuda").to(dtype), torch.randn(777, generator=g, device="cuda").to(BF16)]
    out = [torch.empty_like(t) for t in grads]
    n64 = norm64(grads)
    norm = mr.clip_grad_norm(grads, 0.25 * n64, out=out)
    assert abs(float(norm) / n64 - 1) <= 2.0 ** -23
    for a, t in zip(out, grads):
        off = (a.double() - t.double() * 0.25).abs()
        assert bool((off <= t.double().abs() * 0.25 * (U[a.dtype] + 2.0 ** -23) + LEAST[a.dtype]).all())


@pytest.mark.parametrize("python", [False, True])
def test_outputs_of_another_layout_share_no_memory(python, monkeypatch):
    """Outputs that are copied to are checked too, together with those written directly."""
    if python:
        monkeypatch.setattr(_lib, "_autograd_mod", None)
        monkeypatch.setattr(_lib, "autograd_ext", lambda: None)
    a, b, o = (torch.zeros(s, device="cuda") for s in ((4, 4), (4, 4), (8, 4)))
    a, b = a + 1, (b + 2).T
    for grads, out in (([a, b], [o[:4], o[:4]]), ([a, b], [o[:4], o[1:5]]), ([b, a], [o[1:5], o[:4]]), ([b, b], [o[:4], o[2:6]]),
                       ([a, b], [o[:4], o[1:5].T]), ([a, b[:2]], [o[:4], o[:4:2]]), ([b[:2], b[:2]], [o[:4:2], o[:4:2]])):
        with pytest.raises(ValueError, match="share memory"):
            mr.clip_grad_norm(grads, 1.0, out=out)
    assert not o.any()
    keep = [a.clone(), b.clone()]
    check(mr.clip_grad_norm([a, b], 1.0, out=[o[:4], o[4:]]), [o[:4], o[4:]], keep, 1.0)   # one behind the other
    o = torch.zeros(4, 8, device="cuda")
    check(mr.clip_grad_norm([a, b], 1.0, out=[o[:, :4], o[:, 4:]]), [o[:, :4], o[:, 4:]], keep, 1.0)   # in the other's gaps
    m = torch.ones(4, 8, device="cuda")
    check(mr.clip_grad_norm([m[:, :4], m[:, 4:]], 1.0), [m[:, :4], m[:, 4:]], [torch.ones(4, 4, device="cuda")] * 2, 1.0)
