"""What the output head's gradients do not offer (GPU): forward-mode and second derivatives are refused, by both
bindings, never left out in silence."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwad

import mlx_recurrence_amd as mr
from mlx_recurrence_amd import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["cpp", "python"])
def binding(request, monkeypatch):
    assert _lib.autograd_ext() is not None
    if request.param == "python":
        monkeypatch.setattr(_lib, "autograd_ext", lambda: None)


def tensors():
    g = torch.Generator(device="cuda").manual_seed(1)
    return [torch.randn(s, generator=g, device="cuda") for s in ((12, 16), (16,), (16,), (30, 16))]


LABELS = list(range(12))


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("grad", [True, False])
def test_layer_norm_refuses_forward_mode(which, grad, binding):
    args = tensors()[:3]
    with fwad.dual_level(), torch.set_grad_enabled(grad):
        args[which] = fwad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="jvp"):
            mr.layer_norm(*args)


@pytest.mark.parametrize("which", [0, 1])
def test_losses_refuse_forward_mode(which, binding):
    x, _, _, w = tensors()
    labels = torch.tensor(LABELS, device="cuda")
    with fwad.dual_level():
        args = [x, w]
        args[which] = fwad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="jvp"):
            mr.linear_cross_entropy(*args, labels)
        with pytest.raises(RuntimeError, match="jvp"):
            mr.linear_distillation(*args, x[:, :4], labels[:, None].repeat(1, 4))


@pytest.mark.parametrize("op", ["norm", "ce", "kd"])
def test_second_derivatives_are_refused(op, binding):
    x, s, b, w = (t.requires_grad_(True) for t in tensors())
    labels = torch.tensor(LABELS, device="cuda")
    if op == "norm":
        leaves, out = (x, s, b), mr.layer_norm(x, s, b).sin().sum()
    elif op == "ce":
        leaves, out = (x, w), mr.linear_cross_entropy(x, w, labels)
    else:
        leaves, out = (x, w), mr.linear_distillation(x, w, x[:, :4], labels[:, None].repeat(1, 4))
    with pytest.raises(RuntimeError, match="no second derivatives"):
        torch.autograd.grad(out, leaves, create_graph=True)
    first = torch.autograd.grad(out, leaves, retain_graph=True)
    assert all(bool(torch.isfinite(a).all()) and a.grad_fn is None for a in first)


@pytest.mark.parametrize("reentrant", [False, True])
def test_under_checkpointing(reentrant, binding):
    """Recomputed forwards run with gradients on inside a backward: that is no second derivative."""
    from torch.utils.checkpoint import checkpoint
    x, s, b, w = (t.requires_grad_(True) for t in tensors())
    labels = torch.tensor(LABELS, device="cuda")

    def f(x, s, b, w):
        return mr.linear_cross_entropy(mr.layer_norm(x, s, b), w, labels)

    want = torch.autograd.grad(f(x, s, b, w), (x, s, b, w))
    checkpoint(f, x, s, b, w, use_reentrant=reentrant).backward()
    for leaf, e in zip((x, s, b, w), want):
        assert torch.equal(leaf.grad, e)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_graph_replays_of_losses_a_row(dtype):
    """reduction="none" and logits that are formed again, captured in a HIP graph: every replay gives the eager bits."""
    g = torch.Generator(device="cuda").manual_seed(4)
    h, w = (torch.randn(s, generator=g, device="cuda").to(dtype).requires_grad_(True) for s in ((300, 72), (1000, 72)))
    labels = torch.randint(0, 1000, (300,), generator=g, device="cuda")
    labels[::6] = -100
    up = torch.logspace(2, -4, 300, device="cuda")

    def step():
        loss = mr.linear_cross_entropy(h, w, labels, reduction="none", keep_logits=False)
        return (loss, *torch.autograd.grad(loss, (h, w), up))

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
