"""The losses' logits between forward and backward (GPU): kept, or with keep_logits=False formed again."""
from __future__ import annotations

import pytest
import torch

import mlx_recurrence_amd as mr
from mlx_recurrence_amd import _lib
from tests import head_oracle as orc
from tests.test_gpu_head import check_all, head_inputs, teacher

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,D,V", [(3, 64, 300), (256, 512, 777), (257, 1000, 1300), (700, 1030, 4099), (3001, 200, 641)])
def test_gradients_with_and_without_kept_logits(rows, D, V, dtype):
    """Few rows, sums in parts, many rows; several tiles and ragged ends: the same loss, gradients to the same bounds."""
    g, h, w, labels = head_inputs(rows, D, V, dtype, rows + D)
    labels[1::7] = -100
    t, ids = teacher(g, rows, 6, V, labels.clamp(min=0))
    up = torch.rand(rows, generator=g, device="cuda") + 0.1
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    ce = dict(z_loss=1e-3, reduction="none")
    wants = (orc.cross_entropy(h.detach(), w.detach(), labels, up, zl=1e-3, reduction="none"),
             orc.distillation(h.detach(), w.detach(), t, ids, up, tau=2.0, reduction="none"))
    for want, loss in zip(wants, (lambda keep: mr.linear_cross_entropy(h, w, labels, keep_logits=keep, **ce),
                                  lambda keep: mr.linear_distillation(h, w, t, ids, temperature=2.0, reduction="none",
                                                                      keep_logits=keep))):
        kept, formed = loss(True), loss(False)
        assert torch.equal(kept, formed)
        with torch.no_grad():
            assert torch.equal(loss(True), kept)
        for out in (kept, formed):
            check_all((out.detach(), *torch.autograd.grad(out, (h, w), up)), want)


def test_both_bindings_keep_the_same(monkeypatch):
    g, h, w, labels = head_inputs(600, 1000, 3000, BF16, 5)
    h, w = h.requires_grad_(True), w.requires_grad_(True)

    def run():
        loss = mr.linear_cross_entropy(h, w, labels, keep_logits=False)
        return (loss.detach(), *torch.autograd.grad(loss, (h, w)))

    cpp = run()
    monkeypatch.setattr(_lib, "autograd_ext", lambda: None)
    for a, b in zip(cpp, run()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_memory_between_forward_and_backward(dtype):
    """4096 x 65536 logits are 1 GiB: with keep_logits=False the call never holds as much in all, and between forward
    and backward a copy of the hidden states and a few numbers a row."""
    rows, D, V = 4096, 1024, 65536
    _, h, w, labels = head_inputs(rows, D, V, dtype, 9)
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    logits, state = rows * V * 4, h.numel() * h.element_size() + rows * 64 + (1 << 20)
    for keep in (True, False):
        torch.cuda.empty_cache()
        torch.cuda.synchronize()
        start = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        loss = mr.linear_cross_entropy(h, w, labels, keep_logits=keep)
        held = torch.cuda.memory_allocated() - start
        assert held <= state + (logits if keep else 0) and (held >= logits) == keep
        grads = torch.autograd.grad(loss, (h, w))
        assert (torch.cuda.max_memory_allocated() - start < logits + w.numel() * w.element_size()) == (not keep)
        del grads, loss
    with torch.no_grad():
        torch.cuda.reset_peak_memory_stats()
        start = torch.cuda.memory_allocated()
        mr.linear_cross_entropy(h, w, labels)
        assert torch.cuda.max_memory_allocated() - start < logits // 8
