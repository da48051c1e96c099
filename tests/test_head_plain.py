"""The plain forms of the output head's losses at the edges of their inputs (CPU)."""
import math

import pytest
import torch

import mlx_recurrence_amd as mr


def _inputs():
    g = torch.Generator().manual_seed(3)
    return torch.randn(4, 6, generator=g), torch.randn(11, 6, generator=g), torch.tensor([[1, 2, 3]] * 4)


@pytest.mark.parametrize("tau", [0.25, 1.0, 3.0])
def test_equal_logits_of_any_size_are_an_even_split(tau):
    h, w, ids = _inputs()
    want = mr.linear_distillation_reference(h, w, torch.zeros(4, 3), ids, temperature=tau)
    for value in (torch.finfo(torch.float32).min, torch.finfo(torch.float32).max):
        assert torch.equal(mr.linear_distillation_reference(h, w, torch.full((4, 3), value), ids, temperature=tau), want)


def test_entries_of_no_weight_and_absent_ones():
    h, w, ids = _inputs()
    t = torch.tensor([[0.5, -1.0, -math.inf]] * 4)
    h.requires_grad_(True)
    want = mr.linear_distillation_reference(h, w, t, ids.masked_fill(t == -math.inf, -1))
    for logits, at in ((t, ids.masked_fill(t == -math.inf, 11)),
                       (t.masked_fill(t == -math.inf, torch.finfo(torch.float32).min), ids)):
        got = mr.linear_distillation_reference(h, w, logits, at)
        assert torch.equal(got, want)
        assert bool(torch.isfinite(torch.autograd.grad(got, h)[0]).all())
