"""Layer norm on the GPU beyond the sizes of test_gpu_head.py."""
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


def test_more_rows_than_a_grid_has_waves():
    """2^26 rows and a few more of one piece each: their waves would be 2^32 threads.  Every row against 64 bits, a
    slice at a time: |y| <= 3, rounded to 8 bits (2^-8 |y| at most) from fp32 sums that are some 2^-20 off."""
    rows, D = (1 << 26) + 3, 8
    x = torch.empty(rows, D, dtype=BF16, device="cuda")
    for part in x.split(1 << 23):
        part.normal_(generator=gen(len(part)))
    y = mr.layer_norm(x, eps=1e-3)
    for a, b in zip(x.split(1 << 22), y.split(1 << 22)):
        want = orc.layer_norm(a, None, None, 1e-3)
        assert float((b.double() - want).abs().max()) <= 3.0 * 2.0 ** -8 + 2.0 ** -18


def test_gradients_of_several_launches_of_rows():
    """More rows than a launch of the forward takes (2^23): the statistics of each reach the backward."""
    rows, D = (1 << 23) + 5, 8
    g = gen(2)
    x = randn(g, rows, D).requires_grad_(True)
    w = (1 + 0.3 * randn(g, D)).requires_grad_(True)
    dy = randn(g, rows, D)
    y = mr.layer_norm(x, w, eps=1e-2)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    wy, wx, ww, _ = orc.layer_norm(x.detach(), w.detach(), None, 1e-2, dy)
    # every value is a few fp32 operations on numbers below 10 (dx: times rstd <= 10); dw sums 2^23 terms of size 1 in
    # partial sums of a few thousand: a walk of 2^11.5 steps of 2^-24 of sums of up to 2^11.5
    for a, b, most in ((y, wy, 2e-5), (dx, wx, 2e-4), (dw, ww, 2e-1)):
        assert float((a.detach().double() - b).abs().max()) <= most
