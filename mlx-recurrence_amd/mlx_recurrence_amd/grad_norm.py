"""grad_norm.py — the norm of a step's gradients taken together, and their clipping by it (no
counterpart in the reference, which has the scans alone).

    global_grad_norm(grads)                          -> norm
    clip_grad_norm(grads, max_norm)                  -> norm, grads scaled in place
    global_grad_norm_reference, clip_grad_norm_reference      (plain torch)

Any number of tensors of any sizes and of the three input types together, in two launches for
each 128 of them; nothing waits for the device.
"""
from __future__ import annotations

import math

import torch

from . import _lib


def _dense(t):
    """Whether the values lie in memory without gaps, in any order of the axes."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != want:
            return False
        want *= size
    return True


def _check_written(written):
    """What is written to must not be another's.  The library sees the copies in place of tensors that are copied
    to, so all are looked at here: the whole of a tensor without gaps, the first value of one with gaps."""
    ranges = sorted((t.data_ptr(), t.data_ptr() + t.element_size() * (t.numel() if _dense(t) else 1))
                    for t in written if t.numel())
    if any(b[0] < a[1] for a, b in zip(ranges, ranges[1:])):
        raise ValueError("two of the tensors to write share memory")


def _run(grads, outs, clip, max_norm):
    """The C++ module's grad_norm for where it is not built."""
    if outs is not None:
        outs = [o for g, o in zip(grads, outs) if g is not None]
        if not all(isinstance(o, torch.Tensor) for o in outs):
            raise ValueError("out must have a tensor of each gradient's shape and type")
    grads = [g for g in grads if g is not None]
    if not all(isinstance(g, torch.Tensor) for g in grads):
        raise TypeError("gradients must be tensors or None")
    if not grads:
        raise ValueError("no gradients to take a norm of")
    for i, g in enumerate(grads):
        if g.layout != torch.strided:
            raise TypeError("gradients must be dense tensors")
        if torch.is_grad_enabled() and g.requires_grad:
            raise ValueError("the norm of gradients is not differentiable; call it under torch.no_grad()")
        if g.dtype not in _lib.DTYPE_CODE:
            raise TypeError("gradients must be float32, bfloat16 or float16")
        if clip and (outs[i] if outs else g).is_inference() and not torch.is_inference_mode_enabled():
            raise ValueError("a tensor to write was made in inference mode; call it there")
        if outs and (outs[i].layout != torch.strided or outs[i].shape != g.shape or outs[i].dtype != g.dtype):
            raise ValueError("out must have a tensor of each gradient's shape and type")
        if outs and torch.is_grad_enabled() and outs[i].requires_grad:
            raise ValueError("out must not need a gradient; call it under torch.no_grad()")
    dev = _lib.require_device(*grads, *(outs or ()))
    with _lib.device_guard(dev), torch.no_grad():
        src = [g if _dense(g) else g.contiguous() for g in grads]
        norm = torch.empty((), dtype=torch.float32, device=dev)
        if not clip:
            _lib.grad_norm(src, None, 0.0, norm)
            return norm
        written = outs or grads
        to, back = [], []
        for o, s in zip(written, src):
            if s.numel() == 0 or (_dense(o) and o.stride() == s.stride()):
                to.append(o)
                continue
            if any(st == 0 and sz > 1 for st, sz in zip(o.stride(), o.shape)):
                raise ValueError("a tensor to write has its values more than once")
            to.append(torch.empty_like(s) if outs else s)
            back.append((o, to[-1]))
        if back:
            _check_written(written)
        _lib.grad_norm(src, to, max_norm, norm)
        for o, t in back:
            o.copy_(t)
        torch.autograd.graph.increment_version([t for t in written if not t.is_inference()])
    return norm


def _listed(tensors):
    return tensors if isinstance(tensors, list) else [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def _tensors(grads):
    grads = [g for g in _listed(grads) if g is not None]
    if not grads:
        raise ValueError("no gradients to take a norm of")
    return grads


def global_grad_norm(grads):
    """The 2-norm of all values of `grads` together, on the GPU.

    Args:
        grads:  tensors of any shapes and of the three input types, on one device (or one
                tensor); entries that are None, of parameters without a gradient, are left out.

    Returns:
        norm:   fp32 scalar on the device.  Sums are in 64 bits, in a fixed order.
    """
    ext = _lib.autograd_ext()
    return (_run if ext is None else ext.grad_norm)(_listed(grads), None, False, 0.0)


def clip_grad_norm(grads, max_norm, *, out=None):
    """Scale `grads` in place so that their norm, taken together, is at most `max_norm`, on the GPU.

    ``g *= max_norm / norm`` where ``norm > max_norm``; otherwise they are not touched.  One value
    that is infinite or NaN leaves them all as they are: the caller sees it in what is returned.

    Args:
        grads:     as for global_grad_norm.  No two may share memory, which is checked (of those
                   with gaps between their values, the first value's place).
        max_norm:  the largest norm, 0 or more (math.inf: take the norm alone).
        out:       tensors of the same shapes and types to write to, in place of `grads` (each
                   a tensor of its own, or the gradient itself).

    Returns:
        norm:      before the clipping, as global_grad_norm's.  Not differentiable.
    """
    if not float(max_norm) >= 0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    grads, outs = _listed(grads), None if out is None else _listed(out)
    if outs is not None and len(grads) != len(outs):
        raise ValueError(f"out must have a tensor for each gradient, got {len(outs)} for {len(grads)}")
    ext = _lib.autograd_ext()
    return (_run if ext is None else ext.grad_norm)(grads, outs, True, float(max_norm))


# ------------------------------------------------------------------ plain forms
def global_grad_norm_reference(grads):
    """global_grad_norm as plain torch ops in 64 bits.  Runs on any device."""
    return torch.stack([g.detach().double().square().sum() for g in _tensors(grads)]).sum().sqrt().float()


def clip_grad_norm_reference(grads, max_norm):
    """clip_grad_norm as plain torch ops in 64 bits: (norm, scaled copies).  Runs on any device."""
    grads = _tensors(grads)
    norm = torch.stack([g.detach().double().square().sum() for g in grads]).sum().sqrt()
    factor = torch.where((norm > max_norm) & (norm < math.inf), max_norm / norm, 1.0)
    return norm.float(), [(g.detach().double() * factor).float().to(g.dtype) for g in grads]
