"""The global norm of many gradients and clipping by it on the HIP kernels (csrc/grad_norm.hip): what a training step
does between its backward and its optimizer.  The reference trains without clipping (train_fineweb.py:161-179).

Tensors are float32 or bfloat16, mixed as they come, on one GPU.  Squares are added in 64 bits, so that no gradient is
too large or too small for the norm, in a fixed order; nothing waits for the host.  None has a gradient of its own:
clip_grad_norm_ runs without autograd, as torch's, the others refuse a tensor that needs one.
"""
from __future__ import annotations

import math

import torch

from . import _ops

__all__ = ["grad_norm", "clip_grads_", "clip_grad_norm_"]

_NORM_2, _NORM_MAX = 0, 1  # HDCM_NORM_2, HDCM_NORM_MAX


def grad_norm(tensors, norm_type=2.0):
    """The norm of all elements of a list of tensors together, as a float32 number on their GPU: ``norm_type`` 2, or
    math.inf for the largest magnitude (a NaN gives NaN in both).  A tensor given twice counts twice."""
    tensors = _listed(tensors)
    kind = _kind(norm_type)
    return _ops.native().grad_norm(tensors, kind) if tensors else torch.zeros(())


def clip_grads_(tensors, max_norm, total_norm):
    """Scale tensors in place by min(1, max_norm / (total_norm + 1e-6)), each product rounded to its tensor's type;
    nothing is written where the factor is 1.  ``total_norm`` is a number, or a tensor of one on their GPU (the norm over
    several ranks).  A norm that is NaN makes all elements NaN, an infinite one 0 (infinite elements NaN).  Tensors with
    gaps in memory and tensors that overlap are refused."""
    tensors, max_norm = _listed(tensors), _limit(max_norm)
    if not tensors:
        return
    if not isinstance(total_norm, torch.Tensor):
        total_norm = torch.full((), total_norm, dtype=torch.float32, device=tensors[0].device)
    _ops.native().clip_grads(tensors, max_norm, total_norm)


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_ on these kernels: clip_grads_ on the gradients of ``parameters`` (an iterable, or
    one) by their own grad_norm, which is returned.  A parameter given twice counts once.  ``error_if_nonfinite`` waits
    for the norm, and raises with the gradients as they were where it is not finite."""
    parameters, kind, max_norm = _listed(parameters), _kind(norm_type), _limit(max_norm)
    if error_if_nonfinite:
        grads = [p.grad for p in {id(p): p for p in parameters}.values() if p.grad is not None]
        if grads and grads[0].is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("error_if_nonfinite waits for the norm, which a recording cannot")
        with torch.no_grad():
            norm = grad_norm(grads, norm_type).item()
        if not math.isfinite(norm):
            raise RuntimeError(f"the gradients' norm is {norm}, not finite: they are not clipped")
    norm = _ops.native().clip_grad_norm(parameters, max_norm, kind)
    return torch.zeros(()) if norm is None else norm


def _listed(tensors):
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def _kind(norm_type):
    p = float(norm_type)
    if p not in (2.0, math.inf):
        raise ValueError(f"norm_type must be 2 or math.inf, got {norm_type}")
    return _NORM_2 if p == 2.0 else _NORM_MAX


def _limit(max_norm):
    limit = float(max_norm)
    if not limit >= 0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    return limit
