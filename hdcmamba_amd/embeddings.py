"""Token rows of an embedding and the weight's gradient on the HIP kernels (csrc/embedding.hip): the first kernel of
an HdcMambaLM's forward and the last of its backward.  The reference's model uses nn.Embedding
(train_fineweb.py:49,87).

An id outside 0..V-1 (a padding id -1, an ignored position) gives a row of zeros and no gradient.
"""
from __future__ import annotations

import torch
import torch.nn as nn
from torch.autograd import forward_ad

from . import _ops
from .quant4 import carries_tangent

__all__ = ["embedding", "embedding_grad", "Embedding"]


def embedding(ids, weight, scale=1.0, padding_idx=None):
    """scale * weight[ids] in fp32, rounded to weight's type: ids of any shape (int64 or int32), weight [V, D] (float32 or bfloat16) ->
    [*ids.shape, D] of weight's type, differentiable in weight (and again in the gradient).  The rows of ``padding_idx``
    (counted from the end where negative) are looked up as others are but give no gradient."""
    if padding_idx is not None:
        padding_idx = _padding(padding_idx, weight.shape[0])
    return _ops.native().embedding(ids, weight, scale, padding_idx)


def embedding_grad(ids, grad, num_embeddings, scale=1.0, padding_idx=None, out=None, accumulate=False):
    """The gradient of ``embedding`` for its weight: row v is scale * the sum of grad's rows [*ids.shape, D] at the ids v,
    summed and scaled in fp32, rounded to grad's type -> [num_embeddings, D].  The ids and the call's sizes and types fix the
    order of every sum: the same call gives the same bits.

    ``out`` ([num_embeddings, D], float32 or bfloat16, contiguous rows) is written instead; with ``accumulate`` the sums
    are added to it, and rows without an id are not touched."""
    if padding_idx is not None:
        padding_idx = _padding(padding_idx, num_embeddings)
    if accumulate and out is None:
        raise RuntimeError("embedding_grad: accumulate needs out")
    if out is not None and ((torch.is_grad_enabled() and (grad.requires_grad or out.requires_grad))
                            or carries_tangent(grad) or carries_tangent(out)):
        raise RuntimeError("embedding_grad with out has no gradient and no tangent: call it under torch.no_grad() or on detached tensors")
    return _ops.native().embedding_grad(ids, grad, num_embeddings, scale, padding_idx, out, accumulate)


def _padding(index, rows):
    if not -rows <= index < rows:
        raise ValueError(f"padding_idx {index} is not one of {rows} tokens")
    return index % rows


def _within(lookup, ids, weight):
    """lookup(ids), with zeros for ids outside 0..V-1: PyTorch's own kernels read wherever such an id points (their
    assertions are compiled out on ROCm)."""
    V = weight.shape[0]
    if V == 0:
        return weight.new_zeros(*ids.shape, weight.shape[1])
    return lookup(ids.clamp(0, V - 1)).masked_fill(((ids < 0) | (ids >= V)).unsqueeze(-1), 0)


_PLAIN = (torch.Tensor, nn.Parameter)


def _traced():
    """Whether PyTorch's operations are looked at rather than only run (a compiler or a tracer, a mode with a __torch_dispatch__),
    which the kernels' calls would pass by."""
    return torch.compiler.is_compiling() or torch._C._len_torch_dispatch_stack() > 0 or torch.jit.is_tracing()


class Embedding(nn.Embedding):
    """nn.Embedding on these kernels, its rows times ``scale``: the same constructor, parameters and initial values.

    What the kernels do not take goes through nn.Embedding's own forward: weights on the CPU or of other types, max_norm,
    sparse and scale_grad_by_freq, forward-mode differentiation and torch.func's transforms (vmap), tracing and compiling,
    dispatch modes, and tensors of a class of their own (sharded, quantized, fake).  On a GPU an id outside 0..V-1 is a row
    of zeros without a gradient there too (max_norm, and the frequencies and rows of a sparse gradient, count it as the
    nearest token); on the CPU nn.Embedding refuses it, and a tensor's class does what it does."""

    def __init__(self, *args, scale=1.0, **kwargs):
        super().__init__(*args, **kwargs)
        self.scale = float(scale)

    def forward(self, ids):
        w = self.weight
        if type(w) not in _PLAIN or type(ids) is not torch.Tensor:
            y = super().forward(ids)
            return y if self.scale == 1.0 else y * self.scale
        if (not w.is_cuda or w.dtype not in _ops._DTYPES or self.max_norm is not None or self.sparse or _traced()
                or self.scale_grad_by_freq or forward_ad._current_level >= 0
                or torch._C._functorch.maybe_current_level() is not None):
            y = _within(super().forward, ids, w) if w.is_cuda else super().forward(ids)
            return y if self.scale == 1.0 else y * self.scale
        return embedding(ids, w, self.scale, self.padding_idx)

    def extra_repr(self):
        return super().extra_repr() + (f", scale={self.scale}" if self.scale != 1.0 else "")
