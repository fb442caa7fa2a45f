"""Calls of Embedding and its gradient that end before any kernel runs: tensors of other classes, modes, refusals."""
import pytest
import torch
import torch.nn as nn
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.utils._python_dispatch import TorchDispatchMode

import hdcmamba_amd as hm


class Held(torch.Tensor):
    """A wrapper that says it is on a GPU and computes on a CPU tensor which it holds."""

    @staticmethod
    def __new__(cls, data):
        return torch.Tensor._make_wrapper_subclass(cls, data.shape, dtype=data.dtype, device="cuda", requires_grad=data.requires_grad)

    def __init__(self, data):
        self.data_held = data.detach()

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        take = lambda x: x.data_held if isinstance(x, Held) else x  # noqa: E731
        out = func(*[take(a) for a in args], **{k: take(v) for k, v in (kwargs or {}).items() if k != "device"})
        return Held(out) if isinstance(out, torch.Tensor) else out


# without gradients: autograd asks a GPU's driver for streams, and there is none here
@pytest.mark.parametrize("scale", [1.0, 3.0])
@torch.no_grad()
def test_tensors_of_another_class_go_to_nn_embedding(scale):
    w = torch.randn(9, 4)
    ids = torch.tensor([[1, 8], [0, 1]])
    m = hm.Embedding(9, 4, _weight=w, scale=scale)
    m.weight = nn.Parameter(Held(w))
    assert m.weight.is_cuda and type(m.weight) is Held
    y = m(ids)
    assert type(y) is Held and torch.equal(y.data_held, w[ids] * scale)
    y = torch.func.functional_call(m, {"weight": Held(w)}, (Held(ids),))
    assert type(y) is Held and torch.equal(y.data_held, w[ids] * scale)


@torch.no_grad()
def test_fake_tensors():
    with FakeTensorMode():
        m = hm.Embedding(9, 4, device="cuda", dtype=torch.bfloat16, scale=2.0)
        ids = torch.zeros(3, 5, dtype=torch.long, device="cuda")
        y = m(ids)
    assert y.shape == (3, 5, 4) and y.dtype == torch.bfloat16 and y.is_cuda


def test_a_mode_sees_the_lookup():
    class Seen(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(func.overloadpacket.__name__)
            return func(*args, **(kwargs or {}))

    m = hm.Embedding(9, 4)
    with Seen() as seen:
        m(torch.tensor([1, 2]))
    assert "embedding" in seen.names


def test_traced_and_compiled_on_the_cpu():
    m = hm.Embedding(9, 4, scale=2.0)
    ids, other = torch.tensor([1, 2, 3]), torch.tensor([8, 0, 5])
    traced = torch.jit.trace(m, (ids,))
    assert torch.equal(traced(other), m(other))
    compiled = torch.compile(m, backend="eager", fullgraph=True)
    assert torch.equal(compiled(other), m(other))


def test_gradient_refusals_before_the_kernels():
    ids, dy = torch.zeros(3, dtype=torch.long), torch.zeros(3, 4)
    for g in (dy, dy.clone().requires_grad_()):
        with pytest.raises(RuntimeError, match="accumulate needs out"):
            hm.embedding_grad(ids, g, 8, accumulate=True)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(dy, torch.ones_like(dy))
        with pytest.raises(RuntimeError, match="accumulate needs out"):
            hm.embedding_grad(ids, dual, 8, accumulate=True)
        out = forward_ad.make_dual(torch.zeros(8, 4), torch.ones(8, 4))
        for accumulate in (False, True):
            with torch.no_grad(), pytest.raises(RuntimeError, match="no tangent"):
                hm.embedding_grad(ids, dy, 8, out=out, accumulate=accumulate)
        assert out.eq(0).all()
