"""Calls of Embedding and its gradient that end before any kernel runs: tensors of other classes, modes, refusals."""
import ctypes

import pytest
import torch
import torch.nn as nn
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.utils._python_dispatch import TorchDispatchMode

import hdcmamba_amd as hm
from hdcmamba_amd import _ops


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


P16 = ctypes.c_void_p(16 * 1024)  # never dereferenced: every call is refused


def test_launches_of_2_to_the_32_threads_are_refused():
    lib, U = _ops.lib(), -3  # HDCM_EUNSUPPORTED
    # ids, id_bytes, w, w_rs, out, out_rs, rows, V, D, scale, dtype, stream
    f = lambda rows, D, dtype: lib.hdcm_embedding_fwd(P16, 4, P16, D, P16, D, rows, 100, D, 1.0, dtype, None)  # noqa: E731
    assert f(1 << 30, 64, _ops.HDCM_BF16) == U  # 2^33 pieces, two a thread
    assert f((1 << 30) - 3, 33, _ops.HDCM_F32) == U
    # ids, id_bytes, dy, dy_bs, dy_rs, dw, dw_rs, dw_dtype, ws, ws_bytes, B, L, V, D, scale, padding, accumulate, dtype, stream
    def g(L, V, D, rs, accumulate=0, dtype=_ops.HDCM_BF16):
        return lib.hdcm_embedding_grad(P16, 4, P16, 0, 0, P16, rs, dtype, P16, 1 << 62, 1, L, V, D, 1.0, -1, accumulate, dtype, None)

    assert g(1 << 30, 100, 513, 513) == U            # sums: 2^23 workgroups of 512 threads
    assert g(0, 1 << 28, 128, 200) == U              # zeros of rows apart
    assert g(9000, 1 << 28, 128, 200) == U
    assert g(9000, 1 << 28, 520, 520) == U           # zeros beside the sorting: more than 2^38 bytes
    assert g(9000, 1 << 28, 520, 520, dtype=_ops.HDCM_F32) == U
