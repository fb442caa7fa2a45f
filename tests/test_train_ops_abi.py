"""The operators at the ends of a training step on the CPU: the C entries refuse arguments before any HIP call and accept
empty inputs, the Python calls refuse CPU tensors and bad settings, and Embedding is nn.Embedding there."""
import ctypes
import math

import pytest
import torch
import torch.nn as nn

import hdcmamba_amd as hm
from hdcmamba_amd import _ops

OK, EINVAL, EALIGN, EUNSUPPORTED, EWORKSPACE = 0, -1, -2, -3, -5
F32, BF16 = _ops.HDCM_F32, _ops.HDCM_BF16
P16 = ctypes.c_void_p(16 * 1024)      # never dereferenced: every call fails validation or is empty
P18 = ctypes.c_void_p(16 * 1024 + 2)
P17 = ctypes.c_void_p(16 * 1024 + 1)


def with_(base, **at):
    a = list(base)
    for k, v in at.items():
        a[int(k[1:])] = v
    return a


def test_embedding_fwd_validation():
    f = _ops.lib().hdcm_embedding_fwd
    # ids, id_bytes, w, w_rs, out, out_rs, rows, V, D, scale, dtype, stream
    base = [P16, 8, P16, 1024, P16, 1024, 16, 50304, 1024, 1.0, BF16, None]
    assert f(*with_(base, _10=7)) == EUNSUPPORTED
    assert f(*with_(base, _1=2)) == EUNSUPPORTED
    assert f(*with_(base, _0=None)) == EINVAL
    assert f(*with_(base, _2=None)) == EINVAL
    assert f(*with_(base, _4=None)) == EINVAL
    assert f(*with_(base, _3=1023)) == EINVAL
    assert f(*with_(base, _5=1023)) == EINVAL
    assert f(*with_(base, _6=-1)) == EINVAL
    assert f(*with_(base, _6=(1 << 30) + 1)) == EUNSUPPORTED
    assert f(*with_(base, _7=(1 << 30) + 1)) == EUNSUPPORTED
    assert f(*with_(base, _8=(1 << 24) + 1, _3=1 << 25, _5=1 << 25)) == EUNSUPPORTED
    assert f(*with_(base, _6=0, _0=None, _4=None)) == OK
    assert f(*with_(base, _8=0, _2=None, _4=None)) == OK


def test_embedding_grad_validation():
    lib = _ops.lib()
    f, need = lib.hdcm_embedding_grad, lib.hdcm_embedding_grad_workspace_bytes
    n = need(2, 4096, 50304, 1024, BF16)
    assert 0 < n < 64 << 20
    assert need(0, 4096, 50304, 1024, BF16) == 0 and need(2, 4096, 0, 1024, BF16) == 0
    assert need(1 << 20, 1 << 20, 50304, 1024, BF16) == 0  # more than the kernels take
    # ids, id_bytes, dy, dy_bs, dy_rs, dw, dw_rs, dw_dtype, ws, ws_bytes, B, L, V, D, scale, padding, accumulate, dtype, stream
    base = [P16, 8, P16, 4096 * 1024, 1024, P16, 1024, BF16, P16, n, 2, 4096, 50304, 1024, 1.0, -1, 0, BF16, None]
    assert f(*with_(base, _17=5)) == EUNSUPPORTED
    assert f(*with_(base, _7=5)) == EUNSUPPORTED
    assert f(*with_(base, _1=1)) == EUNSUPPORTED
    assert f(*with_(base, _0=None)) == EINVAL
    assert f(*with_(base, _2=None)) == EINVAL
    assert f(*with_(base, _5=None)) == EINVAL
    assert f(*with_(base, _6=1023)) == EINVAL
    assert f(*with_(base, _4=1023)) == EINVAL
    assert f(*with_(base, _3=-1)) == EINVAL
    assert f(*with_(base, _15=50304)) == EINVAL
    assert f(*with_(base, _15=-2)) == EINVAL
    assert f(*with_(base, _10=-1)) == EINVAL
    assert f(*with_(base, _8=None)) == EWORKSPACE
    assert f(*with_(base, _9=n - 1)) == EWORKSPACE
    assert f(*with_(base, _8=P18)) == EALIGN
    assert f(*with_(base, _10=1 << 20, _11=1 << 20)) == EUNSUPPORTED
    assert f(*with_(base, _12=0, _5=None)) == OK
    assert f(*with_(base, _13=0, _5=None)) == OK
    assert f(*with_(base, _10=0, _16=1, _5=None)) == OK  # nothing to add


def tensors(*specs):
    a = (_ops.TensorRef * len(specs))()
    for t, (data, count, dtype) in zip(a, specs):
        t.data, t.count, t.dtype = data.value if data else None, count, dtype
    return a


def test_grad_norm_validation():
    lib = _ops.lib()
    f, need = lib.hdcm_grad_norm, lib.hdcm_grad_norm_workspace_bytes
    good = tensors((P16, 1000, BF16), (P18, 7, BF16), (P16, 1 << 31, F32))
    n = need(good, 3)
    assert n > 0 and n % 8 == 0 and need(good, 0) == 0
    # tensors, n, norm, out, ws, ws_bytes, stream
    base = [good, 3, 0, P16, P16, n, None]
    assert f(*with_(base, _2=2)) == EUNSUPPORTED
    assert f(*with_(base, _3=None)) == EINVAL
    assert f(*with_(base, _1=-1)) == EINVAL
    assert f(*with_(base, _0=None)) == EINVAL
    assert f(*with_(base, _4=None)) == EWORKSPACE
    assert f(*with_(base, _5=n - 8)) == EWORKSPACE
    assert f(*with_(base, _4=P18)) == EALIGN
    for bad, code in (((P16, 10, 3), EUNSUPPORTED), ((P16, -1, F32), EINVAL), ((None, 10, F32), EINVAL), ((P18, 10, F32), EALIGN),
                      ((P17, 10, BF16), EALIGN)):
        t = tensors(bad)
        assert f(*with_(base, _0=t, _1=1)) == code and need(t, 1) == 0
    h = lib.hdcm_clip_grad_norm  # tensors, n, norm, max_norm, out, ws, ws_bytes, stream
    both = [good, 3, 0, 1.0, P16, P16, n, None]
    assert h(*with_(both, _2=2)) == EUNSUPPORTED
    assert h(*with_(both, _3=-1.0)) == EINVAL
    assert h(*with_(both, _3=float("nan"))) == EINVAL
    assert h(*with_(both, _4=None)) == EINVAL
    assert h(*with_(both, _6=n - 8)) == EWORKSPACE
    assert h(*with_(both, _5=P18)) == EALIGN
    g = lib.hdcm_grad_scale  # tensors, n, norm, max_norm, stream
    assert g(good, 3, None, 1.0, None) == EINVAL
    assert g(good, 3, P16, -1.0, None) == EINVAL
    assert g(good, 3, P16, float("nan"), None) == EINVAL
    assert g(tensors((P16, 10, 3)), 1, P16, 1.0, None) == EUNSUPPORTED
    assert g(None, 0, P16, 1.0, None) == OK
    assert g(tensors((None, 0, F32)), 1, P16, 1.0, None) == OK


@pytest.mark.parametrize("call", [
    lambda: hm.embedding(torch.zeros(3, dtype=torch.long), torch.zeros(8, 4)),
    lambda: hm.embedding_grad(torch.zeros(3, dtype=torch.long), torch.zeros(3, 4), 8),
    lambda: hm.grad_norm([torch.zeros(4)]),
    lambda: hm.clip_grads_([torch.zeros(4)], 1.0, torch.zeros(())),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(RuntimeError, match="no CPU path"):
        call()


def test_settings_are_refused():
    p = nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="no CPU path"):
        hm.clip_grad_norm_([p], 1.0)
    for norm_type in (1, 0, -math.inf, 3.0):
        with pytest.raises(ValueError, match="norm_type"):
            hm.clip_grad_norm_([p], 1.0, norm_type)
        with pytest.raises(ValueError, match="norm_type"):
            hm.grad_norm([p.grad], norm_type)
    for limit in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            hm.clip_grad_norm_([p], limit)
        with pytest.raises(ValueError, match="max_norm"):
            hm.clip_grads_([p.grad], limit, 1.0)
    for index in (8, -9):
        with pytest.raises(ValueError, match="padding_idx"):
            hm.embedding(torch.zeros(3, dtype=torch.long), torch.zeros(8, 4), padding_idx=index)
        with pytest.raises(ValueError, match="padding_idx"):
            hm.embedding_grad(torch.zeros(3, dtype=torch.long), torch.zeros(3, 4), 8, padding_idx=index)
    assert p.grad.eq(1).all()


def test_nothing_to_clip():
    """As torch's: no tensors, or parameters without gradients, have the norm 0."""
    assert hm.grad_norm([]).item() == 0.0
    assert hm.clip_grad_norm_([nn.Parameter(torch.zeros(3))], 1.0).item() == 0.0
    assert hm.clip_grads_([], 1.0, 2.0) is None
    assert hm.clip_grad_norm_([nn.Parameter(torch.zeros(3))], 1.0, error_if_nonfinite=True).item() == 0.0


def test_embedding_module_is_nn_embedding_on_the_cpu():
    """The same initial values from the same generator state, and nn.Embedding's own forward where the kernels do not run."""
    torch.manual_seed(5)
    a, after_a = nn.Embedding(11, 6, padding_idx=-2), torch.rand(1)
    torch.manual_seed(5)
    b, after_b = hm.Embedding(11, 6, padding_idx=-2, scale=3.0), torch.rand(1)
    assert torch.equal(a.weight, b.weight) and torch.equal(after_a, after_b) and a.padding_idx == b.padding_idx == 9
    assert isinstance(b, nn.Embedding) and list(b.state_dict()) == ["weight"] and "scale=3.0" in repr(b)
    ids = torch.tensor([[1, 9, 1], [0, 10, 4]])
    (a(ids) * 3).square().sum().backward()
    b(ids).square().sum().backward()
    assert torch.equal(a(ids) * 3, b(ids)) and torch.equal(a.weight.grad, b.weight.grad)
    c = hm.Embedding.from_pretrained(a.weight.detach(), freeze=False)
    assert c.scale == 1.0 and torch.equal(c(ids), a(ids)) and c.weight.requires_grad
    lm = hm.HdcMambaLM(64, 1, 16, 2, vocab_size=32)
    assert isinstance(lm.embedding, hm.Embedding) and lm.lm_head.weight is lm.embedding.weight
