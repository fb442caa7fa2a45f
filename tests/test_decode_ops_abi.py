"""The C entries of the decode-side operators on the CPU: arguments are refused before any HIP call,
empty inputs are accepted, and CPU tensors are refused by the Python calls."""
import ctypes

import pytest
import torch

import hdcmamba_amd as hm
from hdcmamba_amd import _ops

OK, EINVAL, EALIGN, EUNSUPPORTED, EWORKSPACE = 0, -1, -2, -3, -5
F32, BF16 = _ops.HDCM_F32, _ops.HDCM_BF16
P16 = ctypes.c_void_p(16 * 1024)      # never dereferenced: every call fails validation or is empty
P18 = ctypes.c_void_p(16 * 1024 + 2)


def with_(base, **at):
    a = list(base)
    for k, v in at.items():
        a[int(k[1:])] = v
    return a


def test_packed_bytes():
    f = _ops.lib().hdcm_w4_packed_bytes
    assert f(16, 128) == 1024 and f(17, 129) == 4 * 1024 and f(1, 1) == 1024
    assert f(50304, 2048) == 50304 * 2048 // 2
    assert f(0, 128) == 0 and f(16, 0) == 0


def test_w4_linear_validation():
    f = _ops.lib().hdcm_w4_linear_fwd
    # x, x_rs, row_sums, eps, packed, scales, scale_dtype, zeros, group, bias, res, res_rs, out, out_rs, M, N, K, dtype, stream
    base = [P16, 2048, None, 1e-5, P16, P16, BF16, None, 128, None, None, 0, P16, 8576, 16, 8576, 2048, BF16, None]
    assert f(*with_(base, _17=7)) == EUNSUPPORTED
    assert f(*with_(base, _6=2)) == EUNSUPPORTED
    assert f(*with_(base, _8=16)) == EUNSUPPORTED
    assert f(*with_(base, _8=256)) == EUNSUPPORTED
    assert f(*with_(base, _16=7)) == EUNSUPPORTED  # shorter than one load
    assert f(*with_(base, _2=P16, _17=F32)) == EUNSUPPORTED
    assert f(*with_(base, _2=P16, _3=-1.0)) == EINVAL
    assert f(*with_(base, _2=P16, _3=float("nan"))) == EINVAL
    assert f(*with_(base, _0=None)) == EINVAL
    assert f(*with_(base, _5=None)) == EINVAL
    assert f(*with_(base, _16=0)) == EINVAL
    assert f(*with_(base, _1=2047)) == EINVAL    # rows overlap
    assert f(*with_(base, _13=8575)) == EINVAL
    assert f(*with_(base, _10=P16, _11=100)) == EINVAL
    assert f(*with_(base, _4=P18)) == EALIGN
    assert f(*with_(base, _5=P18)) == EALIGN
    assert f(*with_(base, _14=-1)) == EINVAL
    assert f(*with_(base, _14=0, _0=None, _12=None)) == OK
    assert f(*with_(base, _15=0, _4=None, _5=None, _12=None)) == OK


def test_w4_pack_quantize_dequant_validation():
    lib = _ops.lib()
    pack = [P16, 256, 64, 256, P16, None]
    assert lib.hdcm_w4_pack(*with_(pack, _0=None)) == EINVAL
    assert lib.hdcm_w4_pack(*with_(pack, _1=255)) == EINVAL
    assert lib.hdcm_w4_pack(*with_(pack, _4=P18)) == EALIGN
    assert lib.hdcm_w4_pack(*with_(pack, _2=0, _0=None, _4=None)) == OK
    quant = [P16, 256, 64, 256, 128, P16, P16, BF16, None, BF16, None]
    assert lib.hdcm_w4_quantize(*with_(quant, _4=100)) == EUNSUPPORTED
    assert lib.hdcm_w4_quantize(*with_(quant, _9=5)) == EUNSUPPORTED
    assert lib.hdcm_w4_quantize(*with_(quant, _6=None)) == EINVAL
    assert lib.hdcm_w4_quantize(*with_(quant, _5=P18)) == EALIGN
    assert lib.hdcm_w4_quantize(*with_(quant, _2=0)) == OK
    deq = [P16, P16, BF16, None, 64, P16, 256, 64, 256, BF16, None]
    assert lib.hdcm_w4_dequant(*with_(deq, _4=48)) == EUNSUPPORTED
    assert lib.hdcm_w4_dequant(*with_(deq, _6=255)) == EINVAL
    assert lib.hdcm_w4_dequant(*with_(deq, _5=None)) == EINVAL
    assert lib.hdcm_w4_dequant(*with_(deq, _7=0, _0=None, _1=None, _5=None)) == OK


def controls(**kw):
    c = _ops.LogitsControls(repetition_all=1.0)
    for k, v in kw.items():
        setattr(c, k, v.value if isinstance(v, ctypes.c_void_p) else v)
    return ctypes.byref(c)


def test_logits_process_validation():
    f = _ops.lib().hdcm_logits_process
    # logits, l_rs, controls, out, o_rs, B, V, dtype, stream
    base = [P16, 1000, controls(), P16, 1000, 4, 1000, BF16, None]
    assert f(*with_(base, _7=3)) == EUNSUPPORTED
    assert f(*with_(base, _0=None)) == EINVAL
    assert f(*with_(base, _2=None)) == EINVAL
    assert f(*with_(base, _1=999)) == EINVAL
    assert f(*with_(base, _4=999)) == EINVAL
    assert f(*with_(base, _6=(1 << 30) + 1, _1=1 << 31, _4=1 << 31)) == EUNSUPPORTED
    assert f(*with_(base, _2=controls(history=P16, history_row_stride=999))) == EINVAL
    assert f(*with_(base, _2=controls(bias=P16, bias_row_stride=10))) == EINVAL
    assert f(*with_(base, _2=controls(bias=P16, bias_dtype=9))) == EUNSUPPORTED
    assert f(*with_(base, _2=controls(mask=P16, mask_row_stride=31))) == EINVAL
    assert f(*with_(base, _5=0, _0=None)) == OK
    assert f(*with_(base, _6=0, _0=None)) == OK


def test_token_select_validation():
    lib = _ops.lib()
    f = lib.hdcm_token_select
    need = lib.hdcm_token_select_workspace_bytes(4, 50304)
    # logits, l_rs, controls, temp, temp_all, noise, n_rs, tokens, logprobs, ws, ws_bytes, B, V, dtype, stream
    base = [P16, 50304, controls(), None, 1.0, None, 0, P16, P16, P16, need, 4, 50304, BF16, None]
    assert f(*with_(base, _13=3)) == EUNSUPPORTED
    assert f(*with_(base, _7=None)) == EINVAL
    assert f(*with_(base, _8=None)) == EINVAL
    assert f(*with_(base, _5=P16, _6=50303)) == EINVAL
    assert f(*with_(base, _12=0)) == EINVAL  # nothing to choose from
    assert f(*with_(base, _11=1 << 16)) == EUNSUPPORTED
    if need:
        assert f(*with_(base, _9=None)) == EWORKSPACE
        assert f(*with_(base, _10=need - 1)) == EWORKSPACE
        assert f(*with_(base, _9=P18)) == EALIGN
    assert f(*with_(base, _11=0, _0=None)) == OK


def test_token_history_validation():
    lib = _ops.lib()
    # table, rs, prompt, p_rs, p_len, P, output, o_rs, o_len, O, B, V, stream
    base = [P16, 1000, P16, 8, None, 8, P16, 4, None, 4, 2, 1000, None]
    f = lib.hdcm_token_history_fill
    assert f(*with_(base, _0=None)) == EINVAL
    assert f(*with_(base, _2=None)) == EINVAL
    assert f(*with_(base, _1=999)) == EINVAL
    assert f(*with_(base, _3=7)) == EINVAL
    assert f(*with_(base, _5=-1)) == EINVAL
    assert f(*with_(base, _10=1 << 16)) == EUNSUPPORTED
    assert f(*with_(base, _10=0)) == OK
    # table, rs, tokens, t_rs, lengths, T, B, V, stream
    g = lib.hdcm_token_history_append
    app = [P16, 1000, P16, 1, None, 1, 2, 1000, None]
    assert g(*with_(app, _2=None)) == EINVAL
    assert g(*with_(app, _3=0)) == EINVAL
    assert g(*with_(app, _5=0, _2=None)) == OK


@pytest.mark.parametrize("call", [
    lambda: hm.Weight4Bit.quantize(torch.zeros(16, 128)),
    lambda: hm.Weight4Bit.from_codes(torch.zeros(16, 128, dtype=torch.uint8), torch.ones(16, 1)),
    lambda: hm.process_logits(torch.zeros(1, 8)),
    lambda: hm.select_tokens(torch.zeros(1, 8)),
    lambda: hm.fill_token_history(torch.zeros(1, 8, dtype=torch.int16)),
    lambda: hm.append_tokens(torch.zeros(1, 8, dtype=torch.int16), torch.zeros(1, dtype=torch.long)),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(RuntimeError, match="no CPU path"):
        call()


def test_new_token_history_pads_rows():
    t = hm.new_token_history(3, 50277, device="cpu")
    assert t.shape == (3, 50277) and t.stride() == (50280, 1) and t.dtype == torch.int16 and not t.any()
