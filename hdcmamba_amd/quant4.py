"""4-bit weights with group scales for the decode step's products (csrc/linear4.hip).

A weight [N, K] is held as codes 0..15 with a scale, and optionally a zero point, per row and group of
32, 64 or 128 columns: w[n, k] = scales[n, g] * (codes[n, k] - zeros[n, g]), zeros 8 where there are
none.  Inference only, on the GPU only, as every operator of this package.  The reference holds its
weights in the activation type (hdcmamba/model.py:313,325; train_fineweb.py:55); 4-bit weights have no
counterpart there.
"""
from __future__ import annotations

from contextlib import contextmanager

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd import forward_ad

from . import _ops

__all__ = ["Weight4Bit", "linear_4bit", "Linear4Bit"]

GROUP_SIZES = (32, 64, 128)


def carries_tangent(x):
    """Whether x is a dual tensor of forward-mode differentiation."""
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None


@contextmanager
def _buffers_on(device):
    """Allocate a weight's buffers: on ``device``, and under inference mode too as tensors that count their writes
    (which keeps the row sums in line with them)."""
    with torch.cuda.device(device), torch.inference_mode(False), torch.no_grad():
        yield


class Weight4Bit:
    """A packed 4-bit weight: made once from codes (``from_codes``) or by rounding a weight
    (``quantize``), then passed to linear_4bit.  Its buffers may be written in place (load_state_dict): the
    row sums that norm_eps reads are formed again, with a wait of the host, by the next call with it.
    Inside a recording that is refused: ``refresh`` first; a graph recorded before sees the new sums after
    ``refresh`` too, and so does any call after a write through ``.data``, which tensors do not count.

    ``shape`` (N, K), ``group_size``; ``packed`` uint8, ``scales`` (float32 or bfloat16) and ``zeros``
    (uint8 or None) in the layout of hdcm_w4_linear_fwd (include/hdcm.h)."""

    __slots__ = ("packed", "scales", "zeros", "shape", "group_size", "_handle")

    def __init__(self, packed, scales, zeros, shape, group_size):
        self.packed, self.scales, self.zeros = packed, scales, zeros
        self.shape, self.group_size = tuple(int(n) for n in shape), int(group_size)
        # on the CPU it can be kept, copied and moved, no more
        self._handle = _ops.native().Weight4(packed, scales, zeros, *self.shape, self.group_size) if packed.is_cuda else None

    def __reduce__(self):  # copies and pickles are made from the buffers
        return Weight4Bit, (self.packed, self.scales, self.zeros, self.shape, self.group_size)

    @staticmethod
    def _groups(N, K, group_size):
        """(padded groups, padded rows) of the scale layout."""
        if group_size not in GROUP_SIZES:
            raise ValueError(f"group_size must be one of {GROUP_SIZES}, got {group_size}")
        if N < 1 or K < 1:
            raise ValueError(f"a 4-bit weight needs rows and columns, got [{N}, {K}]")
        return -(-K // 128) * 128 // group_size, -(-N // 16) * 16

    @classmethod
    def from_codes(cls, codes, scales, zeros=None, group_size=128):
        """codes [N, K] uint8 in 0..15, one per byte; scales [N, ceil(K / group_size)] float32 or
        bfloat16; zeros (zero points, 0..15) uint8 of the scales' shape, or None for 8."""
        _ops._on_gpu(codes, scales, zeros)
        if codes.dim() != 2 or codes.dtype != torch.uint8:
            raise TypeError(f"codes must be a uint8 [N, K] tensor, got {codes.dtype} {tuple(codes.shape)}")
        N, K = codes.shape
        G, Np = cls._groups(N, K, group_size)
        _ops._dtype(scales)
        shape = (N, -(-K // group_size))
        for name, t in (("scales", scales), ("zeros", zeros)):
            if t is not None and (tuple(t.shape) != shape or t.device != codes.device):
                raise ValueError(f"{name} must be {shape} on {codes.device}, got {tuple(t.shape)} on {t.device}")
        if zeros is not None and zeros.dtype != torch.uint8:
            raise TypeError(f"zeros must be uint8, got {zeros.dtype}")
        for name, t in (("codes", codes), ("zeros", zeros)):
            if t is not None and int(t.max()) > 15:
                raise ValueError(f"{name} must be in 0..15, got {int(t.max())}")
        with _buffers_on(codes.device):
            codes = codes.contiguous()
            packed = torch.empty(int(_ops.lib().hdcm_w4_packed_bytes(N, K)), dtype=torch.uint8, device=codes.device)
            _ops._check("hdcm_w4_pack", _ops.lib().hdcm_w4_pack(codes.data_ptr(), codes.stride(0), N, K, packed.data_ptr(),
                                                                _ops._stream(codes)))

            def by_group(t, fill):
                full = torch.full((G, Np), fill, dtype=t.dtype, device=t.device)
                full[:shape[1], :N] = t.detach().t()
                return full

            return cls(packed, by_group(scales, 0), None if zeros is None else by_group(zeros, 8), (N, K), group_size)

    @classmethod
    def quantize(cls, weight, group_size=128, zero_points=False, scale_dtype=None):
        """weight [N, K] (float32 or bfloat16, finite) rounded to 4 bits per group of a row: without
        zero points to -7..7 times the group's largest magnitude / 7, with them to the 16 steps from
        the group's smallest to its largest value (0 among them).  ``scale_dtype``: the weight's by
        default."""
        _ops._on_gpu(weight)
        dtype = _ops._dtype(weight)
        if weight.dim() != 2:
            raise ValueError(f"a weight [N, K] is expected, got {tuple(weight.shape)}")
        weight = weight.detach()
        scale_dtype = weight.dtype if scale_dtype is None else scale_dtype
        if scale_dtype not in _ops._DTYPES:
            raise TypeError(f"scale_dtype must be float32 or bfloat16, got {scale_dtype}")
        N, K = weight.shape
        G, Np = cls._groups(N, K, group_size)
        if not bool(torch.isfinite(weight).all()):
            raise ValueError("a weight with infinities or NaN cannot be rounded to 4 bits")
        dev = weight.device
        with _buffers_on(dev):
            weight = weight.contiguous()
            packed = torch.empty(int(_ops.lib().hdcm_w4_packed_bytes(N, K)), dtype=torch.uint8, device=dev)
            scales = torch.empty(G, Np, dtype=scale_dtype, device=dev)
            zeros = torch.empty(G, Np, dtype=torch.uint8, device=dev) if zero_points else None
            _ops._check("hdcm_w4_quantize", _ops.lib().hdcm_w4_quantize(
                weight.data_ptr(), weight.stride(0), N, K, group_size, packed.data_ptr(), scales.data_ptr(),
                _ops._DTYPES[scale_dtype], None if zeros is None else zeros.data_ptr(), dtype, _ops._stream(weight)))
        return cls(packed, scales, zeros, (N, K), group_size)

    def dequantize(self, dtype=torch.bfloat16):
        """The weight [N, K] it stands for, rounded once to ``dtype`` (float32 or bfloat16)."""
        if dtype not in _ops._DTYPES:
            raise TypeError(f"dtype must be float32 or bfloat16, got {dtype}")
        _ops._on_gpu(self.packed)
        self._handle.check()
        N, K = self.shape
        with torch.cuda.device(self.packed.device):
            out = torch.empty(N, K, dtype=dtype, device=self.packed.device)
            _ops._check("hdcm_w4_dequant", _ops.lib().hdcm_w4_dequant(
                self.packed.data_ptr(), self.scales.data_ptr(), _ops._dtype(self.scales),
                None if self.zeros is None else self.zeros.data_ptr(), self.group_size, out.data_ptr(), K, N, K,
                _ops._DTYPES[dtype], _ops._stream(out)))
        return out

    def to(self, device):
        """The same weight on another device."""
        move = lambda t: None if t is None else t.to(device)  # noqa: E731
        return Weight4Bit(move(self.packed), move(self.scales), move(self.zeros), self.shape, self.group_size)

    def refresh(self):
        """Bring what the weight keeps beside its buffers (the row sums of norm_eps) in line with them."""
        _ops._on_gpu(self.packed)
        self._handle.refresh()

    def __repr__(self):
        return (f"Weight4Bit({self.shape[0]}x{self.shape[1]}, group_size={self.group_size}, "
                f"zero_points={self.zeros is not None}, scales={self.scales.dtype}, device={self.packed.device})")


def linear_4bit(x, weight, bias=None, residual=None, out=None, norm_eps=None):
    """x [..., K] times a Weight4Bit [N, K], transposed, (+ bias [N]) (+ residual [..., N]) -> [..., N] in
    x's type (float32 or bfloat16): fp32 sums of exact code products, the scales applied to the groups'
    sums, one rounding.  At most 16 * 65535 rows.  ``out`` may be ``residual``.  ``norm_eps`` (bfloat16 rows of at least 8 columns):
    the product of the rows after a LayerNorm without affine, in the same launch; its variance is the
    difference of two fp32 sums, for rows whose mean is not far above their deviation.  bf16 rows hold
    values up to 2^115 (4e34): larger ones may become infinite or NaN in the sums of x (16 + c), and a row
    that holds an infinity becomes NaN.  No gradient: refused where one would be recorded or carried forward."""
    if weight._handle is None:
        _ops._on_gpu(weight.packed)
    return _ops.native().linear_4bit(x, weight._handle, bias, residual, out, norm_eps)


class Linear4Bit(nn.Module):
    """nn.Linear with a Weight4Bit in place of its weight, for inference: the packed weight, its scales and
    zero points are buffers, the bias (or None) a parameter that takes no gradient.

    Up to ``direct_rows`` rows go through linear_4bit; more multiply by the weight brought back to x's
    type, which rounds it once more (measured at d_model 2048, us: in_proj with 256 rows 21 against 37,
    384 25 against 34, 768 44 against 46; the head with 768 198 against 185; in groups of 32 the in_proj
    with 256 rows 28 against 36, 384 37 against 33).  In an autocast region x is cast to its type first,
    as nn.Linear does (float16, which the kernels do not take, is refused)."""

    direct_rows = 384

    def __init__(self, weight, bias=None):
        super().__init__()
        self.out_features, self.in_features = weight.shape
        self.group_size = weight.group_size
        self.register_buffer("packed", weight.packed)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("zeros", weight.zeros)
        self.bias = None if bias is None else nn.Parameter(bias.detach(), requires_grad=False)
        self._weight4 = weight

    @classmethod
    def from_linear(cls, linear, group_size=128, zero_points=False, scale_dtype=None):
        """The nn.Linear's weight rounded to 4 bits (Weight4Bit.quantize); the bias is shared."""
        return cls(Weight4Bit.quantize(linear.weight, group_size, zero_points, scale_dtype), linear.bias)

    @property
    def weight4(self) -> Weight4Bit:
        """The buffers as the packed weight that linear_4bit takes."""
        w = self._weight4
        if w is None or w.packed is not self.packed or w.scales is not self.scales or w.zeros is not self.zeros:
            w = self._weight4 = Weight4Bit(self.packed, self.scales, self.zeros, (self.out_features, self.in_features),
                                           self.group_size)
        return w

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        if self.packed.is_cuda and self.scales.dtype in _ops._DTYPES:
            self.weight4  # the same one (which recordings read) where nothing was moved
        else:
            self._weight4 = None  # nothing holds the buffers from before
        return self

    def __getstate__(self):  # the buffers once
        return dict(self.__dict__, _weight4=None)

    def _load_from_state_dict(self, *args, **kwargs):
        super()._load_from_state_dict(*args, **kwargs)
        if self.packed.is_cuda:
            self.weight4.refresh()
        else:
            self._weight4 = None

    def forward(self, x):
        if (torch.is_grad_enabled() and x.requires_grad) or carries_tangent(x):
            raise RuntimeError("a Linear4Bit has no gradient: call it under torch.no_grad() or on detached tensors")
        if torch.is_autocast_enabled("cuda"):  # as nn.Linear's, one type for any number of rows
            x = x.to(torch.get_autocast_dtype("cuda"))
        rows = x.numel() // max(x.shape[-1], 1)
        if rows > self.direct_rows:
            return F.linear(x, self.weight4.dequantize(x.dtype), None if self.bias is None else self.bias.to(x.dtype))
        return linear_4bit(x, self.weight4, self.bias)

    def extra_repr(self):
        return (f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, "
                f"group_size={self.group_size}, zero_points={self.zeros is not None}")
