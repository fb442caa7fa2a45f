"""4-bit products, logits processing, token choice and token history against plain implementations.

Products: every output within the rounding of its type plus what fp32 sums of exact products may lose.
fp32 rows sum K products x (c - z), bf16 rows the 2 K products x (16 + c) and -x (16 + z): a step of
2^-23 per addition (covers an accumulator that truncates) of the sum of their magnitudes.  Processed logits: bit for bit the fp32 formula, operation by operation.
"""
import copy
import pickle

import pytest
import torch

import hdcmamba_amd as hm
from hdcmamba_amd import _ops

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _say(*a):
    print(*a, flush=True)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------------------- 4-bit products
def _weight(N, K, group, zeros, sdt, seed):
    g = _gen(seed)
    codes = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8)
    n = -(-K // group)
    scales = (0.01 + 0.02 * torch.rand(N, n, generator=g)).to(sdt)
    z = torch.randint(0, 16, (N, n), generator=g, dtype=torch.uint8) if zeros else None
    return codes, scales, z


def _dense(codes, scales, z, group):
    K = codes.shape[1]
    wide = lambda t: t.double().repeat_interleave(group, 1)[:, :K]  # noqa: E731
    return (codes.double() - (wide(z) if z is not None else 8.0)) * wide(scales)


def _check_linear(got, x, codes, scales, z, group, bias, res):
    """got against x w^T + bias + res in 64 bits, elementwise."""
    N, K = codes.shape
    w, x = _dense(codes, scales, z, group), x.double()
    ref = x @ w.t()
    if got.dtype == F32:
        mag, n = x.abs() @ w.abs().t(), K
    else:
        wide = lambda t: t.double().repeat_interleave(group, 1)[:, :K]  # noqa: E731
        mag, n = x.abs() @ ((32 + codes.double() + (wide(z) if z is not None else 8.0)) * wide(scales)).t(), 2 * K
    for t in (bias, res):
        if t is not None:
            ref, mag = ref + t.double(), mag + t.double().abs()
    tol = torch.finfo(got.dtype).eps / 2 * ref.abs() + (n + 8) * 2.0**-23 * mag
    err = (got.cpu().double() - ref).abs()
    worst = float((err / tol.clamp_min(1e-300)).max()) if err.numel() else 0.0
    _say("  worst error / tolerance", worst)
    assert worst <= 1.0


LINEAR = [
    # M, K, N, group, zeros, scale type, x type
    (1, 128, 16, 128, False, BF, BF),
    (1, 1152, 1024, 128, False, BF, BF),
    (2, 1, 1, 32, True, F32, BF),          # one column, one row
    (3, 768, 3264, 64, True, F32, F32),
    (16, 2048, 544, 128, False, BF, BF),
    (17, 832, 300, 128, True, BF, BF),     # a last group of 64 columns, a row past a tile
    (5, 1000, 77, 32, True, F32, BF),      # ragged everywhere
    (33, 333, 129, 64, False, BF, F32),    # odd K: unaligned rows
    (64, 256, 48, 32, False, F32, BF),
    (65, 384, 130, 128, True, BF, BF),     # a second block of rows
    (200, 130, 40, 64, True, F32, F32),
    (7, 4224, 96, 128, False, BF, BF),     # more column tiles than waves take at once
    (31, 96, 1, 32, False, BF, F32),
    (40, 2048, 100, 128, True, BF, BF),    # three row tiles
    (16, 2176, 2048, 128, False, BF, BF),  # seventeen column tiles
    (50, 3000, 70, 32, True, F32, BF),     # too many column tiles for three
    (20, 2500, 33, 64, False, BF, F32),
    (70, 3200, 50, 32, True, BF, BF),      # longer rows than the registers take
    (3, 5001, 40, 64, False, F32, F32),
    (2, 7, 20, 32, False, BF, BF),         # rows shorter than a 16-byte load
    (2, 3, 20, 32, True, BF, F32),
    (4, 9, 17, 64, True, F32, BF),
    (129, 128, 4200, 64, False, BF, BF),   # more output tiles than workgroups
    (64, 4096, 200, 128, False, BF, BF),   # two segments of K
    (41, 4000, 4200, 64, True, F32, BF),
    (90, 3300, 150, 32, True, BF, BF),
    (2, 9000, 8200, 128, True, BF, BF),
    (1100, 3300, 5200, 128, False, BF, BF),  # more sums to hold than a workgroup has room for
    (30, 6500, 100, 64, False, BF, F32),
    (70, 256, 4096, 128, False, BF, BF),   # five row tiles where four blocks would fill the card
    (90, 100, 3000, 64, True, BF, BF),     # one wave a workgroup
]


@pytest.mark.parametrize("M,K,N,group,zeros,sdt,dtype", LINEAR)
@pytest.mark.parametrize("extra", ["", "bias", "both"])
def test_linear_4bit(dev, M, K, N, group, zeros, sdt, dtype, extra):
    _say("linear_4bit", M, K, N, group, zeros, sdt, dtype, extra)
    codes, scales, z = _weight(N, K, group, zeros, sdt, seed=K + N)
    g = _gen(M)
    x = torch.randn(M, K, generator=g).to(dtype)
    bias = torch.randn(N, generator=g).to(dtype) if extra else None
    res = torch.randn(M, N, generator=g).to(dtype) if extra == "both" else None
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    w = hm.Weight4Bit.from_codes(to(codes), to(scales), to(z), group)
    got = hm.linear_4bit(to(x), w, bias=to(bias), residual=to(res))
    assert got.shape == (M, N) and got.dtype == dtype
    _check_linear(got, x, codes, scales, z, group, bias, res)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_linear_4bit_layouts(dev, dtype):
    """Rows of a wider buffer, unaligned starts, extra leading dimensions, a single row as [K], no rows,
    an output of its own in place of the residual: the same values as contiguous operands give."""
    N, K, group = 144, 200, 32
    codes, scales, z = (t.to(dev) for t in _weight(N, K, group, True, BF, 3))
    w = hm.Weight4Bit.from_codes(codes, scales, z, group)
    x = torch.randn(6, K, generator=_gen(1)).to(dtype).to(dev)
    want = hm.linear_4bit(x, w)
    wide = torch.full((6, K + 37), float("nan"), dtype=dtype, device=dev)  # what lies past the K columns is not read
    wide[:, 1:1 + K] = x
    assert torch.equal(hm.linear_4bit(wide[:, 1:1 + K], w), want)
    assert torch.equal(hm.linear_4bit(x.t().contiguous().t(), w), want)
    assert torch.equal(hm.linear_4bit(x.view(2, 3, K), w), want.view(2, 3, N))
    assert torch.equal(hm.linear_4bit(x[2], w), want[2])
    assert torch.equal(hm.linear_4bit(x[:1].expand(4, K), w), want[:1].expand(4, N))
    assert hm.linear_4bit(x[:0], w).shape == (0, N)
    out = torch.full((6, N + 5), 7.0, dtype=dtype, device=dev)
    r = torch.randn(6, N, generator=_gen(2)).to(dtype).to(dev)
    out[:, 2:2 + N] = r
    view = out[:, 2:2 + N]
    assert hm.linear_4bit(x, w, residual=view, out=view).data_ptr() == view.data_ptr()
    assert torch.equal(view, hm.linear_4bit(x, w, residual=r))
    assert (out[:, :2] == 7).all() and (out[:, 2 + N:] == 7).all()


@pytest.mark.parametrize("M,K,N,group,zeros", [
    (1, 8, 16, 32, False), (1, 1152, 100, 128, False), (16, 2176, 70, 128, True), (5, 333, 33, 32, True),
    (40, 2048, 50, 64, False), (64, 832, 60, 128, False), (100, 1000, 20, 128, True), (3, 23 * 128, 64, 64, True),
    (33, 5000, 300, 128, False), (33, 17 * 128 + 1, 48, 32, False), (16, 768, 8500, 128, True),
    (40, 100, 70, 64, True), (70, 256, 4096, 128, False)])
def test_linear_4bit_with_layer_norm(dev, M, K, N, group, zeros):
    """norm_eps against the LayerNorm and product in 64 bits.

    out = rstd (x w - mean sum w): the two terms in fp32 sums of K exact products each, rounded at most 2 K + 8 times by
    2^-24 of the sum of magnitudes of code products (|c| <= 31 + 24 scales, as for the product alone), times rstd; row_sums
    likewise, times mean.  rstd from v = q / K - mean^2, sums of K positive terms: relative error of v up to
    (K + 4) 2^-24 (q / K + mean^2) / (v + eps), half of that in rstd, times the result without residual."""
    codes, scales, z = _weight(N, K, group, zeros, BF, seed=K)
    x = (torch.randn(M, K, generator=_gen(M)) * 2 + 6 * torch.rand(M, 1, generator=_gen(M + 1)) - 3).to(BF)
    x[0] = 0  # no variance: eps alone
    res = torch.randn(M, N, generator=_gen(M)).to(BF)
    w = hm.Weight4Bit.from_codes(codes.to(dev), scales.to(dev), None if z is None else z.to(dev), group)
    got = hm.linear_4bit(x.to(dev), w, residual=res.to(dev), norm_eps=1e-5).cpu().double()
    xd = x.double()
    mean, var = xd.mean(1, keepdim=True), xd.var(1, unbiased=False, keepdim=True)
    rstd = (var + 1e-5).rsqrt()
    dense = _dense(codes, scales, z, group)
    y = ((xd - mean) * rstd) @ dense.t()
    ref = y + res.double()
    big = (dense.abs() + 48 * scales.double().max()).t()
    sums = (xd.abs() @ big + mean.abs() * big.sum(0)) * rstd
    stat = (K + 4) * 2.0**-24 * ((xd**2).mean(1, keepdim=True) + mean**2) / (var + 1e-5)
    tol = 2.0**-8 * ref.abs() + (2 * K + 8) * 2.0**-24 * sums + stat * (y.abs() + rstd * mean.abs() * dense.sum(1).abs()) + 1e-6
    _say("  worst", float(((got - ref).abs() / tol).max()))
    assert ((got - ref).abs() <= tol).all()
    assert torch.equal(got[0], res[0].double())  # zero rows stay zero
    assert hm.linear_4bit(x[:0].to(dev), w, norm_eps=1e-5).shape == (0, N)


def test_linear_4bit_layer_norm_rows_apart(dev):
    """A row's NaN or infinity stays in its row."""
    w = hm.Weight4Bit.quantize(torch.randn(64, 640, generator=_gen(3)).to(BF).to(dev))
    x = torch.randn(19, 640, generator=_gen(4)).to(BF).to(dev)
    plain = hm.linear_4bit(x, w, norm_eps=1e-5)
    bad = x.clone()
    bad[4, 17], bad[18, 0] = float("nan"), float("inf")
    got = hm.linear_4bit(bad, w, norm_eps=1e-5)
    assert got[4].isnan().all() and got[18].isnan().all()
    keep = [r for r in range(19) if r not in (4, 18)]
    assert torch.equal(got[keep], plain[keep])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_linear_4bit_infinities(dev, dtype):
    """A row's infinity or NaN stays in its row: a bf16 row becomes NaN, an fp32 row what the weights give."""
    N, K = 32, 256
    codes, scales, _ = _weight(N, K, 128, False, F32, 5)
    w = hm.Weight4Bit.from_codes(codes.to(dev), scales.to(dev), None, 128)
    x = torch.randn(4, K, generator=_gen(1)).to(dtype)
    x[1, 7], x[2, 9] = float("inf"), float("nan")
    got = hm.linear_4bit(x.to(dev), w).cpu()
    assert got[0].isfinite().all() and got[3].isfinite().all() and got[2].isnan().all()
    if dtype == BF:
        assert got[1].isnan().all()
    else:  # an infinity times a weight of 0 is NaN
        want = (x[1].double() * _dense(codes, scales, None, 128)).sum(1)
        assert torch.equal(torch.nan_to_num(got[1].double()), torch.nan_to_num(want.float().double()))


@pytest.mark.parametrize("N,K,group,zeros,sdt,dtype", [
    (64, 512, 128, False, BF, BF), (50, 300, 32, True, F32, BF), (33, 130, 64, True, BF, F32), (16, 64, 128, False, F32, F32)])
def test_quantize_and_dequantize(dev, N, K, group, zeros, sdt, dtype):
    """The rounding against the same formula in torch: scales and zero points equal, every value within half a
    step of its own (the clamp at an end of the range, after the scale's own rounding, may add what that
    rounding moved the end by), and dequantize equal to scale * (code - zero) rounded once."""
    _say("quantize", N, K, group, zeros, sdt, dtype)
    w = torch.randn(N, K, generator=_gen(N)).to(dtype)
    w[0] = 0  # a row of zeros
    w[1, :group] = 3.0  # a constant group
    q = hm.Weight4Bit.quantize(w.to(dev), group, zero_points=zeros, scale_dtype=sdt)
    groups = -(-K // group)
    pad = torch.zeros(N, groups * group)
    pad[:, :K] = w.float()
    by = pad.view(N, groups, group)
    hi, lo = by.amax(2).clamp_min(0), by.amin(2).clamp_max(0)
    s = ((hi / 15 - lo / 15) if zeros else torch.maximum(hi, -lo) / 7).to(sdt).float()
    assert torch.equal(q.scales[:groups, :N].t().cpu().float(), s)
    assert not q.scales[groups:].any() and not q.scales[:, N:].any()
    z = torch.full_like(s, 8.0)
    if zeros:
        z = torch.where(s > 0, (-lo / s).round().clamp(max=15), 8.0)
        assert torch.equal(q.zeros[:groups, :N].t().cpu().float(), z)
    d = q.dequantize(F32).cpu()
    step = s.repeat_interleave(group, 1)[:, :K]
    # z's own rounding moves the range by up to half a step as well, the scale's rounding by 15 steps' worth of it
    most = step * (0.5 + (0.5 if zeros else 0.0) + 15 * torch.finfo(sdt).eps / 2 + 1e-5)
    assert ((d - w.float()).abs() <= most).all()
    codes = (d / step.clamp_min(1e-30)).round() + z.repeat_interleave(group, 1)[:, :K]
    assert codes.min() >= 0 and codes.max() <= 15
    again = hm.Weight4Bit.from_codes(codes.to(torch.uint8).to(dev), s.to(sdt).to(dev),
                                     z.to(torch.uint8).to(dev) if zeros else None, group)
    assert torch.equal(again.packed, q.packed)
    assert torch.equal(again.dequantize(BF), q.dequantize(F32).to(BF))
    x = torch.randn(3, K, generator=_gen(9)).to(dtype)
    _check_linear(hm.linear_4bit(x.to(dev), q), x, codes, s, z if zeros else None, group, None, None)


def test_weight_refusals(dev):
    codes, scales, z = (t.to(dev) for t in _weight(32, 128, 64, True, BF, 0))
    make = hm.Weight4Bit.from_codes
    with pytest.raises(ValueError, match="0..15"):
        make(codes + 1, scales, z, 64)
    with pytest.raises(ValueError, match="0..15"):
        make(codes, scales, z + 1, 64)
    with pytest.raises(ValueError, match="scales must be"):
        make(codes, scales[:, :1], z, 64)
    with pytest.raises(ValueError, match="zeros must be"):
        make(codes, scales, z[:8], 64)
    with pytest.raises(ValueError, match="group_size"):
        make(codes, scales, z, 48)
    with pytest.raises(TypeError):
        make(codes.int(), scales, z, 64)
    with pytest.raises(TypeError):
        make(codes, scales.half(), z, 64)
    with pytest.raises(ValueError, match="rows and columns"):
        make(codes[:0], scales[:0], None, 64)
    bad = torch.randn(16, 128, device=dev)
    bad[3, 3] = float("inf")
    with pytest.raises(ValueError, match="infinities"):
        hm.Weight4Bit.quantize(bad)
    with pytest.raises(TypeError):
        hm.Weight4Bit.quantize(bad.half())
    w = make(codes, scales, z, 64)
    with pytest.raises(RuntimeError, match="do not hold"):
        hm.Weight4Bit(w.packed, w.scales, w.zeros, (33, 128), 64)
    x = torch.randn(4, 128, device=dev, dtype=BF)
    for other in (copy.deepcopy(w), pickle.loads(pickle.dumps(w)), w.to(dev)):
        assert torch.equal(hm.linear_4bit(x, other), hm.linear_4bit(x, w)) and "32x128" in repr(other)
    with pytest.raises(RuntimeError, match="no CPU path"):
        hm.linear_4bit(x.cpu(), w)
    with pytest.raises(RuntimeError, match="128 columns"):
        hm.linear_4bit(x[:, :64], w)
    with pytest.raises(TypeError):
        hm.linear_4bit(x.half(), w)
    with pytest.raises(RuntimeError, match="bias"):
        hm.linear_4bit(x, w, bias=x[0, :31])
    with pytest.raises(RuntimeError, match="residual"):
        hm.linear_4bit(x, w, residual=x[:, :31])
    with pytest.raises(RuntimeError, match="residual"):
        hm.linear_4bit(x, w, residual=torch.zeros(4, 32, device=dev))
    with pytest.raises(RuntimeError, match="out must be"):
        hm.linear_4bit(x, w, out=torch.zeros(4, 31, device=dev, dtype=BF))
    with pytest.raises(RuntimeError, match="no gradient"):
        hm.linear_4bit(x.float().requires_grad_(), w)
    with pytest.raises(RuntimeError, match="norm_eps"):
        hm.linear_4bit(x, w, norm_eps=-1.0)
    with pytest.raises(RuntimeError, match="norm_eps"):
        hm.linear_4bit(x.float(), w, norm_eps=1e-5)
    buf = torch.zeros(4, 256, device=dev, dtype=BF)
    with pytest.raises(RuntimeError, match="share no other memory"):
        hm.linear_4bit(buf[:, :128], w, out=buf[:, 100:132])
    hm.linear_4bit(buf[:, :128], w, out=buf[:, 128:160])  # other columns of one buffer
    with pytest.raises(RuntimeError, match="share no other memory"):
        hm.linear_4bit(x, w, residual=buf[:, 1:33], out=buf[:, :32])
    with pytest.raises(RuntimeError, match="apart"):
        hm.linear_4bit(x, w, out=torch.zeros(1, 32, device=dev, dtype=BF).expand(4, 32))


# ------------------------------------------------------------------------------- logits
def _processed(l, h, r, f, p, bias, mask):
    """The controls in fp32, one rounding per operation, on the CPU."""
    z = l.float()
    if h is not None:
        h = h.int()
        n = (h & 0x7FFF).float()
        col = lambda t: t[:, None] if isinstance(t, torch.Tensor) else torch.tensor(float(t))  # noqa: E731
        z = torch.where(h != 0, torch.where(z > 0, z / col(r), z * col(r)), z)
        z = z - col(f) * n
        z = z - torch.where(n > 0, col(p), torch.tensor(0.0))
    if bias is not None:
        z = z + bias.float()
    if mask is not None:
        V = l.shape[1]
        at = torch.arange(V)
        m = mask.view(-1, mask.shape[-1])[:, at // 32] >> (at % 32).int() & 1
        z = torch.where(m != 0, z, float("-inf"))
    return z


def _bits(allowed):
    B, V = allowed.shape
    pad = torch.zeros(B, -(-V // 32) * 32, dtype=torch.bool)
    pad[:, :V] = allowed
    return (pad.view(B, -1, 32).long() << torch.arange(32)).sum(-1).to(torch.int32)


def _controls(B, V, seed, dtype, which):
    g = _gen(seed)
    l = (torch.randn(B, V, generator=g) * 3).to(dtype)
    c = dict(history=None, repetition=None, frequency=None, presence=None, bias=None, mask=None)
    if "p" in which:
        h = torch.randint(1, 5, (B, V), generator=g) * (torch.rand(B, V, generator=g) < 0.3)
        h = h | (torch.rand(B, V, generator=g) < 0.2).long() << 15
        h[:, ::97] = 0x7FFF
        c["history"] = (h - ((h >> 15) << 16)).to(torch.int16)
        c["repetition"] = 0.5 + torch.rand(B, generator=g)
        c["frequency"] = torch.rand(B, generator=g) - 0.3
        c["presence"] = torch.rand(B, generator=g) - 0.3
        if B > 1:  # a row without penalties
            c["repetition"][1], c["frequency"][1], c["presence"][1] = 1, 0, 0
    if "b" in which:
        c["bias"] = torch.randn(V, generator=g)
    if "B" in which:
        c["bias"] = torch.randn(B, V, generator=g).to(BF)
    if "m" in which:
        c["mask"] = _bits(torch.rand(B, V, generator=g) < 0.4)
    return l, c


def _on(dev, c):
    return {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in c.items()}


def _plain(l, c):
    return _processed(l, c["history"], 1.0 if c["repetition"] is None else c["repetition"],
                      0.0 if c["frequency"] is None else c["frequency"], 0.0 if c["presence"] is None else c["presence"], c["bias"],
                      c["mask"])


SHAPES = [(1, 1), (1, 7), (3, 8), (2, 33), (4, 1000), (3, 4097), (2, 50277), (1, 131072), (5, 8192)]


@pytest.mark.parametrize("B,V", SHAPES)
@pytest.mark.parametrize("which", ["", "p", "bm", "pBm"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_process_logits(dev, B, V, which, dtype):
    _say("process_logits", B, V, which, dtype)
    l, c = _controls(B, V, V + B, dtype, which)
    want = _plain(l, c).to(dtype)
    d, cd = l.to(dev), _on(dev, c)
    got = hm.process_logits(d, **cd)
    assert torch.equal(got.cpu(), want)
    assert torch.equal(d.cpu(), l)  # the input is left alone
    assert hm.process_logits(d, out=d, **cd) is d and torch.equal(d.cpu(), want)


@pytest.mark.parametrize("B,V", SHAPES + [(300, 513)])
@pytest.mark.parametrize("which", ["", "p", "bm", "pBm"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_select_tokens(dev, B, V, which, dtype):
    """Tokens equal to the fp32 formula's.  Log-probabilities: the sum of up to 256 terms a thread and the
    joins, each term off by less than (1.5 |x| + 3) 2^-24 with |x| at most log V on the softmax's average,
    give 320 2^-24 of the sum; the value, the maximum and the result each add their own rounding."""
    _say("select_tokens", B, V, which, dtype)
    l, c = _controls(B, V, V + B, dtype, which)
    g = _gen(V)
    temp = 0.3 + torch.rand(B, generator=g)
    temp[0] = 0  # a greedy row
    u = torch.rand(B, V, generator=g).clamp(1e-6, 1 - 1e-6)
    noise = -torch.log(-torch.log(u))
    d, cd = l.to(dev), _on(dev, c)
    for t, n in ((None, None), (0.0, noise), (temp, None), (temp, noise)):
        z = _plain(l, c)
        if t is not None:
            tt = (t if isinstance(t, torch.Tensor) else torch.full((B,), t))[:, None]
            z = torch.where(tt > 0, z / torch.where(tt > 0, tt, 1.0), z)
        else:
            tt = torch.ones(B, 1)
        v = z if n is None else torch.where(tt > 0, z + n, z)
        best = v.amax(1, keepdim=True)
        tok = torch.where(v == best, torch.arange(V), V).amin(1)
        none = best[:, 0] == float("-inf")
        lp = z.double().log_softmax(1).gather(1, tok.clamp(max=V - 1)[:, None])[:, 0]
        got, glp = hm.select_tokens(d, temperature=t.to(dev) if isinstance(t, torch.Tensor) else t,
                                    noise=None if n is None else n.to(dev), **cd)
        got, glp = got.cpu(), glp.cpu().double()
        assert torch.equal(got, torch.where(none, -1, tok))
        assert (glp[none] == float("-inf")).all()
        ok = ~none
        at = z.gather(1, tok.clamp(max=V - 1)[:, None])[:, 0].abs()[ok].double() + z.amax(1).abs()[ok].double() + lp[ok].abs()
        assert ((glp[ok] - lp[ok]).abs() <= 320 * 2.0**-24 + 2.0**-23 * at).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_masked_values_do_not_matter(dev, dtype):
    """NaN, infinities and the type's lowest value in masked places leave no trace; a row with nothing allowed
    has no token; an allowed NaN is not chosen and makes the log-probability NaN; ties go to the lowest index."""
    B, V = 6, 9000
    l, c = _controls(B, V, 1, dtype, "m")
    allowed = torch.zeros(B, V, dtype=torch.bool)
    allowed[:, ::3] = True
    allowed[2] = False
    c["mask"] = _bits(allowed)
    l[:, 1::3], l[:, 2::3] = float("nan"), float("inf")
    l[0, 1::3] = torch.finfo(dtype).min
    l[3, 300] = float("nan")
    l[4, 600] = l[4, 6000] = 50.0
    l[5, 0::3] = float("-inf")
    clean = torch.where(allowed, l.float(), float("-inf"))
    got = hm.process_logits(l.to(dev), mask=c["mask"].to(dev)).cpu()
    assert torch.equal(got[:3], clean.to(dtype)[:3]) and torch.equal(got.isnan(), clean.isnan())
    tok, lp = (t.cpu() for t in hm.select_tokens(l.to(dev), mask=c["mask"].to(dev)))
    best = torch.where(clean.isnan(), float("-inf"), clean)
    want = torch.where(best == best.amax(1, keepdim=True), torch.arange(V), V).amin(1)
    want[2] = want[5] = -1
    assert torch.equal(tok, want) and tok[4] == 600
    assert lp[2] == float("-inf") and lp[5] == float("-inf") and lp[3].isnan() and lp[[0, 1, 4]].isfinite().all()


def test_logits_layouts(dev):
    """Rows of a wider buffer at odd offsets, shared rows of bias and mask, penalties as numbers, another
    stream: the values of contiguous operands; what lies outside the rows stays."""
    B, V = 4, 1003
    l, c = _controls(B, V, 5, BF, "pBm")
    cd, d = _on(dev, c), l.to(dev)
    want, pick = hm.process_logits(d, **cd), hm.select_tokens(d, **cd)
    wide = torch.full((B, V + 9), 5.0, dtype=BF, device=dev)
    wide[:, 3:3 + V] = d
    view = wide[:, 3:3 + V]
    h = torch.zeros(B, V + 1, dtype=torch.int16, device=dev)
    h[:, 1:] = cd["history"]
    ck = dict(cd, history=h[:, 1:], bias=cd["bias"].t().contiguous().t())
    assert torch.equal(hm.process_logits(view, **ck), want)
    assert all(torch.equal(a, b) for a, b in zip(hm.select_tokens(view, **ck), pick))
    hm.process_logits(view, out=view, **ck)
    assert torch.equal(view, want) and (wide[:, :3] == 5).all() and (wide[:, 3 + V:] == 5).all()
    shared = dict(cd, repetition=1.25, frequency=0.5, presence=-0.25, bias=cd["bias"][0], mask=cd["mask"][:1])
    plain = _processed(l, c["history"], 1.25, 0.5, -0.25, c["bias"][:1], c["mask"][:1]).to(BF)
    assert torch.equal(hm.process_logits(d, **shared).cpu(), plain)
    assert torch.equal(hm.process_logits(d, **dict(shared, bias=cd["bias"][:1].expand(B, V), mask=cd["mask"][0].expand(B, -1))).cpu(),
                       plain)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = hm.process_logits(d, **cd)
    side.synchronize()
    assert torch.equal(other, want)
    assert hm.process_logits(d[:0], mask=cd["mask"][0]).shape == (0, V)
    assert hm.select_tokens(d[:0])[0].shape == (0,)


def test_logits_refusals(dev):
    B, V = 3, 100
    l = torch.randn(B, V, device=dev)
    h = hm.new_token_history(B, V, dev)
    for kw, match in ((dict(repetition=1.2), "history"), (dict(history=h, repetition=0.0), "above 0"),
                      (dict(history=h, repetition=torch.ones(2, device=dev)), "3 values"), (dict(history=h[:, :99]), "int16 table"),
                      (dict(history=h.int()), "int16 table"), (dict(bias=l[:, :99]), "bias"), (dict(bias=l[:2]), "bias"),
                      (dict(mask=torch.zeros(B, 3, dtype=torch.int32, device=dev)), "mask"),
                      (dict(mask=torch.zeros(B, 4, dtype=torch.int64, device=dev)), "int32"),
                      (dict(history=h.cpu()), "is on cpu")):
        for call in (hm.process_logits, hm.select_tokens):
            with pytest.raises(RuntimeError, match=match):
                call(l, **kw)
    with pytest.raises(TypeError):
        hm.process_logits(l.half())
    with pytest.raises(TypeError):
        hm.process_logits(l, bias=l.half())
    with pytest.raises(RuntimeError, match="sequences, vocabulary"):
        hm.process_logits(l[0])
    with pytest.raises(RuntimeError, match="sequences, vocabulary"):
        hm.select_tokens(l[:, :0])
    with pytest.raises(RuntimeError, match="noise"):
        hm.select_tokens(l, noise=l[:, :50])
    with pytest.raises(RuntimeError, match="noise"):
        hm.select_tokens(l, noise=l.to(BF))
    with pytest.raises(RuntimeError, match="temperature"):
        hm.select_tokens(l, temperature=torch.ones(2, device=dev))
    buf = torch.zeros(B, V + 1, device=dev)
    with pytest.raises(RuntimeError, match="share no other memory"):
        hm.process_logits(buf[:, :V], out=buf[:, 1:])
    with pytest.raises(RuntimeError, match="bias or the mask"):
        hm.process_logits(l, bias=buf[:, :V], out=buf[:, 1:])
    with pytest.raises(RuntimeError, match="out must match"):
        hm.process_logits(l, out=buf)
    with pytest.raises(RuntimeError, match="no gradient"):
        hm.process_logits(l.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="no gradient"):
        hm.select_tokens(l.clone().requires_grad_())


# ------------------------------------------------------------------------------- token history
def _table(B, V, prompt, plen, output, olen, start=None):
    t = torch.zeros(B, V, dtype=torch.long) if start is None else start.long() & 0xFFFF
    for b in range(B):
        for i, v in enumerate(prompt[b].tolist() if prompt is not None else []):
            if i < plen[b] and 0 <= v < V:
                t[b, v] |= 0x8000
        for i, v in enumerate(output[b].tolist() if output is not None else []):
            if i < olen[b] and 0 <= v < V and (t[b, v] & 0x7FFF) < 0x7FFF:
                t[b, v] += 1
    return (t - ((t >> 15) << 16)).to(torch.int16)


@pytest.mark.parametrize("B,V,P,O", [(1, 1, 3, 3), (2, 10, 50, 0), (3, 4096, 0, 40), (2, 4097, 300, 100), (1, 50277, 700, 17),
                                     (4, 9000, 64, 257)])
def test_token_history(dev, B, V, P, O):
    _say("token history", B, V, P, O)
    g = _gen(V + P)
    prompt = torch.randint(-2, V + 3, (B, P), generator=g)  # ids outside the vocabulary are passed over
    output = (torch.rand(B, O, generator=g) ** 4 * V).long()
    plen = torch.randint(0, P + 3, (B,), generator=g)
    olen = torch.randint(-2, O + 1, (B,), generator=g)
    full = torch.full((B, V + 3), 77, dtype=torch.int16, device=dev)
    table = full[:, 1:1 + V]
    hm.fill_token_history(table, prompt.to(dev), plen.to(dev), output.to(dev), olen.int().to(dev))
    want = _table(B, V, prompt, plen, output, olen)
    assert torch.equal(table.cpu(), want)
    assert (full[:, 0] == 77).all() and (full[:, 1 + V:] == 77).all()
    for T in (1, 3, 16, 17, 40):  # single entries and the slice-wise count
        more = (torch.rand(B, T, generator=g) ** 4 * (V + 1)).long() - 1
        hm.append_tokens(table, more.to(dev) if T > 1 else more[:, 0].to(dev))
        want = _table(B, V, None, None, more, [T] * B, want)
        assert torch.equal(table.cpu(), want), T
    n = torch.randint(0, 4, (B,), generator=g)
    hm.append_tokens(table, more[:, :5].to(dev), n.to(dev))
    assert torch.equal(table.cpu(), _table(B, V, None, None, more[:, :5], n, want))
    assert (full[:, 0] == 77).all() and (full[:, 1 + V:] == 77).all()
    hm.fill_token_history(table)
    assert not table.any()


def test_token_counts_stop_at_their_largest(dev):
    t = hm.new_token_history(2, 64, dev)
    ids = torch.full((2, 40000), 5, device=dev)
    n = torch.tensor([40000, 32766], device=dev)
    hm.fill_token_history(t, ids[:, :1], None, ids, n)
    assert t[0, 5] == -1 and t[1, 5] == -2  # 0xFFFF, 0xFFFE: prompt bit and count
    for want in (-1, -1):
        hm.append_tokens(t, ids[:, 0])
        assert t[0, 5] == -1 and t[1, 5] == want
    hm.append_tokens(t, ids[:, :100])
    assert t[0, 5] == -1 and t[1, 5] == -1 and int((t != 0).sum()) == 2


def test_history_refusals(dev):
    t = hm.new_token_history(2, 64, dev)
    ids = torch.zeros(2, 4, dtype=torch.long, device=dev)
    with pytest.raises(RuntimeError, match="int16"):
        hm.fill_token_history(t.int(), ids)
    with pytest.raises(RuntimeError, match="token ids"):
        hm.fill_token_history(t, ids[:1])
    with pytest.raises(RuntimeError, match="token ids"):
        hm.fill_token_history(t, ids.float())
    with pytest.raises(RuntimeError, match="lengths"):
        hm.fill_token_history(t, ids, torch.zeros(3, dtype=torch.long, device=dev))
    with pytest.raises(RuntimeError, match="without"):
        hm.fill_token_history(t, prompt_lengths=torch.zeros(2, dtype=torch.long, device=dev))
    with pytest.raises(RuntimeError, match="is on cpu"):
        hm.append_tokens(t, torch.zeros(2, dtype=torch.long))
    with pytest.raises(RuntimeError, match="contiguous rows"):
        hm.append_tokens(t.t(), torch.zeros(64, dtype=torch.long, device=dev))


# ------------------------------------------------------------------------------- graphs
def test_recorded_step_matches_eager(dev):
    """A head product, the choice under all controls and the history's update recorded as one graph: every
    replay equals the eager calls on copies, with eager work and synchronisations between."""
    B, K, V = 4, 256, 1003
    codes, scales, z = (t.to(dev) for t in _weight(V, K, 64, True, BF, 2))
    w = hm.Weight4Bit.from_codes(codes, scales, z, 64)
    _, c = _controls(B, V, 3, BF, "pBm")
    c = _on(dev, c)
    x, noise = torch.randn(B, K, device=dev).to(BF), torch.zeros(B, V, device=dev)
    temp = torch.tensor([0.7, 0.0, 1.3, 1.0], device=dev)

    def step(c):
        tok, lp = hm.select_tokens(hm.linear_4bit(x, w), temperature=temp, noise=noise, **c)
        hm.append_tokens(c["history"], tok)
        return tok, lp

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step(dict(c, history=c["history"].clone()))
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(c)
    eager = dict(c, history=c["history"].clone())
    for i in range(6):
        x.copy_(torch.randn(B, K, generator=_gen(i)))
        noise.copy_(torch.rand(B, V, generator=_gen(i + 50)))
        want = step(eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i
        assert torch.equal(c["history"], eager["history"]), i


def test_row_sums_follow_the_weight(dev):
    """A loaded state dict changes the weight in place: norm_eps uses the new weight's row sums, eagerly and, the module
    having loaded it, in a graph recorded before."""
    one, two = (torch.nn.Linear(256, 96, bias=False, device=dev, dtype=BF) for _ in range(2))
    layer, other = hm.Linear4Bit.from_linear(one, 64), hm.Linear4Bit.from_linear(two, 64)
    x = (torch.randn(5, 256, generator=_gen(1)) + 2).to(BF).to(dev)
    with torch.no_grad():
        want = hm.linear_4bit(x, other.weight4, norm_eps=1e-5)
        hm.linear_4bit(x, layer.weight4, norm_eps=1e-5)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = hm.linear_4bit(x, layer.weight4, norm_eps=1e-5)
        layer.load_state_dict(other.state_dict())
        for _ in range(3):
            out.zero_()
            graph.replay()
            assert torch.equal(out, want)
            assert torch.equal(hm.linear_4bit(x, layer.weight4, norm_eps=1e-5), want)
        w = hm.Weight4Bit.quantize(one.weight, 64)
        for name in ("packed", "scales"):  # by hand
            getattr(w, name).copy_(getattr(other.weight4, name))
        assert torch.equal(hm.linear_4bit(x, w, norm_eps=1e-5), want)


def test_shared_memory_is_refused(dev):
    w = hm.Weight4Bit.quantize(torch.randn(32, 64, generator=_gen(5)).to(dev), 32)
    out = torch.zeros(3, 32, device=dev)
    with torch.no_grad(), pytest.raises(RuntimeError, match="memory"):
        hm.linear_4bit(torch.zeros(3, 64, device=dev), w, bias=out[1], out=out)
    logits, table = torch.zeros(4, 64, device=dev), torch.zeros(4, 64, device=dev, dtype=torch.int16)
    out = torch.zeros(4, 64, device=dev)
    with pytest.raises(RuntimeError, match="memory"):
        hm.process_logits(logits, history=table, repetition=out[2, :4], out=out)
    with pytest.raises(RuntimeError, match="memory"):
        hm.process_logits(logits, history=out.view(torch.int16)[:, :64], presence=1.0, out=out)
    with pytest.raises(RuntimeError, match="memory"):
        hm.process_logits(logits, bias=out[0], out=out)


@pytest.mark.parametrize("rows", [2, 500])
def test_linear4bit_module_has_no_gradient(dev, rows):
    layer = hm.Linear4Bit.from_linear(torch.nn.Linear(64, 32, device=dev), 32)
    x = torch.randn(rows, 64, device=dev, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        layer(x)
    assert not layer(x.detach()).requires_grad


def test_history_passes_over_any_other_id(dev):
    far = [-(2**63), 2**63 - 1, -1, 40, 2**32 + 3, -(2**32) + 3]
    table = hm.new_token_history(1, 40, dev)
    hm.fill_token_history(table, prompt=torch.tensor([far + [3]], device=dev), output=torch.tensor([far + [5, 5]], device=dev))
    want = torch.zeros(40, dtype=torch.int16)
    want[3], want[5] = -(2**15), 2
    assert torch.equal(table[0].cpu(), want)
    hm.append_tokens(table, torch.tensor([far + [3]], device=dev))
    hm.append_tokens(table, torch.tensor([far * 3 + [3]], device=dev))
    want[3] = -(2**15) + 2
    assert torch.equal(table[0].cpu(), want)


def test_many_rows(dev):
    """More rows than a grid has blocks in y: process_logits walks them, select_tokens refuses them; a product's are row
    blocks."""
    B, V = 70000, 9
    l = torch.randn(B, V, generator=_gen(1)).to(dev)
    bias = torch.randn(V, generator=_gen(2)).to(dev)
    assert torch.equal(hm.process_logits(l, bias=bias), l + bias)
    with pytest.raises(_ops.HdcmError):
        hm.select_tokens(l)
    token, _ = hm.select_tokens(l[:65535])
    assert torch.equal(token, l[:65535].argmax(1))
    for dtype in (BF, F32):
        codes, scales, _ = _weight(16, 40, 32, False, BF, seed=3)
        w = hm.Weight4Bit.from_codes(codes.to(dev), scales.to(dev), None, 32)
        x = torch.randn(B, 40, generator=_gen(4)).to(dtype)
        _check_linear(hm.linear_4bit(x.to(dev), w), x, codes, scales, None, 32, None, None)


def test_two_streams_at_once(dev):
    """Calls in flight on two streams share nothing."""
    V = 50000
    w = hm.Weight4Bit.quantize(torch.randn(V // 10, 512, generator=_gen(1)).to(dev), 64)
    jobs = [(torch.randn(8, V, generator=_gen(s)).to(dev), torch.randn(8, 512, generator=_gen(s)).to(BF).to(dev)) for s in (2, 3)]
    want = [(hm.select_tokens(l), hm.linear_4bit(x, w, norm_eps=1e-5)) for l, x in jobs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(50):
        for i, (l, x) in enumerate(jobs):
            with torch.cuda.stream(streams[i]):
                got[i].append((hm.select_tokens(l), hm.linear_4bit(x, w, norm_eps=1e-5)))
    torch.cuda.synchronize()
    for i in range(2):
        for (token, logprob), y in got[i]:
            assert torch.equal(token, want[i][0][0]) and torch.equal(logprob, want[i][0][1]) and torch.equal(y, want[i][1])


def test_graphs_share_no_workspace(dev):
    """Two recorded graphs of the same calls, replayed in turn and at once on two streams."""
    V = 40000
    w = hm.Weight4Bit.quantize(torch.randn(2000, 640, generator=_gen(1)).to(dev))
    x = [torch.randn(5, 640, generator=_gen(s)).to(BF).to(dev) for s in (2, 3)]
    l = [torch.randn(5, V, generator=_gen(s)).to(dev) for s in (4, 5)]
    want = [(hm.select_tokens(l[i]), hm.linear_4bit(x[i], w, norm_eps=1e-5)) for i in range(2)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append((hm.select_tokens(l[i]), hm.linear_4bit(x[i], w, norm_eps=1e-5)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for n in range(6):
        for (token, logprob), y in outs:
            token.zero_(), logprob.zero_(), y.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            if n % 2:
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
            else:
                graphs[i].replay()
        torch.cuda.synchronize()
        for ((token, logprob), y), ((t, p), z) in zip(outs, want):
            assert torch.equal(token, t) and torch.equal(logprob, p) and torch.equal(y, z)


# ------------------------------------------------------------------------------- row sums of norm_eps
def _norm_weights(dev):
    """Rows with a mean, a weight and another of its shape, and the other's product behind a LayerNorm."""
    one, two = (hm.Weight4Bit.quantize(torch.randn(96, 256, generator=_gen(s)).to(BF).to(dev), 64, True) for s in (1, 2))
    x = (torch.randn(5, 256, generator=_gen(3)) + 2).to(BF).to(dev)
    return x, one, two, hm.linear_4bit(x, two, norm_eps=1e-5)


def _write(to, other):
    for name in ("packed", "scales", "zeros"):
        getattr(to, name).copy_(getattr(other, name))


def test_row_sums_are_finished_for_every_stream(dev):
    """A weight is written in place and both streams are past that: the first call forms the row sums behind a busy
    stream, the second, on another one, must not read them unwritten.  The same for a module that was moved."""
    x, w, other, want = _norm_weights(dev)
    hm.linear_4bit(x, w, norm_eps=1e-5)
    layer = hm.Linear4Bit(w)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for moved in (False, True):
        _write(w, other)
        if moved:
            layer.cpu().to(dev)
        torch.cuda.synchronize()
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                if i == 0:
                    torch.cuda._sleep(20_000_000)
                got.append(hm.linear_4bit(x, layer.weight4 if moved else w, norm_eps=1e-5))
        torch.cuda.synchronize()
        assert torch.equal(got[0], want) and torch.equal(got[1], want), moved
        w.scales.zero_()
        hm.linear_4bit(x, w, norm_eps=1e-5)


def test_row_sums_are_not_left_to_a_recording(dev):
    """The first call after a write is one being recorded: refused, and no later call takes the sums for formed."""
    x, w, other, want = _norm_weights(dev)
    hm.linear_4bit(x, w, norm_eps=1e-5)
    _write(w, other)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="recording"), torch.cuda.graph(torch.cuda.CUDAGraph()):
        hm.linear_4bit(x, w, norm_eps=1e-5)
    assert torch.equal(hm.linear_4bit(x, w, norm_eps=1e-5), want)
    w.scales.mul_(2)
    w.refresh()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = hm.linear_4bit(x, w, norm_eps=1e-5)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, hm.linear_4bit(x, w, norm_eps=1e-5))
        torch.cuda.synchronize()


def test_row_sums_follow_writes_under_inference_mode(dev):
    x, w, other, want = _norm_weights(dev)
    with torch.inference_mode():
        made = hm.Weight4Bit.quantize(torch.randn(96, 256, generator=_gen(1)).to(BF).to(dev), 64, True)
        clones = hm.Weight4Bit(w.packed.clone(), w.scales.clone(), w.zeros.clone(), w.shape, w.group_size)
        assert clones.packed.is_inference()
        for v in (made, clones):
            hm.linear_4bit(x, v, norm_eps=1e-5)
            _write(v, other)
            assert torch.equal(hm.linear_4bit(x, v, norm_eps=1e-5), want)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = hm.linear_4bit(x, clones, norm_eps=1e-5)
        for factor in (1, 2, 4):  # scales by powers of two: the normalised product likewise
            clones.scales.copy_(other.scales * factor)
            graph.replay()
            assert torch.equal(out, want * factor)
            torch.cuda.synchronize()
    made.scales.mul_(2)
    assert torch.equal(hm.linear_4bit(x, made, norm_eps=1e-5), want * 2)


# ------------------------------------------------------------------------------- gradients
def test_controls_that_need_a_gradient_are_refused(dev):
    B, V = 2, 40
    l, h = torch.zeros(B, V, device=dev), hm.new_token_history(B, V, dev)
    need = lambda *n: torch.ones(*n, device=dev, requires_grad=True)  # noqa: E731
    for kw in (dict(history=h, repetition=need(B)), dict(history=h, frequency=need(B)), dict(history=h, presence=need(B)),
               dict(bias=need(V)), dict(temperature=need(B)), dict(noise=need(B, V))):
        with pytest.raises(RuntimeError, match="no gradient"):
            hm.select_tokens(l, **kw)
        with torch.no_grad():
            hm.select_tokens(l, **kw)
        if "temperature" not in kw and "noise" not in kw:
            with pytest.raises(RuntimeError, match="no gradient"):
                hm.process_logits(l, **kw)


def test_tangents_are_refused(dev):
    """Forward mode: no operator drops a tangent, whatever the number of rows and with backward mode off."""
    from torch.autograd import forward_ad

    B, V = 2, 40
    l, h = torch.zeros(B, V, device=dev), hm.new_token_history(B, V, dev)
    layer = hm.Linear4Bit.from_linear(torch.nn.Linear(64, V, device=dev), 32)
    with forward_ad.dual_level(), torch.no_grad():
        dual = lambda *n: forward_ad.make_dual(torch.ones(*n, device=dev), torch.ones(*n, device=dev))  # noqa: E731
        for call in (lambda: hm.process_logits(dual(B, V)), lambda: hm.process_logits(l, history=h, presence=dual(B)),
                     lambda: hm.select_tokens(l, temperature=dual(B)), lambda: hm.select_tokens(l, noise=dual(B, V)),
                     lambda: hm.linear_4bit(dual(3, 64), layer.weight4),
                     lambda: hm.linear_4bit(torch.ones(3, 64, device=dev), layer.weight4, residual=dual(3, V)),
                     lambda: layer(dual(3, 64)), lambda: layer(dual(500, 64))):
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
        assert layer(torch.ones(500, 64, device=dev)).shape == (500, V)


def test_linear4bit_module_under_autocast(dev):
    """One result type on both sides of direct_rows, nn.Linear's; values those of rows cast beforehand."""
    linear = torch.nn.Linear(64, 40, device=dev)
    layer = hm.Linear4Bit.from_linear(linear, 32)
    x = torch.randn(layer.direct_rows + 1, 64, generator=_gen(1)).to(dev)
    with torch.no_grad():
        for rows in (1, layer.direct_rows, layer.direct_rows + 1):
            want = layer(x[:rows].to(BF))
            with torch.amp.autocast("cuda", dtype=BF):
                got = layer(x[:rows])
                assert got.dtype == linear(x[:rows]).dtype == BF and torch.equal(got, want)
                with torch.amp.autocast("cuda", enabled=False):
                    assert layer(x[:rows]).dtype == F32
            with torch.amp.autocast("cuda", dtype=torch.float16), pytest.raises(TypeError, match="dtype"):
                layer(x[:rows])


# ------------------------------------------------------------------------------- where a weight is held
def test_weight_and_module_on_the_cpu(dev):
    """A weight and a module that were moved to the CPU hold no GPU memory, are copied, saved and loaded there (also what was
    saved on the GPU), refuse to compute, and moved back give the same products."""
    import io

    N, K = 4096, 1024
    x = torch.randn(3, K, generator=_gen(1)).to(BF).to(dev)
    linear = torch.nn.Linear(K, N, device=dev, dtype=BF)
    layer = hm.Linear4Bit.from_linear(linear, 64, zero_points=True)
    want, normed = layer(x), hm.linear_4bit(x, layer.weight4, norm_eps=1e-5)
    torch.cuda.synchronize()
    size = layer.packed.numel()
    files = [io.BytesIO(), io.BytesIO()]
    for f, thing in zip(files, (layer, layer.weight4)):
        torch.save(thing, f)
        assert size < f.tell() < 1.3 * size  # the buffers once
        f.seek(0)
    del thing
    before = torch.cuda.memory_allocated(dev)
    layer.cpu()
    assert before - torch.cuda.memory_allocated(dev) >= size
    with pytest.raises(RuntimeError, match="no CPU path"):
        layer(x.cpu())
    with pytest.raises(RuntimeError, match="no CPU path"):
        hm.linear_4bit(x, layer.weight4)
    copies = [layer, copy.deepcopy(layer), pickle.loads(pickle.dumps(layer)), *(torch.load(f, map_location="cpu", weights_only=False) for f in files)]
    state = hm.Linear4Bit.from_linear(linear, 64, zero_points=True).cpu()
    state.packed.zero_()
    state.load_state_dict(layer.state_dict())
    for c in [*copies, state]:
        assert c.packed.device.type == "cpu" and torch.equal(c.packed, layer.packed if c is not layer else c.packed)
    layer.to(dev)
    for c in copies[1:] + [state]:
        c = c.to(dev)
        w = c if isinstance(c, hm.Weight4Bit) else c.weight4
        assert torch.equal(hm.linear_4bit(x, w, bias=linear.bias.detach()), want)
        assert torch.equal(hm.linear_4bit(x, w, norm_eps=1e-5), normed)
    assert torch.equal(layer(x), want)
    layer.cpu().to(dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # the first product after a move
        out = hm.linear_4bit(x, layer.weight4, norm_eps=1e-5)
    graph.replay()
    assert torch.equal(out, normed)


@pytest.mark.parametrize("V", [5, 3000, 50277])
def test_log_probabilities_of_large_logits(dev, V):
    """Logits far from 0, and small temperatures: the sum as in test_select_tokens, 320 2^-24 of it; the difference to the
    largest logit and the result rounded once each.  Nothing is rounded at the logits' own magnitude."""
    g = _gen(V)
    l = torch.randn(4, V, generator=g) * 2 + torch.tensor([5000.0, -20000.0, 3.0, 1e6])[:, None]
    noise = -torch.log(-torch.log(torch.rand(4, V, generator=g).clamp(1e-6, 1 - 1e-6)))
    temp = torch.tensor([1.0, 0.9, 0.003, 2.0])
    for n in (None, noise):
        tok, lp = (t.cpu() for t in hm.select_tokens(l.to(dev), temperature=temp.to(dev), noise=None if n is None else n.to(dev)))
        t = l / temp[:, None]
        assert torch.equal(tok, (t if n is None else t + n).argmax(1))
        want = t.double().log_softmax(1).gather(1, tok[:, None])[:, 0]
        below = (t.amax(1) - t.gather(1, tok[:, None])[:, 0]).double()
        assert ((lp.double() - want).abs() <= 320 * 2.0**-24 + 2.0**-23 * (below + want.abs())).all()


def test_writes_into_given_memory_are_counted(dev):
    """out= and the history table: a write is seen by autograd's check of the tensors it saved, as torch's own are."""
    w = hm.Weight4Bit.quantize(torch.randn(40, 64, generator=_gen(5)).to(dev), 32)
    x, leaf = torch.ones(3, 64, device=dev), torch.zeros(3, 40, device=dev, requires_grad=True)
    for write in (lambda t: hm.process_logits(t, bias=torch.ones(40, device=dev), out=t), lambda t: hm.linear_4bit(x, w, out=t),
                  lambda t: hm.linear_4bit(x, w, residual=t, out=t)):
        y = leaf.exp()  # saved for its own gradient
        with torch.no_grad():
            assert write(y.detach()).data_ptr() == y.data_ptr()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    table = hm.new_token_history(3, 40, dev)
    for write in (lambda: hm.fill_token_history(table), lambda: hm.append_tokens(table, torch.zeros(3, dtype=torch.long, device=dev))):
        before = table._version
        write()
        assert table._version > before
    with torch.inference_mode():
        t = torch.zeros(3, 40, device=dev)
        assert hm.process_logits(t, out=t) is t


def test_a_weight_whose_buffer_was_replaced_is_refused(dev):
    """A buffer with another storage under it (t.data = other) is checked again at every use."""
    x = torch.zeros(2, 128, device=dev, dtype=BF)
    for name, other, match in (("packed", lambda t: t[:1024].clone(), "do not hold"), ("scales", lambda t: t[:1].clone(), "do not hold"),
                               ("scales", lambda t: t.t().contiguous().t(), "do not hold"), ("zeros", lambda t: t[:1].clone(), "one byte"),
                               ("packed", lambda t: t.cpu(), "cpu")):
        w = hm.Weight4Bit.quantize(torch.randn(64, 128, generator=_gen(5)).to(dev), 32, True)
        t = getattr(w, name)
        t.data = other(t)
        for call in (lambda: hm.linear_4bit(x, w), lambda: hm.linear_4bit(x, w, norm_eps=1e-5), lambda: w.dequantize(), w.refresh):
            with pytest.raises(RuntimeError, match=match):
                call()
    x, w, other, want = _norm_weights(dev)
    for name in ("packed", "scales", "zeros"):  # of the same size: the weight is the other, and so are its row sums
        getattr(w, name).data = getattr(other, name).clone()
    assert torch.equal(hm.linear_4bit(x, w, norm_eps=1e-5), want)


@pytest.mark.parametrize("which", ["frequency", "presence"])
@pytest.mark.parametrize("per_row", [False, True])
def test_infinite_penalties_ban_the_output(dev, which, per_row):
    """Tokens of the output become -inf; what lies beside them, prompt tokens among it, keeps its logit."""
    B, V = 2, 40
    l = torch.randn(B, V, generator=_gen(1))
    l[:, 3] = 9
    prompt, output = torch.tensor([[3, 4, 30], [3, 7, 31]]), torch.tensor([[5, 30, 30], [3, 5, 22]])
    table = hm.fill_token_history(hm.new_token_history(B, V, dev), prompt.to(dev), None, output.to(dev))
    kw = {"history": table, which: torch.full((B,), float("inf"), device=dev) if per_row else float("inf")}
    want = l.scatter(1, output, float("-inf"))
    assert torch.equal(hm.process_logits(l.to(dev), **kw).cpu(), want)
    token, lp = hm.select_tokens(l.to(dev), **kw)
    assert torch.equal(token.cpu(), want.argmax(1)) and lp.isfinite().all()


def test_a_move_to_the_same_place_keeps_the_weight(dev):
    """... which a recording reads: a state dict loaded after it reaches the recording."""
    x, one, two, want = _norm_weights(dev)
    layer = hm.Linear4Bit(one)
    hm.linear_4bit(x, layer.weight4, norm_eps=1e-5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = hm.linear_4bit(x, layer.weight4, norm_eps=1e-5)
    assert layer.to(dev).weight4 is one
    layer.load_state_dict(hm.Linear4Bit(two).state_dict())
    graph.replay()
    assert torch.equal(out, want)
