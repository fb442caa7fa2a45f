"""4-bit products whose results are known exactly: small whole rows, scales of powers of two, so that every fp32 sum in any
order is exact and the result is the exact one rounded once.  A lost or doubled group, tile, segment or wave, or a wrong
zero point, shows in the value itself, however long the rows are.

Magnitudes: |x| <= 2, 16 + c <= 31, scales 1/2 to 2: sums stay below 2 * 31 * 2 * K = 124 K in steps of 1/2, under
2^24 steps up to K = 67000."""
import pytest
import torch

import hdcmamba_amd as hm

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _weight(N, K, group, zeros, sdt, seed):
    g = _gen(seed)
    n = -(-K // group)
    codes = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8)
    scales = 2.0 ** torch.randint(-1, 2, (N, n), generator=g)
    z = torch.randint(0, 16, (N, n), generator=g, dtype=torch.uint8) if zeros else None
    wide = lambda t: t.double().repeat_interleave(group, 1)[:, :K]  # noqa: E731
    dense = (codes.double() - (wide(z) if zeros else 8.0)) * wide(scales)
    return codes, scales.to(sdt), z, dense


def _pack(dev, codes, scales, z, group):
    return hm.Weight4Bit.from_codes(codes.to(dev), scales.to(dev), None if z is None else z.to(dev), group)


# every way through the rules: row tiles and blocks, one or two column tiles a wave, segments of K, ends of every kind
CASES = [
    (1, 128, 16, 128), (1, 1152, 1024, 128), (1, 1000, 9000, 32), (2, 2048, 8208, 64), (1, 2049, 77, 128), (1, 9000, 50, 64),
    (3, 768, 3264, 64), (16, 2048, 8576, 128), (16, 3100, 200, 32), (17, 832, 300, 128), (24, 3000, 500, 64), (32, 4096, 96, 128),
    (33, 768, 5003, 32), (40, 2048, 1000, 128), (50, 3000, 70, 32), (64, 2176, 2048, 64), (64, 4352, 4096, 128), (64, 300, 20000, 128),
    (65, 384, 130, 128), (90, 100, 3000, 64), (128, 1200, 3000, 128), (129, 128, 4200, 64), (200, 6200, 77, 128), (384, 2048, 800, 32),
    (2, 9000, 8200, 128), (41, 8300, 4200, 64), (300, 3300, 5200, 128), (5, 20000, 40, 32), (70, 12345, 33, 128)]


@pytest.mark.parametrize("M,K,N,group", CASES)
@pytest.mark.parametrize("dtype,sdt,zeros", [(BF, BF, False), (BF, F32, True), (F32, BF, True)])
def test_exact_products(dev, M, K, N, group, dtype, sdt, zeros):
    print("exact", M, K, N, group, dtype, sdt, zeros, flush=True)
    codes, scales, z, dense = _weight(N, K, group, zeros, sdt, K + N)
    g = _gen(M)
    x = torch.randint(-2, 3, (M, K), generator=g).double()
    bias, res = (torch.randint(-50, 51, s, generator=g).double() for s in ((N,), (M, N)))
    w = _pack(dev, codes, scales, z, group)
    ref = x @ dense.t()
    xd, bd, rd = (t.to(dtype).to(dev) for t in (x, bias, res))
    assert torch.equal(hm.linear_4bit(xd, w).cpu(), ref.to(dtype))
    assert torch.equal(hm.linear_4bit(xd, w, bias=bd, residual=rd).cpu(), (ref + bias + res).to(dtype))


@pytest.mark.parametrize("K,N", [(128, 16), (2048, 500), (7000, 300)])
def test_exact_products_of_long_fp32_mantissas(dev, K, N):
    """Every bit of an fp32 row counts: one value of 24 bits a row, weights that are powers of two; then 64 values of 12 bits."""
    g = _gen(K)
    codes = (8 + 2 ** torch.randint(0, 3, (N, K), generator=g)).to(torch.uint8)
    scales = 2.0 ** torch.randint(-1, 2, (N, -(-K // 64)), generator=g)
    dense = (codes.double() - 8) * scales.double().repeat_interleave(64, 1)[:, :K]
    w = _pack(dev, codes, scales, None, 64)
    for M in (1, 5, 33):
        x = torch.zeros(M, K, dtype=torch.double)
        x[torch.arange(M), torch.randint(0, K, (M,), generator=g)] = (torch.randint(2**23, 2**24, (M,), generator=g) | 1).double()
        assert torch.equal(hm.linear_4bit(x.float().to(dev), w).cpu().double(), x @ dense.t())
        x = torch.zeros(M, K, dtype=torch.double)
        x.scatter_(1, torch.stack([torch.randperm(K, generator=g)[:64] for _ in range(M)]),
                   torch.randint(-4095, 4096, (M, 64), generator=g).double())
        assert torch.equal(hm.linear_4bit(x.float().to(dev), w).cpu().double(), x @ dense.t())


@pytest.mark.parametrize("M,K,N,group", [c for c in CASES if c[1] >= 8])
@pytest.mark.parametrize("zeros", [False, True])
def test_layer_norm_of_whole_rows(dev, M, K, N, group, zeros):
    """norm_eps on rows of small whole numbers with a mean: x w, the rows' sums, sums of squares and the weight's sums are exact
    in fp32, so what is left is a handful of roundings (2^-24 each): the mean 1, mean * sum w 2 more, the difference 1; s2 / K 1,
    mean^2 3, their difference and + eps 2 in the variance, half of it in rstd; rstd itself (rsqrtf, 2 ulp) and the product 5.
    No bound grows with K: an rstd or a mean that is off by a percent fails."""
    print("layer norm", M, K, N, group, zeros, flush=True)
    codes, scales, z, dense = _weight(N, K, group, zeros, BF, K + N + 1)
    g = _gen(M + 1)
    # rows with means from -1.5 to 1.5 and unequal deviations
    x = (torch.randint(-2, 3, (M, K), generator=g) * torch.randint(1, 3, (M, 1), generator=g)
         + (torch.rand(M, K, generator=g) < 0.5) * torch.randint(-3, 4, (M, 1), generator=g)).double()
    ref_x = x - x.mean(1, keepdim=True)
    var = (ref_x**2).mean(1, keepdim=True)
    assert (var > 0.1).all()  # no row of one value
    rstd = (var + 1e-5).rsqrt()
    mean = x.mean(1, keepdim=True)
    # from sums that are exact in 64 bits: where x w and sum w are both 0 (one element here) the result is 0, which a sum of
    # normalised values misses by 1e-14
    ref = (x @ dense.t() - mean * dense.sum(1)) * rstd
    got = hm.linear_4bit(x.to(BF).to(dev), _pack(dev, codes, scales, z, group), norm_eps=1e-5).cpu().double()
    u = 2.0**-24
    terms = ((x @ dense.t()).abs() + 4 * (mean * dense.sum(1)).abs()) * rstd
    stat = 0.5 * (4 * (x**2).mean(1, keepdim=True) + 4 * mean**2 + 2 * (var + 1e-5)) / (var + 1e-5)
    tol = 2.0**-8 * ref.abs() + u * (terms + (stat + 5) * ref.abs()) * 1.01
    print("  worst", float(((got - ref).abs() / tol.clamp_min(1e-300)).max()), flush=True)
    assert ((got - ref).abs() <= tol).all()
    # what the bound is worth, on the oracle: an rstd off by a percent, a mean off by a percent, a lost group
    for bad in (ref * 1.01, ref - 0.01 * mean * rstd * dense.sum(1)):
        assert not ((bad - ref).abs() <= tol).all()
    bad = ref_x.clone()
    bad[:, -(K % group or group):] = 0
    assert not (((bad * rstd) @ dense.t() - ref).abs() <= tol).all()


@pytest.mark.parametrize("dtype,largest", [(BF, 2.0**115), (F32, 2.0**120)])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True), (128, False)])
def test_range_of_rows(dev, dtype, largest, group, zeros):
    """Rows at the ends of the documented range: the products of rows times a power of two are the products times it.  (fp32:
    codes of at most 15 times 2^120 times 128 columns would not be finite; these rows' largest sums are 2^6 times smaller.)"""
    K, N = 1000, 70
    codes, scales, z, dense = _weight(N, K, group, zeros, F32, 3)
    w = _pack(dev, codes, scales / 2**20, z, group)
    x = torch.randint(-2, 3, (6, K), generator=_gen(4)).float()
    x[2] = 2  # all of the largest
    x[3, 1:] = 0
    want = hm.linear_4bit(x.to(dtype).to(dev), w).cpu().double()
    assert want.abs().max() > 0
    up = largest / 2 if dtype == BF else largest / 2**7
    assert torch.equal(hm.linear_4bit((x * up).to(dtype).to(dev), w).cpu().double(), want * up)
    down = 2.0**-100
    assert torch.equal(hm.linear_4bit((x * down).to(dtype).to(dev), w).cpu().double(), want * down)
