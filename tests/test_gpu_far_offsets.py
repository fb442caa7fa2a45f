"""Decode-side operators on rows that lie more than 2^32 elements apart and on a weight of more than 2^32 bytes: the values of
operands that lie close together."""
import pytest
import torch

import hdcmamba_amd as hm

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
FAR = 2**32 + 24  # bf16 elements from row to row: 8.6 GB


def _gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.fixture
def far(dev):
    """Columns of a two-row buffer whose rows lie far apart, uninitialised but for what a test writes."""
    buf = torch.empty(FAR + 8192, dtype=BF, device=dev)
    at = [0]

    def place(t):
        """A copy of t [2, n] in the next columns (float32 in twice as many)."""
        n = t.shape[1] * t.element_size() // 2
        n += -n % 8
        v = torch.as_strided(buf, (2, n), (FAR, 1), at[0]).view(t.dtype)[:, :t.shape[1]]
        at[0] += n
        assert at[0] <= 8192 and v.stride(0) * v.element_size() > 2**32
        return v.copy_(t)

    yield place
    del buf
    torch.cuda.empty_cache()


def test_rows_far_apart(dev, far):
    print("linear_4bit", flush=True)
    w = hm.Weight4Bit.quantize(torch.randn(200, 328, generator=_gen(1)).to(dev), 64, True)
    x, r = (torch.randn(2, n, generator=_gen(n)).to(BF).to(dev) for n in (328, 200))
    out = far(torch.zeros_like(r))
    assert torch.equal(hm.linear_4bit(far(x), w, residual=far(r), out=out), hm.linear_4bit(x, w, residual=r))
    assert torch.equal(hm.linear_4bit(far(x), w, norm_eps=1e-5), hm.linear_4bit(x, w, norm_eps=1e-5))
    print("logits", flush=True)
    V = 1000
    l, bias = (torch.randn(2, V, generator=_gen(s)).to(BF).to(dev) for s in (4, 5))
    noise = torch.randn(2, 500, generator=_gen(6)).to(dev)
    table = far(torch.zeros(2, V, dtype=torch.int16, device=dev))
    ids = torch.randint(0, V, (2, 40), generator=_gen(7)).to(dev)
    near = hm.new_token_history(2, V, dev)
    for t in (table, near):
        hm.fill_token_history(t, ids[:, :20], None, ids[:, 20:])
        hm.append_tokens(t, ids[:, 5:9])
        hm.append_tokens(t, ids)
    assert torch.equal(table, near)
    kw = dict(repetition=1.3, frequency=0.4, presence=0.2)
    got = hm.process_logits(far(l), history=table, bias=far(bias), out=far(torch.zeros_like(l)), **kw)
    assert torch.equal(got, hm.process_logits(l, history=near, bias=bias, **kw))
    got = hm.select_tokens(far(l[:, :500]), history=table[:, :500], noise=far(noise), **kw)
    want = hm.select_tokens(l[:, :500], history=near[:, :500], noise=noise, **kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_weight_of_many_bytes(dev):
    """2^20 + 16 rows of 8192 columns, 4.3 GB packed: the rows at the end, packed from codes, rounded, multiplied, brought back."""
    N, K, last = 2**20 + 16, 8192, 48
    print("pack", flush=True)
    codes = torch.randint(0, 16, (N, K), dtype=torch.uint8, device=dev)
    scales = (torch.rand(N, K // 128, device=dev) + 0.5).to(BF)
    x = torch.randn(3, K, generator=_gen(2)).to(BF).to(dev)
    w = hm.Weight4Bit.from_codes(codes, scales)
    end = hm.Weight4Bit.from_codes(codes[-last:], scales[-last:])
    assert w.packed.numel() > 2**32
    del codes, scales
    print("multiply", flush=True)
    assert torch.equal(hm.linear_4bit(x, w)[:, -last:], hm.linear_4bit(x, end))
    print("bring back", flush=True)
    dense = w.dequantize(BF)
    assert torch.equal(dense[-last:], end.dequantize(BF))
    del w
    print("round", flush=True)
    again, end = hm.Weight4Bit.quantize(dense), hm.Weight4Bit.quantize(dense[-last:])
    assert torch.equal(hm.linear_4bit(x, again)[:, -last:], hm.linear_4bit(x, end))
    del dense, again
    torch.cuda.empty_cache()
