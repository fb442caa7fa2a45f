"""Token rows and their gradient, the gradients' norm and clipping on the GPU, against plain forms in 64 bits on the CPU.

Tolerances.  A product or sum in fp32 is off by at most 2^-24 of its value, a sum of m terms in any order by m 2^-24 of the
sum of their magnitudes, and a result rounded to its type by half a step, finfo.eps / 2 of its value.  Squares are
added in 64 bits, so a norm is off by its own rounding.
"""
import math

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

import hdcmamba_amd as hm
from cfgs import reinit_block_

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF, FP = torch.bfloat16, torch.float32


def _say(*a):
    print(*a, flush=True)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make_ids(kind, n, V, seed=0):
    """n token ids on the CPU."""
    g = gen(seed)
    if kind == "uniform":
        return torch.randint(0, V, (n,), generator=g)
    if kind == "text":  # the k-th most frequent token about 1/k as often as the first
        return (torch.exp(torch.rand(n, generator=g, dtype=torch.float64) * math.log(V + 1)).long() - 1).clamp(0, V - 1)
    if kind == "same":
        return torch.full((n,), V // 2)
    if kind == "two":  # two long runs that meet inside a unit
        return torch.where(torch.arange(n) < (n * 3) // 7, V - 1, 0)
    if kind == "none":
        return torch.full((n,), -1)
    if kind == "wild":  # ids that are no rows among ids that are
        ids = torch.randint(0, V, (n,), generator=g)
        bad = torch.tensor([-1, V, V + 1, -(2 ** 31), 2 ** 31 - 1])
        return torch.where(torch.rand(n, generator=g) < 0.4, bad[torch.randint(0, 5, (n,), generator=g)], ids)
    raise ValueError(kind)


def lookup64(ids, w, scale):
    i = ids.long().flatten()
    ok = (i >= 0) & (i < w.shape[0])
    y = torch.zeros(i.numel(), w.shape[1], dtype=torch.float64)
    y[ok] = w.double()[i[ok]] * torch.tensor(scale, dtype=FP).double()
    return y.view(*ids.shape, w.shape[1])


def grad64(ids, dy, V, scale=1.0, padding=None):
    """(the gradient in 64 bits, how far a right one may be off before its last rounding)"""
    i = ids.long().flatten()
    dy = dy.double().reshape(i.numel(), dy.shape[-1])
    ok = (i >= 0) & (i < V)
    if padding is not None:
        ok &= i != padding
    s = torch.tensor(scale, dtype=FP).double()
    dw = torch.zeros(V, dy.shape[1], dtype=torch.float64).index_add_(0, i[ok], dy[ok]) * s
    mag = torch.zeros(V, dy.shape[1], dtype=torch.float64).index_add_(0, i[ok], dy[ok].abs()) * s.abs()
    terms = torch.bincount(i[ok], minlength=V).double()[:, None]
    return dw, (terms + 1) * U * mag


def check_grad(got, ref, before_rounding):
    assert got.shape == ref.shape
    err = (got.double().cpu() - ref).abs()
    tol = before_rounding + half_step(got.dtype) * (ref.abs() + before_rounding) + 1e-40
    assert bool((err <= tol).all()), f"worst error over its bound {(err / tol).max().item():.3f}"


# ------------------------------------------------------------------ lookup
@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("idt", [torch.int64, torch.int32])
@pytest.mark.parametrize("T,D,V", [(0, 64, 10), (1, 1, 1), (1, 2048, 50304), (17, 7, 5), (16, 1024, 333), (1000, 100, 65),
                                   (2500, 333, 1000), (4097, 256, 50277)])
@pytest.mark.parametrize("scale", [1.0, 2.7])
def test_lookup(dev, T, D, V, scale, idt, dtype):
    _say("lookup", T, D, V, scale, idt, dtype)
    w = torch.randn(V, D, generator=gen(1)).to(dtype)
    ids = make_ids("wild" if T > 1 else "uniform", T, V, seed=T).clamp(-2 ** 31, 2 ** 31 - 1).to(idt)
    got = hm.embedding(ids.to(dev), w.to(dev), scale=scale)
    ref = lookup64(ids, w, scale)
    assert got.dtype == dtype and got.shape == (T, D)
    if scale == 1.0:
        assert torch.equal(got.double().cpu(), ref)
    else:
        assert bool(((got.double().cpu() - ref).abs() <= ref.abs() * (U + half_step(dtype) * (1 + U))).all())


@pytest.mark.parametrize("dtype", [FP, BF])
def test_lookup_layouts(dev, dtype):
    """Ids of any shape and stride, weights with padded and unaligned rows, values that a product would change."""
    w = torch.randn(40, 70, generator=gen(2)).to(dtype).to(dev)
    w[3, :4] = torch.tensor([float("inf"), float("nan"), -0.0, torch.finfo(dtype).tiny / 4])
    ids = make_ids("uniform", 6 * 9, 40).view(6, 9).to(dev)
    ids[0, 0] = 3
    for i in (ids, ids[:, :-1], ids.t(), ids[2, 3], ids[:, :0], ids[None, ::2, :, None]):
        got = hm.embedding(i, w)
        assert got.shape == (*i.shape, 70)
        assert torch.equal(got.view(torch.int16 if dtype == BF else torch.int32),
                           w[i].contiguous().view(torch.int16 if dtype == BF else torch.int32))
    for v in (w[:, 1:], w[5:, 3:36], w[::2], w.t(), w[:1]):
        i = ids % v.shape[0]
        assert torch.equal(hm.embedding(i, v).nan_to_num(7), v[i].nan_to_num(7))
    big = torch.tensor([0, 2 ** 40, -(2 ** 63), 2 ** 32 + 1, 2 ** 63 - 1], device=dev)
    got = hm.embedding(big, w, scale=float("inf"))
    assert bool(got[1:].eq(0).all()) and bool(got[0].isinf().all())


# ------------------------------------------------------------------ its gradient
SIZES = [(1, 1, 1, 1), (1, 31, 8, 10), (1, 32, 8, 10), (1, 33, 520, 40), (3, 64, 7, 511), (2, 100, 333, 512), (1, 2047, 64, 513),
         (1, 2048, 40, 1000), (5, 410, 256, 65), (2, 3001, 96, 50277), (1, 9000, 1030, 700)]


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("kind", ["uniform", "text", "same", "two", "none", "wild"])
@pytest.mark.parametrize("B,L,D,V", SIZES)
def test_gradient(dev, B, L, D, V, kind, dtype):
    _say("gradient", B, L, D, V, kind, dtype)
    ids = make_ids(kind, B * L, V, seed=L + V).view(B, L)
    dy = torch.randn(B, L, D, generator=gen(L)).to(dtype)
    got = hm.embedding_grad(ids.to(dev), dy.to(dev), V)
    assert got.dtype == dtype and got.is_contiguous()
    check_grad(got, *grad64(ids, dy, V))
    again = hm.embedding_grad(ids.to(dev).int(), dy.to(dev), V)
    assert torch.equal(got, again)  # the same order of every sum


@pytest.mark.parametrize("T,D,V,kind", [(300000, 8, 65, "text"), (300000, 4, 300000, "uniform"), (270000, 16, 2 ** 20 + 3, "text"),
                                        (131072, 40, 50304, "same"), (20000, 24, 2 ** 18 - 1, "wild"), (20000, 24, 2 ** 18, "text")])
def test_gradient_of_many_positions(dev, T, D, V, kind):
    """More positions than one round of the sorting workgroups, and vocabularies of one to three passes."""
    _say("gradient of many", T, D, V, kind)
    ids = make_ids(kind, T, V, seed=3)
    dy = torch.randn(T, D, generator=gen(4)).to(BF)
    check_grad(hm.embedding_grad(ids.to(dev), dy.to(dev), V), *grad64(ids, dy, V))


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("odt", [FP, BF])
@pytest.mark.parametrize("T,D,V", [(5, 12, 30), (700, 130, 90), (6000, 72, 2000)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient_into(dev, T, D, V, accumulate, odt, dtype):
    """Scale, padding index, and a given output of either type, with its other columns and rows as they were."""
    _say("gradient into", T, D, V, accumulate, odt, dtype)
    ids = make_ids("text", T, V, seed=T)
    ids[::7] = V // 3
    dy = torch.randn(T, D, generator=gen(6)).to(dtype)
    whole = torch.randn(V + 2, D + 11, generator=gen(7)).to(odt)
    buf = whole.to(dev)
    out = buf[1:V + 1, 3:D + 3]
    version = buf._version
    got = hm.embedding_grad(ids.to(dev), dy.to(dev), V, scale=0.37, padding_idx=V // 3 - V, out=out, accumulate=accumulate)
    assert got.data_ptr() == out.data_ptr() and buf._version > version
    ref, off = grad64(ids, dy, V, 0.37, V // 3)
    old = whole[1:V + 1, 3:D + 3].double()
    if accumulate:
        named = (torch.bincount(ids, minlength=V) > 0) & (torch.arange(V) != V // 3)
        assert torch.equal(out.cpu()[~named], whole[1:V + 1, 3:D + 3][~named])
        ref, off = ref + old, off + U * (ref.abs() + old.abs() + off)
    check_grad(out, ref, off)
    rest = torch.ones_like(whole, dtype=torch.bool)
    rest[1:V + 1, 3:D + 3] = False
    assert torch.equal(buf.cpu()[rest], whole[rest])


@pytest.mark.parametrize("dtype", [FP, BF])
def test_gradient_layouts(dev, dtype):
    """dy behind a left padding, of every second row, broadcast over rows, positions or all, transposed; ids likewise."""
    B, L, D, V = 3, 50, 36, 20
    ids = make_ids("uniform", B * L, V).view(B, L)
    base = torch.randn(B, 2 * L + 7, D + 5, generator=gen(8)).to(dtype)
    views = lambda t: (t[:, 7:L + 7, :D], t[:, :2 * L:2, 2:D + 2], t[:1, :L, :D].expand(B, L, D), t[:, :1, :D].expand(B, L, D),  # noqa: E731
                       t[:1, :1, :1].expand(B, L, D), t[:, :1, :1].expand(B, L, D), t[:, :L, :1].expand(B, L, D),
                       t[:, :L, :D].transpose(0, 1).contiguous().transpose(0, 1), t[:, :D, :L // 2].transpose(1, 2))
    for dy, on in zip(views(base), views(base.to(dev))):
        i = ids[:, :dy.shape[1]]
        check_grad(hm.embedding_grad(i.to(dev), on, V), *grad64(i, dy, V))
    dy = base[:, :L, :D]
    check_grad(hm.embedding_grad(ids.t().to(dev), dy.to(dev).transpose(0, 1), V), *grad64(ids.t(), dy.transpose(0, 1), V))
    check_grad(hm.embedding_grad(ids.view(B, 5, 10).to(dev), dy.reshape(B, 5, 10, D).to(dev), V), *grad64(ids, dy, V))
    check_grad(hm.embedding_grad(ids[0, 0].to(dev), dy[0, 0].to(dev), V), *grad64(ids[0, 0], dy[0, 0], V))


@pytest.mark.parametrize("T", [511, 512, 513, 8191, 8192, 8193])
@pytest.mark.parametrize("V", [511, 512, 50304])
@pytest.mark.parametrize("dtype", [FP, BF])
def test_gradient_on_either_side_of_its_ways(dev, T, V, dtype):
    """Sizes around the last call that is one launch and the last that one workgroup sorts; the zeros of tokens that do not occur are
    zeros under any scale; accumulating in every way."""
    _say("gradient ways", T, V, dtype)
    D = 520
    ids = make_ids("text", T, V, seed=T)
    dy = torch.randn(T, D, generator=gen(T)).to(dtype)
    for scale in (1.0, -0.5, float("inf")):
        got = hm.embedding_grad(ids.to(dev), dy.to(dev), V, scale=scale).cpu()
        absent = torch.bincount(ids, minlength=V) == 0
        zeros = got[absent]
        assert torch.equal(zeros.view(torch.int32 if dtype == FP else torch.int16), torch.zeros_like(zeros, dtype=torch.int32 if dtype == FP else torch.int16))
        if scale != float("inf"):
            check_grad(got, *grad64(ids, dy, V, scale))
    old = torch.randn(V, D, generator=gen(1)).to(dtype)
    out = old.to(dev)
    hm.embedding_grad(ids.to(dev), dy.to(dev), V, out=out, accumulate=True)
    ref, off = grad64(ids, dy, V)
    assert torch.equal(out.cpu()[absent], old[absent])
    check_grad(out, ref + old.double(), off + U * (ref.abs() + old.double().abs() + off))


def test_rows_past_the_caches(dev):
    """Lookups and gradients of more than the caches hold, and units of 32 positions."""
    T, D, V = 70000, 1030, 40000
    ids, w = make_ids("text", T, V).to(dev), torch.randn(V, D, generator=gen(1)).to(BF).to(dev)
    assert torch.equal(hm.embedding(ids, w), w[ids])
    dy = torch.randn(T, D, generator=gen(2)).to(BF)
    check_grad(hm.embedding_grad(ids, dy.to(dev), V), *grad64(ids.cpu(), dy, V))
    T, D = 540000, 8
    ids = make_ids("two", T, V)
    ids[::3] = make_ids("text", T, V)[::3]
    dy = torch.randn(T, D, generator=gen(3))
    check_grad(hm.embedding_grad(ids.to(dev), dy.to(dev), V), *grad64(ids, dy, V))


@pytest.mark.parametrize("L", [301, 3001])
def test_gradient_layouts_of_many(dev, L):
    """Behind a left padding, broadcast over sequences or positions, added to a given fp32 gradient: sorted by one workgroup and by many."""
    B, D, V = 3, 72, 500
    ids = make_ids("text", B * L, V).view(B, L)
    base = torch.randn(B, L + 9, D + 8, generator=gen(1)).to(BF)
    views = lambda t: (t[:, 9:, :D], t[:1, 9:, 3:D + 3].expand(B, L, D), t[:, :1, :D].expand(B, L, D))  # noqa: E731
    for dy, on in zip(views(base), views(base.to(dev))):
        ref, off = grad64(ids, dy, V)
        check_grad(hm.embedding_grad(ids.to(dev), on, V), ref, off)
        old = torch.randn(V, D, generator=gen(2))
        total = hm.embedding_grad(ids.to(dev), on, V, out=old.to(dev), accumulate=True)
        check_grad(total, ref + old.double(), off + U * (ref.abs() + old.double().abs() + off))


def test_gradient_of_nothing(dev):
    none = torch.zeros(3, 0, dtype=torch.long, device=dev)
    for dtype in (FP, BF):
        got = hm.embedding_grad(none, torch.zeros(3, 0, 40, dtype=dtype, device=dev), 7)
        assert got.shape == (7, 40) and bool(got.eq(0).all())
        old = torch.ones(7, 40, dtype=dtype, device=dev)
        hm.embedding_grad(none, torch.zeros(3, 0, 40, dtype=dtype, device=dev), 7, out=old, accumulate=True)
        assert bool(old.eq(1).all())
        assert hm.embedding_grad(torch.zeros(4, dtype=torch.long, device=dev), torch.zeros(4, 0, device=dev, dtype=dtype), 7).shape == (7, 0)
    assert hm.embedding(none, torch.zeros(0, 5, device=dev)).shape == (3, 0, 5)
    assert bool(hm.embedding(torch.zeros(4, dtype=torch.long, device=dev), torch.zeros(0, 5, device=dev)).eq(0).all())


def test_gradient_with_infinities(dev):
    """Infinities and NaN reach their own token's row and no other, not from masked positions."""
    ids = torch.tensor([4, 1, -1, 2, 4, 9, 1, 3] * 9)
    dy = torch.randn(72, 24, generator=gen(9))
    dy[0, 5], dy[2], dy[5, 7], dy[7, 0] = float("inf"), float("nan"), float("nan"), -float("inf")
    got = hm.embedding_grad(ids.to(dev), dy.to(dev), 10, padding_idx=9).cpu()
    assert bool(got[9].eq(0).all()) and got[4, 5].isinf() and got[3, 0] == -float("inf")
    assert got.isfinite().sum() == got.numel() - 2


# ------------------------------------------------------------------ autograd
@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("padding_idx", [None, 3, -1])
def test_embedding_autograd(dev, dtype, padding_idx):
    """The gradient and the gradient's gradient against autograd through F.embedding in 64 bits."""
    V, D = 30, 50
    w = torch.randn(V, D, generator=gen(11)).to(dtype)
    ids = make_ids("text", 2 * 70, V).view(2, 70)
    R = torch.randn(2, 70, D, generator=gen(12)).to(dtype)
    S = torch.randn(V, D, generator=gen(13)).to(dtype)
    wd, Rd = w.to(dev).requires_grad_(), R.to(dev).requires_grad_()
    y = hm.embedding(ids.to(dev), wd, scale=1.5, padding_idx=padding_idx)
    (dw,) = torch.autograd.grad(y, wd, Rd, create_graph=True)
    (dR,) = torch.autograd.grad(dw, Rd, S.to(dev))
    check_grad(dw, *grad64(ids, R, V, 1.5, None if padding_idx is None else padding_idx % V))
    masked = ids if padding_idx is None else ids.masked_fill(ids == padding_idx % V, -1)
    ref = lookup64(masked, S, 1.5)
    assert bool(((dR.double().cpu() - ref).abs() <= ref.abs() * (U + half_step(dtype) * (1 + U))).all())
    # differences: the lookup is linear in the weight
    step = torch.randn(V, D, generator=gen(14)).double()
    if padding_idx is not None:
        step[padding_idx] = 0
    change = ((lookup64(ids, w.double() + step, 1.5) - lookup64(ids, w, 1.5)) * R.double()).sum()
    along = (dw.double().cpu() * step).sum()
    mag = (grad64(ids, R.abs(), V, 1.5)[0] * step.abs()).sum()
    assert abs(change - along) <= (half_step(dtype) + 200 * U) * mag


def test_embedding_module(dev):
    """Embedding beside nn.Embedding: the same rows, the gradient within what two orders of summing differ by; a broadcast
    upstream gradient; and what the kernels do not take."""
    ids = make_ids("text", 4 * 300, 200).view(4, 300).to(dev)
    for kw in ({}, dict(padding_idx=5)):
        torch.manual_seed(1)
        a = nn.Embedding(200, 48, **kw).to(dev)
        torch.manual_seed(1)
        b = hm.Embedding(200, 48, **kw).to(dev)
        assert torch.equal(a(ids), b(ids))
        R = torch.randn(4, 300, 48, generator=gen(3)).to(dev)
        (a(ids) * R).sum().backward()
        (b(ids) * R).sum().backward()
        check_grad(b.weight.grad, *grad64(ids.cpu(), R.cpu(), 200, 1.0, kw.get("padding_idx")))
        b.weight.grad = None
        b(ids).sum().backward()  # an expanded gradient
        assert torch.equal(b.weight.grad, F.one_hot(ids.flatten(), 200).sum(0).float()[:, None].expand(200, 48)
                           * (torch.arange(200, device=dev) != kw.get("padding_idx", -1)).float()[:, None])
    c = hm.Embedding(20, 6, sparse=True, scale=2.0).to(dev)
    c(ids % 20).sum().backward()
    assert c.weight.grad.is_sparse
    d = hm.Embedding(20, 6, dtype=torch.float64).to(dev)
    assert d(ids % 20).dtype == torch.float64
    h = hm.Embedding(20, 6, scale=2.0).to(dev)
    y, dy = torch.func.jvp(lambda w: torch.func.functional_call(h, {"weight": w}, (ids % 20,)), (h.weight.detach(),), (torch.ones(20, 6, device=dev),))
    assert torch.equal(y, h(ids % 20)) and bool(dy.eq(2).all())
    want = 2 * F.one_hot(ids.flatten() % 20, 20).sum(0).float()[:, None].expand(20, 6)
    for lookup in (lambda w, i: torch.func.functional_call(h, {"weight": w}, (i,)), lambda w, i: hm.embedding(i, w, 2.0)):
        assert torch.equal(torch.func.grad(lambda w: lookup(w, ids % 20).sum())(h.weight.detach()), want)
    per = torch.func.vmap(torch.func.grad(lambda w, i: torch.func.functional_call(h, {"weight": w}, (i,)).sum()), (None, 0))
    assert torch.equal(per(h.weight.detach(), ids % 20).sum(0), want)  # a gradient for each sequence


def test_ids_written_between_forward_and_backward(dev):
    """The backward reads the ids again: ids that changed meanwhile are reported, as by nn.Embedding."""
    w = torch.randn(10, 8, device=dev, requires_grad=True)
    ids = torch.arange(6, device=dev)
    y = hm.embedding(ids, w)
    ids.add_(1)
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.sum().backward()


# ------------------------------------------------------------------ norm and clipping
def make_tensors(shapes, dtypes, seed=0, std=1.0):
    g = gen(seed)
    return [(std * torch.randn(s, generator=g)).to(dtypes[i % len(dtypes)]) for i, s in enumerate(shapes)]


def norm64(ts, kind=2.0):
    v = torch.cat([t.double().flatten() for t in ts]) if ts else torch.zeros(0, dtype=torch.float64)
    return v.abs().max() if kind == math.inf and v.numel() else v.square().sum().sqrt()


LISTS = {
    "one": [(1,)], "few": [(3,), (0,), (65, 7), (5, 1, 4)], "edges": [(16383,), (16384,), (16385,), (32767,), (32768,), (32769,), (8,), (9,)],
    "many": [(i % 37,) for i in range(500)], "large": [(3001, 2003), (17,), (1000003,)],
}


@pytest.mark.parametrize("dtypes", [(FP,), (BF,), (BF, FP, FP)], ids=["fp32", "bf16", "mixed"])
@pytest.mark.parametrize("name", LISTS)
@pytest.mark.parametrize("kind", [2.0, math.inf])
def test_grad_norm(dev, name, kind, dtypes):
    _say("grad_norm", name, kind, dtypes)
    ts = make_tensors(LISTS[name], dtypes, std=1e-3)
    on = [t.to(dev) for t in ts]
    got, ref = hm.grad_norm(on, kind), norm64(ts, kind)
    assert got.dtype == FP and got.shape == () and got.device == on[0].device
    assert abs(got.double().cpu() - ref) <= (U + 1e-9) * ref
    assert torch.equal(got, hm.grad_norm(iter(on), kind))
    assert all(torch.equal(a.cpu(), b) for a, b in zip(on, ts))


@pytest.mark.parametrize("dtype", [FP, BF])
def test_grad_norm_values(dev, dtype):
    """Squares beyond fp32's range on either side, infinities and NaN."""
    big, tiny = torch.full((1000,), 2.0 ** 120), torch.full((999,), 2.0 ** -126)
    for t in (big, tiny, torch.cat([big, tiny])):
        t = t.to(dtype)
        assert abs(hm.grad_norm([t.to(dev)]).double().cpu() - norm64([t])) <= (U + 1e-9) * norm64([t])
    top = torch.full((64,), torch.finfo(dtype).max, dtype=dtype)
    assert hm.grad_norm([top.to(dev)]).isinf()  # 8 times the largest bf16 is above fp32's range
    x = torch.randn(5000, generator=gen(2)).to(dtype)
    for value in (float("inf"), -float("inf"), float("nan")):
        y = x.clone()
        y[4321] = value
        for kind in (2.0, math.inf):
            got = hm.grad_norm([x.to(dev), y.to(dev)], kind)
            assert got.isnan() if value != value else got.item() == float("inf")
    assert hm.grad_norm([torch.zeros(70, device=dev, dtype=dtype)]).item() == 0.0
    assert hm.grad_norm([torch.zeros(0, device=dev, dtype=dtype)], math.inf).item() == 0.0


def test_grad_norm_layouts(dev):
    """Slices of a buffer at any element, transposed and gapped tensors, the same tensor twice, a single tensor."""
    buf = torch.randn(3, 1000, 77, generator=gen(5))
    on = buf.to(dev)
    views = lambda t: [t[0], t[1].flatten()[1:40001], t[2].t(), t[0, ::2], t[:, :, 3], t[1, 4].expand(6, 77)]  # noqa: E731
    ref = norm64([v.contiguous() for v in views(buf)])
    assert abs(hm.grad_norm(views(on)).double().cpu() - ref) <= (U + 1e-9) * ref
    assert torch.equal(hm.grad_norm(on), hm.grad_norm([on]))
    assert abs(hm.grad_norm([on, on]).double().cpu() - 2 ** 0.5 * norm64([buf])) <= (U + 1e-9) * 2 * norm64([buf])


@pytest.mark.parametrize("dtypes", [(FP,), (BF,), (BF, FP, FP)], ids=["fp32", "bf16", "mixed"])
@pytest.mark.parametrize("name", LISTS)
@pytest.mark.parametrize("share", [0.0, 0.3, 0.999, 1.5, math.inf])
def test_clip(dev, name, share, dtypes):
    """Bit for bit what the formula gives in fp32 operations; untouched where the factor is 1."""
    _say("clip", name, share, dtypes)
    ts = make_tensors(LISTS[name], dtypes, seed=1)
    limit = float(norm64(ts)) * share if share != math.inf else math.inf
    params = [nn.Parameter(torch.zeros_like(t, device=dev)) for t in ts] + [nn.Parameter(torch.zeros(3, device=dev))]
    for p, t in zip(params, ts):
        p.grad = t.to(dev)
    versions = [p.grad._version for p in params[:-1]]
    norm = hm.clip_grad_norm_(iter(params), limit)
    assert abs(norm.double().cpu() - norm64(ts)) <= (U + 1e-9) * norm64(ts)
    assert torch.equal(norm, hm.grad_norm([t.to(dev) for t in ts]))
    factor = (torch.tensor(limit, dtype=FP) / (norm.cpu() + 1e-6)).clamp(max=1.0)
    for p, t in zip(params, ts):
        assert torch.equal(p.grad.cpu(), (t.float() * factor).to(t.dtype))
    assert all(p.grad._version > v for p, v in zip(params, versions))
    if share > 1:
        assert all(torch.equal(p.grad.cpu(), t) for p, t in zip(params, ts))
    # the same through the two operators, the norm as a tensor and as a number
    for total in (norm, norm.double().view(1, 1), norm.item()):
        on = [t.to(dev) for t in ts]
        assert hm.clip_grads_(on, limit, total) is None
        assert all(torch.equal(a, p.grad) for a, p in zip(on, params))


def test_clip_as_torch_does(dev):
    """torch.nn.utils.clip_grad_norm_ on copies, both norms, norms that are not finite."""
    for value in (None, float("inf"), float("nan")):
        for kind in (2.0, math.inf):
            ts = make_tensors([(50, 40), (7,), (1000,)], (FP,), seed=3)
            if value is not None:
                ts[0][3, 3] = value
            a, b = ([nn.Parameter(torch.zeros_like(t, device=dev)) for t in ts] for _ in range(2))
            for p, q, t in zip(a, b, ts):
                p.grad, q.grad = t.to(dev), t.to(dev)
            na, nb = hm.clip_grad_norm_(a, 1.5, kind), torch.nn.utils.clip_grad_norm_(b, 1.5, kind)
            torch.testing.assert_close(na, nb, rtol=1e-5, atol=0, equal_nan=True)
            for p, q in zip(a, b):
                torch.testing.assert_close(p.grad, q.grad, rtol=1e-5, atol=0, equal_nan=True)


def test_clip_nonfinite_can_raise(dev):
    p = nn.Parameter(torch.zeros(5, device=dev))
    p.grad = torch.tensor([1.0, float("nan"), 2, 3, 4], device=dev)
    with pytest.raises(RuntimeError, match="not finite"):
        hm.clip_grad_norm_(p, 1.0, error_if_nonfinite=True)
    assert p.grad[2] == 2
    p.grad = torch.full((5,), 2.0, device=dev)
    assert abs(hm.clip_grad_norm_(p, 1.0, error_if_nonfinite=True).item() - 20 ** 0.5) < 1e-6
    assert abs(p.grad[0].item() - 2 * 20 ** -0.5) < 1e-6


def test_a_parameter_given_twice_counts_once(dev):
    p, q = nn.Parameter(torch.zeros(9, device=dev)), nn.Parameter(torch.zeros(4, device=dev))
    p.grad, q.grad = torch.full((9,), 2.0, device=dev), torch.full((4,), 3.0, device=dev)
    assert abs(hm.clip_grad_norm_([p, q, p], 1.0).item() - 72 ** 0.5) < 1e-5
    assert abs(p.grad[0].item() - 2 / 72 ** 0.5) < 1e-6


def test_clip_layouts(dev):
    """Dense tensors in other orders and at any element are scaled; what lies between them is not touched."""
    buf = torch.randn(4, 300, 77, generator=gen(5))
    for dtype in (FP, BF):
        b = buf.to(dtype)
        on = b.to(dev)
        hm.clip_grads_([on[0].flatten()[1:20000], on[1].t(), on[2][None], on[3, 1:2, 3:50]], 1.0, 4.0)
        ref = b.clone()
        f = torch.tensor(1.0) / (torch.tensor(4.0) + 1e-6)
        for v in (ref[0].flatten()[1:20000], ref[1], ref[2], ref[3, 1:2, 3:50]):
            v.copy_((v.float() * f).to(dtype))
        assert torch.equal(on.cpu(), ref)


# ------------------------------------------------------------------ refusals
def test_embedding_refusals(dev):
    w, ids = torch.zeros(10, 8, device=dev), torch.zeros(4, dtype=torch.long, device=dev)
    dy = torch.zeros(4, 8, device=dev)
    with pytest.raises(RuntimeError, match="no CPU path"):
        hm.embedding(ids.cpu(), w)
    with pytest.raises(RuntimeError, match="no CPU path"):
        hm.embedding(ids, w.cpu())
    for bad in (ids.float(), ids.short(), ids.bool()):
        with pytest.raises(TypeError, match="token ids"):
            hm.embedding(bad, w)
        with pytest.raises(TypeError, match="token ids"):
            hm.embedding_grad(bad, dy, 10)
    with pytest.raises(TypeError, match="unsupported dtype"):
        hm.embedding(ids, w.half())
    with pytest.raises(TypeError, match="unsupported dtype"):
        hm.embedding_grad(ids, dy.double(), 10)
    with pytest.raises(RuntimeError, match="tokens, width"):
        hm.embedding(ids, w[0])
    with pytest.raises(RuntimeError, match="a row for each"):
        hm.embedding_grad(ids, dy[:3], 10)
    with pytest.raises(RuntimeError, match="a row for each"):
        hm.embedding_grad(ids[:, None], dy, 10)
    for out in (torch.zeros(9, 8, device=dev), torch.zeros(10, 7, device=dev), torch.zeros(8, 10, device=dev).t(), torch.zeros(80, device=dev)):
        with pytest.raises(RuntimeError, match="out must be"):
            hm.embedding_grad(ids, dy, 10, out=out)
    with pytest.raises(RuntimeError, match="accumulate needs out"):
        hm.embedding_grad(ids, dy, 10, accumulate=True)
    with pytest.raises(RuntimeError):
        hm.embedding_grad(ids, dy, 10, out=torch.zeros(10, 8))
    with pytest.raises(TypeError, match="unsupported dtype"):
        hm.embedding_grad(ids, dy, 10, out=torch.zeros(10, 8, device=dev, dtype=torch.half))
    buf = torch.zeros(20, 8, device=dev)
    with pytest.raises(RuntimeError, match="shares memory"):
        hm.embedding_grad(ids, buf[8:12], 10, out=buf[:10])
    hm.embedding_grad(ids, buf[10:14], 10, out=buf[:10])
    with pytest.raises(RuntimeError, match="no gradient"):
        hm.embedding_grad(ids, dy.clone().requires_grad_(), 10, out=torch.zeros(10, 8, device=dev))
    with pytest.raises(RuntimeError):
        hm.embedding_grad(ids, dy, -1)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(w, torch.ones_like(w))
        with pytest.raises(RuntimeError, match="forward"):
            hm.embedding(ids, dual)


def test_norm_refusals(dev):
    x = torch.ones(40, device=dev)
    with pytest.raises(TypeError, match="unsupported dtype"):
        hm.grad_norm([x, x.half()])
    with pytest.raises(RuntimeError, match="no CPU path"):
        hm.grad_norm([x, x.cpu()])
    with pytest.raises(RuntimeError, match="takes? dense|take dense"):
        hm.grad_norm([x.to_sparse()])
    with pytest.raises(RuntimeError, match="no gradient"):
        hm.grad_norm([x.clone().requires_grad_()])
    with torch.no_grad():
        hm.grad_norm([x.clone().requires_grad_()])
    p = nn.Parameter(x.clone())
    p.pow(3).sum().backward(create_graph=True)  # a gradient that needs one: clipped without autograd, as by torch
    assert p.grad.requires_grad and abs(hm.clip_grad_norm_(p, 1.0).item() - 360 ** 0.5) < 1e-4
    assert abs(p.grad.norm().item() - 1) < 1e-5
    p.grad = None
    for bad in (x[::2], x[:1].expand(9)):
        with pytest.raises(RuntimeError, match="gaps or overlaps"):
            hm.clip_grads_([bad], 1.0, 2.0)
    for bad in ([x, x], [x[:20], x[19:]], [x[5:], x[:6]], [x, x.view(BF)[3:5]]):
        with pytest.raises(RuntimeError, match="share memory"):
            hm.clip_grads_(bad, 1.0, 2.0)
    with pytest.raises(RuntimeError, match="share memory"):
        hm.clip_grads_([x], 1.0, x[3])
    with pytest.raises(RuntimeError, match="total_norm"):
        hm.clip_grads_([x], 1.0, torch.ones(2, device=dev))
    with pytest.raises(RuntimeError, match="total_norm"):
        hm.clip_grads_([x], 1.0, torch.ones(()))
    with pytest.raises(RuntimeError, match="total_norm"):
        hm.clip_grads_([x], 1.0, torch.ones((), dtype=torch.long, device=dev))
    with pytest.raises(RuntimeError, match="no gradient"):
        hm.clip_grads_([x], 1.0, torch.full((), 2.0, device=dev, requires_grad=True))
    assert bool(x.eq(1).all())
    hm.clip_grads_([x[:20], x[20:]], 1.0, 2.0)
    assert bool(x.lt(1).all())


# ------------------------------------------------------------------ streams, graphs, the model
def test_on_another_stream(dev):
    """Calls on two streams at once, each behind its own stream's work."""
    V, D, T = 5000, 256, 6000
    ids = [make_ids("text", T, V, seed=s).to(dev) for s in (1, 2)]
    dy = [torch.randn(T, D, generator=gen(s)).to(BF).to(dev) for s in (3, 4)]
    want = [(hm.embedding_grad(i, d, V), hm.grad_norm([d, d])) for i, d in zip(ids, dy)]
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                d = dy[k] + 0
                got.append((k, hm.embedding_grad(ids[k], d, V), hm.grad_norm([d, d])))
    torch.cuda.synchronize()
    for k, g, n in got:
        assert torch.equal(g, want[k][0]) and torch.equal(n, want[k][1])


def test_recorded(dev):
    """Lookup, gradient, norm and clipping in one recording; two recordings replayed in turn, the ids and gradients new each
    time, against the eager calls."""
    V, D = 700, 200

    class Rec:
        def __init__(self, T):
            self.ids = torch.zeros(T, dtype=torch.long, device=dev)
            self.w = torch.randn(V, D, generator=gen(1)).to(BF).to(dev)
            self.dy = torch.zeros(T, D, dtype=BF, device=dev)
            self.out = self.run()
            torch.cuda.synchronize()
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self.out = self.run()

        def run(self):
            y = hm.embedding(self.ids, self.w, scale=3.0)
            dw = hm.embedding_grad(self.ids, self.dy, V)
            more = dw.float()
            norm = hm.grad_norm([dw, more])
            hm.clip_grads_([dw, more], 1.0, norm)
            return y, dw, more, norm

    recs = [Rec(3000), Rec(90), Rec(9000)]
    for turn in range(4):
        for k, r in enumerate(recs):
            r.ids.copy_(make_ids("text" if turn % 2 else "same", r.ids.numel(), V, seed=turn))
            r.dy.copy_(torch.randn(r.dy.shape, generator=gen(10 * turn + k)))
        for r in recs:
            r.graph.replay()
        for r in recs:
            assert all(torch.equal(a, b) for a, b in zip(r.out, r.run()))


def test_recorded_step(dev):
    """Forward, backward and clipping of an embedding with a tied head in one recording, replayed with new ids, against the same
    step run eagerly on a copy."""
    V, D, T = 600, 128, 1500

    def make():
        e = hm.Embedding(V, D, scale=2.0).to(BF).to(dev)
        torch.nn.init.normal_(e.weight, std=0.1)
        return e

    torch.manual_seed(3)
    e = make()
    ids = torch.zeros(T, dtype=torch.long, device=dev)

    def step(m, i):
        m.weight.grad = None
        y = m(i)
        (y.float() @ m.weight.float().t()).logsumexp(1).mean().backward()
        return y.detach(), hm.clip_grad_norm_(m.parameters(), 1e-3)

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        for _ in range(2):
            step(e, ids)
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize()
    e.weight.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y, norm = step(e, ids)
    grad = e.weight.grad
    for turn in range(4):
        ids.copy_(make_ids("text" if turn % 2 else "wild", T, V, seed=turn))
        graph.replay()
        other = make()
        other.weight.data.copy_(e.weight)
        y2, norm2 = step(other, ids)
        assert torch.equal(y, y2) and torch.equal(norm, norm2) and torch.equal(grad, other.weight.grad)
        assert norm > 1e-3


def _lm(dev, dtype=BF, mixer=True):
    torch.manual_seed(0)
    lm = hm.HdcMambaLM(256, 2, 64, 4, vocab_size=512, chunk_size=64)
    for i, blk in enumerate(lm.backbone.layers):
        reinit_block_(blk, seed=30 + i, decays_uniform=True)
    lm = lm.to(dtype).to(dev).train()
    hm.set_differentiable_mixer(lm, mixer)
    return lm


@pytest.mark.parametrize("dtype", [FP, BF])
def test_training_step_of_the_model(dev, dtype):
    """A step as a trainer runs it (a left-padded length, the ids a slice of a batch): the same logits and gradients as with
    nn.Embedding and torch's clipping in the model's place, and parameters that move."""
    a, b = _lm(dev, dtype), _lm(dev, dtype)
    old = nn.Embedding(512, 256, _weight=b.embedding.weight.detach().clone()).to(dev)
    b.embedding = old
    b.lm_head.weight = old.weight
    batch = make_ids("text", 2 * 151, 512).view(2, 151).to(dev)
    losses, norms = [], []
    for m, clip in ((a, hm.clip_grad_norm_), (b, torch.nn.utils.clip_grad_norm_)):
        logits = m(batch[:, :-1])
        loss = F.cross_entropy(logits.float().reshape(-1, 512), batch[:, 1:].reshape(-1))
        loss.backward()
        losses.append(loss)
        norms.append(clip(m.parameters(), 0.1))
    assert torch.equal(losses[0], losses[1])  # the lookup copies rows
    assert type(a.embedding) is hm.Embedding and norms[0] > 0.1
    # both norms are of the same gradients but for the embedding's, whose sums have another order; torch's rounds the norm
    # of each bf16 tensor to bf16
    assert abs(norms[0].item() - norms[1].item()) <= (8 * half_step(dtype) if dtype == BF else 1e-5) * norms[1].item()
    for (n, p), q in zip(a.named_parameters(), b.parameters()):
        assert (p.grad is None) == (q.grad is None), n
        if p.grad is not None:
            lim = 16 * half_step(dtype) if dtype == BF else 1e-5
            assert (p.grad.float() - q.grad.float()).norm() <= lim * q.grad.float().norm(), n
    total = hm.grad_norm([p.grad for p in a.parameters() if p.grad is not None])
    assert abs(total.item() - 0.1) <= 0.1 * (2 * half_step(dtype) + 8 * U + 1e-6 / norms[0].item())  # the 1e-6 of the factor
    before = [p.detach().clone() for p in a.parameters()]
    torch.optim.SGD(a.parameters(), lr=1e4).step()
    assert all(torch.equal(p, q) == (p.grad is None) for p, q in zip(a.parameters(), before))


def test_rows_far_apart(dev):
    """Offsets past 32 bits in elements: the last rows of a long weight, a gradient whose rows lie far apart, its weight's last rows."""
    V, D = 2 ** 21 + 5, 2056
    w = torch.zeros(V, D, dtype=BF, device=dev)  # 8.6 GB
    w[-3:] = torch.randn(3, D, generator=gen(1)).to(BF).to(dev)
    ids = torch.tensor([V - 1, 0, V - 3, V - 2, V], device=dev)
    got = hm.embedding(ids, w)
    assert torch.equal(got[[0, 2, 3]], w[[V - 1, V - 3, V - 2]]) and bool(got[[1, 4]].eq(0).all())
    dy = torch.randn(5, D, generator=gen(2)).to(BF)
    hm.embedding_grad(ids, dy.to(dev), V, out=w)
    assert torch.equal(w[[V - 1, 0, V - 3, V - 2]].cpu(), dy[:4]) and bool(w[1:V - 3].any().eq(False))
    far = w.view(-1)[:1100 * 3919000].view(1100, 3919000)[:, :40]
    far.copy_(torch.randn(1100, 40, generator=gen(3)))
    i = make_ids("text", 1100, 37)
    check_grad(hm.embedding_grad(i.to(dev), far, 37), *grad64(i, far.cpu(), 37))
    n = 2 ** 31 + 77  # a tensor of more than 2^31 elements
    t = w.view(-1)[:n]
    t.zero_()
    t[-1], t[0] = 3.0, 4.0
    assert hm.grad_norm([t]).item() == 5.0
    hm.clip_grads_([t], 1.0, 2.0)
    assert t[-1] == 1.5 and t[0] == 2.0
