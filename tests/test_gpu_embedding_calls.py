"""Calls around the token rows, the gradients' norm and clipping that the operators' own tests leave out: ids outside the
vocabulary through the whole model, lookups that go past the kernels, gradients of every kind, and the largest lists.

Tolerances.  A product or sum in fp32 is off by at most 2^-24 of its value, a sum of m terms in any order by m 2^-24 of the
sum of their magnitudes, and a result rounded to its type by half a step, finfo.eps / 2 of its value.  Squares are
added in 64 bits, so a norm is off by its own rounding.
"""
import copy
import math

import pytest
import torch
import torch.nn as nn

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


def _lm(dev, dtype=BF, V=300):
    torch.manual_seed(0)
    lm = hm.HdcMambaLM(256, 2, 64, 4, vocab_size=V, chunk_size=32)
    for i, blk in enumerate(lm.backbone.layers):
        reinit_block_(blk, seed=30 + i, decays_uniform=True)
    return lm.to(dtype).to(dev)


# ------------------------------------------------------------------ ids outside the vocabulary
@pytest.mark.parametrize("plain", [False, True])
@pytest.mark.parametrize("dtype", [FP, BF])
def test_an_id_outside_the_vocabulary_is_a_row_of_zeros_everywhere(dev, dtype, plain):
    """forward, prefill, step and a recorded step take ids that are no token as they take a token whose row is zeros; in a step
    also where an nn.Embedding stands in the module's place."""
    _say("ids outside the vocabulary", dtype, plain)
    V, zero = 300, 3
    lm = _lm(dev, dtype, V).eval()
    with torch.no_grad():
        lm.embedding.weight[zero] = 0
    bad = torch.tensor([-1, V, -7, 2 ** 40 + 5], device=dev)
    ids = torch.randint(0, V, (5, 40), generator=gen(1)).to(dev)
    wild, tame = ids.clone(), ids.clone()
    wild[1:, 11], tame[1:, 11] = bad, zero
    wild[1:, 39], tame[1:, 39] = bad, zero
    with torch.no_grad():
        assert torch.equal(lm(wild), lm(tame))
        last, states = lm.prefill(wild)
        assert torch.equal(last, lm.prefill(tame)[0])
        if plain:
            old = nn.Embedding(V, 256, _weight=lm.embedding.weight.detach())
            lm.embedding = old
        got, ref, rec, tok = (copy.deepcopy(states) for _ in range(4))
        assert torch.equal(lm.step(wild[:, 11].contiguous(), got), lm.step(tame[:, 11].contiguous(), ref))
        a, b = lm.capture_decode(rec), lm.capture_decode(tok)
        for _ in range(3):
            assert torch.equal(a.step(wild[:, 11]), b.step(tame[:, 11]))
            assert torch.equal(a.step(ids[:, 0]), b.step(ids[:, 0]))


WILD = [4, -1, 2, 20, 4, 2 ** 40, 9, -(2 ** 63), 0, 19, 21, 4]


@pytest.mark.parametrize("kw", [dict(dtype=torch.float64), dict(dtype=torch.half), dict(max_norm=0.7), dict(sparse=True),
                                dict(scale_grad_by_freq=True), dict(scale_grad_by_freq=True, padding_idx=4)])
def test_ids_outside_past_the_kernels(dev, kw):
    """Where Embedding goes through nn.Embedding's forward an id that is no token is a row of zeros without a gradient too.
    The rows are sums of at most three small whole numbers: exact in every type."""
    _say("ids outside, past the kernels", kw)
    ids = torch.tensor(WILD)
    there = (ids >= 0) & (ids < 20)
    w = torch.randint(-8, 9, (20, 6), generator=gen(1)).to(kw.get("dtype", FP))
    m = hm.Embedding(20, 6, _weight=w.to(dev), scale=2.0, **kw)
    ref = nn.Embedding(20, 6, _weight=w.clone(), **kw)
    near = ids.clamp(0, 19)
    y = m(ids.view(3, 4).to(dev))
    want = ref(near) * 2 * there[:, None]
    tol = 1e-6 if "max_norm" in kw else 0
    torch.testing.assert_close(y.cpu().view(12, 6), want.detach(), rtol=tol, atol=0)
    torch.testing.assert_close(m.weight.detach().cpu(), ref.weight.detach(), rtol=tol, atol=0)
    R = torch.randint(-3, 4, (12, 6), generator=gen(2)).to(w.dtype)
    (y.view(12, 6) * R.to(dev)).sum().backward()
    (want * R).sum().backward()
    assert m.weight.grad.is_sparse == kw.get("sparse", False)
    assert torch.equal(m.weight.grad.to_dense().cpu(), ref.weight.grad.to_dense())
    assert not hm.Embedding(0, 6, device=dev, dtype=torch.float64)(ids.to(dev)).any()


@pytest.mark.parametrize("dtype", [FP, BF])
def test_ids_outside_under_transforms(dev, dtype):
    """Tangents and gradients for each sequence of a batch that is padded with ids that are no token."""
    ids = torch.tensor(WILD, device=dev).view(3, 4)
    there = (ids >= 0) & (ids < 20)
    m = hm.Embedding(20, 6, device=dev, dtype=dtype, scale=2.0)
    w = m.weight.detach()
    call = lambda w, i: torch.func.functional_call(m, {"weight": w}, (i,))  # noqa: E731
    y, dy = torch.func.jvp(lambda w: call(w, ids), (w,), (torch.ones_like(w),))
    assert torch.equal(y, m(ids)) and torch.equal(dy, 2 * there[..., None].expand_as(dy).to(dtype))
    per = torch.func.vmap(torch.func.grad(lambda w, i: call(w, i).sum()), (None, 0))(w, ids)
    for i, t, g in zip(ids, there, per):
        count = torch.bincount(i[t], minlength=20)
        assert torch.equal(g, 2 * count[:, None].expand(20, 6).to(dtype))


def test_traced_compiled_and_seen_by_a_mode(dev):
    """What follows the lookup's operations finds PyTorch's: no constant in a trace, one graph, an operation that a mode sees."""
    from torch.utils.flop_counter import FlopCounterMode

    m = hm.Embedding(20, 6, device=dev, scale=2.0)
    ids, other = (torch.randint(0, 20, (2, 9), generator=gen(s)).to(dev) for s in (1, 2))
    with torch.no_grad():
        traced = torch.jit.trace(m, (ids,))
        assert torch.equal(traced(other), m(other))
    compiled = torch.compile(m, backend="eager", fullgraph=True)
    for i in (ids, other):
        y = compiled(i)
        assert torch.equal(y, m(i))
        y.sum().backward()
        assert torch.equal(m.weight.grad, 2.0 * torch.bincount(i.flatten(), minlength=20)[:, None].expand(20, 6))
        m.weight.grad = None
    with FlopCounterMode(display=False):
        assert torch.equal(m(other), traced(other))


# ------------------------------------------------------------------ gradients of every kind
def _sums(ids, dy, V, scale, padding=None):
    """The gradient in 64 bits: whole numbers, exact in every type."""
    i = ids.flatten()
    ok = (i >= 0) & (i < V)
    if padding is not None:
        ok &= i != padding
    return scale * torch.zeros(V, dy.shape[-1], dtype=torch.float64).index_add_(0, i[ok], dy.double().reshape(-1, dy.shape[-1])[ok])


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("padding_idx", [None, 4])
def test_batched_gradients_and_transforms(dev, dtype, padding_idx):
    """vmap over a backward's gradients, and both operators under torch.func: ids that are no token among the others."""
    V, D = 20, 6
    ids = torch.tensor(WILD).view(3, 4)
    on = ids.to(dev)
    w = torch.randint(-8, 9, (V, D), generator=gen(1)).to(dtype).to(dev)
    Rs = torch.randint(-3, 4, (5, 3, 4, D), generator=gen(2)).to(dtype)
    want = torch.stack([_sums(ids, R, V, 2.0, padding_idx) for R in Rs])
    m = hm.Embedding(V, D, padding_idx=padding_idx, _weight=w.clone(), scale=2.0)
    for y, leaf in ((m(on), m.weight), (hm.embedding(on, w.requires_grad_(), 2.0, padding_idx), w)):
        (got,) = torch.autograd.grad(y, leaf, Rs.to(dev), is_grads_batched=True)
        assert torch.equal(got.double().cpu(), want)
    w = w.detach()
    call = lambda w, i=on: hm.embedding(i, w, 2.0, padding_idx)  # noqa: E731
    y, pull = torch.func.vjp(call, w)
    assert torch.equal(y, call(w))
    assert torch.equal(torch.func.vmap(lambda R: pull(R)[0])(Rs.to(dev)).double().cpu(), want)
    y, dy = torch.func.jvp(call, (w,), (w + 1,))
    rows = call(w + 1)
    if padding_idx is not None:  # its rows are constants for the derivative
        rows = rows.masked_fill((on == padding_idx)[..., None], 0)
    assert torch.equal(y, call(w)) and torch.equal(dy, rows)
    assert torch.equal(torch.func.vmap(call, (None, 0))(w, on), call(w))
    grads = lambda R: hm.embedding_grad(on, R, V, 2.0, padding_idx)  # noqa: E731
    assert torch.equal(torch.func.vmap(grads)(Rs.to(dev)).double().cpu(), want)
    back = torch.func.grad(lambda R: (grads(R) * w).sum())(Rs[0].to(dev))
    ref = 2 * w.cpu()[ids.clamp(0, V - 1)].masked_fill(((ids < 0) | (ids >= V) | (ids == padding_idx))[..., None], 0)
    assert torch.equal(back.cpu(), ref)
    with pytest.raises(RuntimeError, match="transforms"):
        torch.func.vmap(lambda R: hm.embedding_grad(on, R, V, out=w))(Rs.to(dev))


def test_gradients_are_formed_without_python(dev):
    """Neither direction runs Python, which the host of a step of few tokens would wait for."""
    w = torch.zeros(9, 4, device=dev, requires_grad=True)
    y = hm.embedding(torch.zeros(3, dtype=torch.long, device=dev), w)
    (dw,) = torch.autograd.grad(y, w, torch.ones_like(y, requires_grad=True), create_graph=True)
    for t in (y, dw):
        assert t.grad_fn is not None and not isinstance(t.grad_fn, torch.autograd.function.BackwardCFunction)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(torch.ones(3, 4, device=dev), torch.ones(3, 4, device=dev))
        with pytest.raises(RuntimeError, match="forward-mode"):
            hm.embedding_grad(torch.zeros(3, dtype=torch.long, device=dev), dual, 9)
    with torch.inference_mode():
        assert not hm.embedding(torch.zeros(3, dtype=torch.long, device=dev), w).any()


# ------------------------------------------------------------------ the largest lists
def test_norm_of_more_than_2_to_the_24_stretches(dev):
    """One tensor of 4 GiB 260 times over, more workgroups than a launch takes; 260 * 2^30 ones, whose sum is exact."""
    t = torch.ones(2 ** 30, device=dev)
    assert hm.grad_norm([t] * 260).item() == torch.tensor(260.0 * 2 ** 30, dtype=torch.float64).sqrt().to(FP).item()


@pytest.mark.parametrize("dtypes", [(FP,), (BF,), (BF, FP, FP)], ids=["fp32", "bf16", "mixed"])
@pytest.mark.parametrize("MiB", [70, 150])
@pytest.mark.parametrize("kind", [2.0, math.inf])
def test_clip_of_large_lists(dev, kind, MiB, dtypes):
    """More than 1024 stretches, whose norm is joined by a launch of its own; 400 tensors, more than one table; above 128 MiB past
    the caches.  Bit for bit what the formula gives in fp32 operations."""
    _say("clip of large lists", kind, MiB, dtypes)
    g = torch.Generator(device=dev).manual_seed(MiB)
    count = (MiB << 20) // sum(4 if dtypes[i % len(dtypes)] == FP else 2 for i in range(400))
    ts = [torch.empty(count + i % 7, device=dev).normal_(generator=g).to(dtypes[i % len(dtypes)]) for i in range(400)]
    ts[399][-1] = 9.0  # the largest, a tensor's last
    if kind == 2.0:
        ref = torch.stack([t.double().square().sum() for t in ts]).sum().sqrt()
    else:
        ref = torch.stack([t.abs().max().double() for t in ts]).max()
    for share in (0.3, 1.5):
        params = [nn.Parameter(torch.empty_like(t)) for t in ts]
        for p, t in zip(params, ts):
            p.grad = t.clone()
        limit = float(ref) * share
        norm = hm.clip_grad_norm_(params, limit, kind)
        assert abs(norm.double() - ref) <= (U + 1e-9) * ref
        assert torch.equal(norm, hm.grad_norm(ts, kind))
        factor = (torch.tensor(limit, dtype=FP) / (norm.cpu() + 1e-6)).clamp(max=1.0).to(dev)
        assert all(torch.equal(p.grad, (t.float() * factor).to(t.dtype)) for p, t in zip(params, ts))
        on = [t.clone() for t in ts]
        hm.clip_grads_(on, limit, norm)
        assert all(torch.equal(a, p.grad) for a, p in zip(on, params))


def _ids(T, V, seed, dev):
    """Token ids as text has them, a sixth of them one token, and some that are none."""
    u = torch.rand(T, generator=gen(seed), dtype=torch.float64)
    ids = (torch.exp(u * math.log(V + 1)).long() - 1).clamp(0, V - 1)
    ids[::6], ids[5::97] = V // 3, -1
    return ids.to(dev)


@pytest.mark.parametrize("dtype,T,D", [(FP, 110000, 1030), (FP, 50000, 700), (BF, 180000, 1030), (BF, 90000, 1030)])
def test_gradient_past_the_caches(dev, dtype, T, D):
    """Units of 16 and of 32 positions whose rows go past the caches, in both types."""
    _say("gradient past the caches", dtype, T, D)
    V = 3000
    ids = _ids(T, V, T, dev)
    dy = torch.empty(T, D, device=dev, dtype=dtype).normal_(generator=torch.Generator(device=dev).manual_seed(1))
    got = hm.embedding_grad(ids, dy, V, scale=0.7)
    there = ids >= 0
    s = torch.tensor(0.7, dtype=FP).double().item()
    ref, mag = torch.zeros(V, D, device=dev, dtype=torch.float64), torch.zeros(V, D, device=dev, dtype=torch.float64)
    ref.index_add_(0, ids[there], dy[there].double()).mul_(s)
    mag.index_add_(0, ids[there], dy[there].double().abs()).mul_(s)
    terms = torch.bincount(ids[there], minlength=V).double()[:, None]
    before = (terms + 1) * U * mag
    assert bool(((got.double() - ref).abs() <= before + half_step(dtype) * (ref.abs() + before) + 1e-40).all())
    assert torch.equal(got, hm.embedding_grad(ids.int(), dy, V, scale=0.7))


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("idt", [torch.int64, torch.int32])
def test_lookup_past_the_caches(dev, dtype, idt):
    """Outputs of more than 128 MiB, scaled and not, ids that are no token among them."""
    T, D, V = 70000, 1030, 3000
    ids = _ids(T, V, 1, dev).to(idt)
    w = torch.empty(V, D, device=dev, dtype=dtype).normal_(generator=torch.Generator(device=dev).manual_seed(2))
    rows = w[ids.clamp(min=0).long()].masked_fill((ids < 0)[:, None], 0)
    assert torch.equal(hm.embedding(ids, w), rows)
    assert torch.equal(hm.embedding(ids, w, scale=2.7), (rows.float() * 2.7).to(dtype))


# ------------------------------------------------------------------ what a trainer wraps a lookup in
def test_gradient_in_a_trainers_wrappers(dev):
    """Checkpointing, saved tensors on the host, anomaly detection, an autocast region, vectorized Jacobians, threads, and an id
    tensor that was written between forward and backward: the gradient is that of the plain call, or the call is refused."""
    import threading

    from torch.utils.checkpoint import checkpoint

    V, D = 50, 24
    ids = torch.randint(-1, V, (4, 33), generator=gen(3)).to(dev)[:, 1:]
    R = torch.randint(-3, 4, (4, 32, D), generator=gen(4)).float().to(dev)
    m = hm.Embedding(V, D, device=dev, padding_idx=7)
    want = _sums(ids.cpu(), R.cpu(), V, 1.0, 7).float().to(dev)

    def backward(call):
        m.weight.grad = None
        (call(ids) * R).sum().backward()
        assert torch.equal(m.weight.grad, want)

    backward(m)
    for reentrant in (False, True):
        backward(lambda i: checkpoint(lambda i, w: hm.embedding(i, w, padding_idx=7), i, m.weight, use_reentrant=reentrant))
    with torch.autograd.graph.save_on_cpu():
        backward(m)
    with torch.autograd.set_detect_anomaly(True):
        backward(m)
    with torch.autocast("cuda", torch.bfloat16):
        y = m(ids)
        assert y.dtype == FP
        backward(m)
    for vectorize in (False, True):
        J = torch.autograd.functional.jacobian(lambda w: hm.embedding(ids[0, :3], w, 2.0).sum(1), m.weight.detach(), vectorize=vectorize)
        ref = torch.zeros(3, V, D, device=dev)
        for k, i in enumerate(ids[0, :3].tolist()):
            if i >= 0:
                ref[k, i] = 2
        assert torch.equal(J, ref)
    got = [None] * 4

    def work(k):
        w = m.weight.detach().clone().requires_grad_()
        for _ in range(20):
            (got[k],) = torch.autograd.grad(hm.embedding(ids, w, padding_idx=7), w, R)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    y = m(ids)
    ids.add_(1)
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.sum().backward()
