"""Models with 4-bit weights, and generation with the choice of the token inside the recorded step.

A quantised model is compared with the oracle on the weights that it holds (brought back from 4
bits, exact in fp32); tolerances are those of the unquantised decode tests (fp32 1e-4 elementwise, bf16 2e-2
normwise).  The chosen tokens are compared with the formula on the CPU, applied to the logits that the
step produced.
"""
import copy

import pytest
import torch

import hdcmamba_amd as hm
import oracle
from cfgs import assert_close, assert_close_normwise, make_lm, max_rel, reinit_block_

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _say(*a):
    print(*a, flush=True)


def _lm(dm, ds, H, C, n_layers, vocab, dtype, seed=0):
    torch.manual_seed(seed)
    lm = hm.HdcMambaLM(dm, n_layers, ds, H, vocab_size=vocab, chunk_size=C)
    for i, blk in enumerate(lm.backbone.layers):
        reinit_block_(blk, seed=seed + i, decays_uniform=True)
    return lm.eval().to(dtype)


def _state(lm):
    """The state_dict of the unquantised model with the weights that lm holds, fp32 values on the CPU."""
    sd = {}
    for name, m in lm.named_modules():
        if isinstance(m, hm.Linear4Bit):
            sd[name + ".weight"] = m.weight4.dequantize(F32).cpu()
            if m.bias is not None:
                sd[name + ".bias"] = m.bias.detach().cpu()
    for k, v in lm.state_dict().items():
        if not k.endswith((".packed", ".scales", ".zeros")):
            sd.setdefault(k, v.detach().cpu())
    return sd


@pytest.mark.parametrize("dtype,group,zeros,B,dm,ds,H,C,n_pre,n_dec", [
    (F32, 64, True, 3, 256, 64, 8, 16, 40, 20),
    (BF, 128, False, 2, 512, 128, 8, 64, 130, 70),    # two chunk ends, padded prefill
    (BF, 32, True, 17, 256, 64, 4, 64, 64, 5),        # more rows than the unquantised step kernels take
    (BF, 128, False, 1, 768, 64, 8, 64, 200, 9),      # a ragged last group in out_proj
])
def test_quantized_block_matches_oracle(dev, dtype, group, zeros, B, dm, ds, H, C, n_pre, n_dec):
    _say("quantized block", dtype, group, zeros, B, dm, ds, H, C, n_pre, n_dec)
    torch.manual_seed(dm)
    blk = reinit_block_(hm.HdcMamba9v3Block(dm, ds, H, C), seed=dm, decays_uniform=True).eval().to(dtype).to(dev)
    hm.quantize_4bit(blk, group, zero_points=zeros)
    assert blk.weights_4bit and "packed" in dict(blk.in_proj.named_buffers())
    x = torch.randn(B, n_pre + n_dec, dm, generator=torch.Generator().manual_seed(B)).to(dtype)
    # the forward multiplies by the weight in x's type, the steps by the codes: one oracle for both within bf16's 2e-2
    sd = {k: v.to(dtype) for k, v in _state(blk).items()}
    ref = oracle.block_forward_stream(sd, x, oracle.BlockCfg(dm, ds, H, C), n_pre)
    xd = x.to(dev)
    with torch.no_grad():
        y0, st = blk.prefill(xd[:, :n_pre])
        y = blk(xd[:, :n_pre])[0]
        ys = torch.stack([blk.step(xd[:, n_pre + t].contiguous(), st) for t in range(n_dec)], 1)
    _say("  decode max rel", max_rel(ys, ref[:, n_pre:]))
    check = assert_close if dtype == F32 else assert_close_normwise
    check(y0, ref[:, :n_pre], dtype, "prefill rows")
    check(ys, ref[:, n_pre:], dtype, "decode rows")
    assert torch.equal(y, y0)


def test_quantized_lm_matches_oracle(dev):
    _say("quantized lm")
    dm, ds, H, C, n_pre, n_dec = 256, 64, 4, 32, 50, 20
    lm = _lm(dm, ds, H, C, 3, 1003, F32).to(dev)
    hm.quantize_4bit(lm, 64, zero_points=True)
    assert isinstance(lm.lm_head, hm.Linear4Bit) and lm.embedding.weight.shape == (1003, dm)
    sd = _state(lm)
    ids = torch.randint(0, 1003, (2, n_pre + n_dec), generator=torch.Generator().manual_seed(2))
    # the oracle's head is the embedding's: its hidden rows are taken before it and multiplied by the held head
    hidden = oracle.model_forward({k[len("backbone."):]: v for k, v in sd.items() if k.startswith("backbone.")},
                                  sd["embedding.weight"][ids], oracle.BlockCfg(dm, ds, H, C), 3, n_prefill=n_pre)
    hidden = torch.nn.functional.layer_norm(hidden, (dm,), sd["norm_f.weight"], sd["norm_f.bias"])
    ref = hidden @ sd["lm_head.weight"].t()
    idd = ids.to(dev)
    last, states = lm.prefill(idd[:, :n_pre])
    steps = torch.stack([lm.step(idd[:, n_pre + t].contiguous(), states) for t in range(n_dec)], 1)
    assert_close_normwise(last[:, -1], ref[:, n_pre - 1], F32, "prefill last logits")
    assert_close_normwise(steps, ref[:, n_pre:], F32, "decode logits")
    with torch.no_grad():
        full = lm(idd[:, :n_pre])
        # a copy, a move and a state_dict keep the weights
        rows = torch.randn(2, dm, device=dev)
        assert torch.equal(copy.deepcopy(lm.lm_head)(rows), lm.lm_head(rows))
        lm.cpu().to(dev)
        assert torch.equal(lm(idd[:, :n_pre]), full)
        fresh = hm.quantize_4bit(_lm(dm, ds, H, C, 3, 1003, F32, seed=5).to(dev), 64, zero_points=True)
        assert not torch.equal(fresh(idd[:, :n_pre]), full)
        fresh.load_state_dict(lm.state_dict())
        assert torch.equal(fresh(idd[:, :n_pre]), full)
        # many rows go through the weight brought back
        assert_close_normwise(lm.lm_head(torch.ones(300, dm, device=dev)), lm.lm_head(torch.ones(2, dm, device=dev))[:1].expand(300, -1),
                              F32, "head of many rows")


def test_quantized_model_is_inference_only(dev):
    blk = hm.quantize_4bit(hm.HdcMamba9v3Block(256, 64, 4, 16).eval().to(dev))
    x = torch.randn(1, 16, 256, device=dev)
    with pytest.raises(RuntimeError, match="inference"):
        blk(x)
    with torch.no_grad():
        blk(x)
        with pytest.raises(RuntimeError, match="inference"):
            blk.train()(x)
    again = blk.in_proj
    assert hm.quantize_4bit(blk).in_proj is again


@pytest.mark.parametrize("quantized", [False, True])
def test_forward_graph_of_quantized_lm(dev, quantized):
    lm = _lm(256, 64, 4, 32, 2, 500, BF).to(dev)
    if quantized:
        hm.quantize_4bit(lm)
    ids = torch.randint(0, 500, (2, 96), generator=torch.Generator().manual_seed(3)).to(dev)
    fg = lm.capture_forward(ids)
    for s in range(3):
        i = ids.roll(s, 1)
        with torch.no_grad():
            want = lm(i)
        got = fg(i).clone()
        torch.cuda.synchronize()
        assert torch.equal(got, want) or max_rel(got, want) < 1e-3


def _expected(logits, history, c):
    """(tokens, margins): the formula on the CPU in fp32, operation by operation, and how far the best value is
    ahead of the second."""
    z = logits.float().cpu()
    h = history.cpu().int()
    n = (h & 0x7FFF).float()
    col = lambda t: t.cpu()[:, None] if isinstance(t, torch.Tensor) else torch.tensor(float(t))  # noqa: E731
    z = torch.where(h != 0, torch.where(z > 0, z / col(c["repetition"]), z * col(c["repetition"])), z)
    z = z - col(c["frequency"]) * n
    z = z - torch.where(n > 0, col(c["presence"]), torch.tensor(0.0))
    z = z + c["bias"].cpu()
    V = z.shape[1]
    at = torch.arange(V)
    z = torch.where((c["mask"].cpu()[:, at // 32] >> (at % 32).int()) & 1 != 0, z, float("-inf"))
    t = c["temperature"].cpu()[:, None]
    z = torch.where(t > 0, z / torch.where(t > 0, t, 1.0) + c["noise"].cpu(), z)
    return torch.where(z == z.amax(1, keepdim=True), at, V).amin(1)


@pytest.mark.parametrize("quantized", [False, True])
def test_recorded_generation(dev, quantized):
    """Prefill, then replays that decode, choose under every control and count, over a chunk end, the mask and the
    noise changed in place between the replays: each token is the formula's for the step's logits, the history
    holds what was chosen, and the states equal those of eager steps fed the same tokens."""
    from hdcmamba_amd.lm import _clone_state

    B, V, n_pre, n_dec = 3, 1003, 20, 40
    lm = _lm(256, 64, 4, 32, 2, V, BF).to(dev)
    if quantized:
        hm.quantize_4bit(lm)
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, V, (B, n_pre), generator=g).to(dev)
    last, states = lm.prefill(ids)
    eager = [_clone_state(st) for st in states]
    c = dict(history=hm.fill_token_history(hm.new_token_history(B, V, dev), ids), repetition=torch.tensor([1.3, 1.0, 0.8], device=dev),
             frequency=0.4, presence=torch.tensor([0.3, 0.0, -0.2], device=dev), bias=torch.randn(V, generator=g).to(dev),
             mask=torch.zeros(B, -(-V // 32), dtype=torch.int32, device=dev), temperature=torch.tensor([0.0, 0.8, 1.2], device=dev),
             noise=torch.zeros(B, V, device=dev))
    graph = lm.capture_decode(states, c)
    assert not (c["history"] & 0x7FFF).any()  # the recording counted nothing
    token = last[:, -1].argmax(1)
    graph.ids.copy_(token)
    for i in range(n_dec):
        c["mask"].copy_(torch.randint(-2**31, 2**31, c["mask"].shape, generator=g, dtype=torch.int64).to(torch.int32))
        c["noise"].copy_(-torch.log(-torch.log(torch.rand(B, V, generator=g).clamp(1e-6, 1 - 1e-6))))
        before = c["history"].clone()
        got, lp = graph.next()
        got = got.clone()
        torch.cuda.synchronize()
        want = lm.step(token, eager)
        assert torch.equal(graph.logits, want) or max_rel(graph.logits, want) < 1e-3, i
        assert torch.equal(got.cpu(), _expected(graph.logits, before, c)), i
        assert torch.equal(graph.ids, got) and lp.isfinite().all()
        counts = before.clone()
        counts[torch.arange(B), got] += 1
        assert torch.equal(counts, c["history"]), i
        token = got
    assert states[0].pos == eager[0].pos == (n_pre + (32 - n_pre % 32) % 32 + n_dec) % 32
    for a, b in zip(states, eager):
        torch.testing.assert_close(a.h, b.h, atol=1e-3, rtol=1e-3)
    with pytest.raises(RuntimeError, match="controls"):
        lm.capture_decode([_clone_state(st) for st in states]).next()


def test_generate(dev):
    B, V = 2, 700
    lm = hm.quantize_4bit(_lm(256, 64, 4, 32, 2, V, BF).to(dev))
    ids = torch.randint(0, V, (B, 10), generator=torch.Generator().manual_seed(4)).to(dev)
    greedy, lp = lm.generate(ids, 12)
    assert greedy.shape == lp.shape == (B, 12) and (lp <= 0).all()
    assert torch.equal(greedy, lm.generate(ids, 12)[0]) and torch.equal(greedy[:, :1], lm.generate(ids, 1)[0])
    last, states = lm.prefill(ids)
    tok = last[:, -1].float().argmax(1)
    for i in range(12):  # the greedy tokens are the eager steps' (up to values that close to each other)
        top = (last[:, -1] if i == 0 else logits).float().topk(2).values
        sure = top[:, 0] - top[:, 1] > 1e-2 * top[:, 0].abs()
        assert torch.equal(greedy[:, i][sure], tok[sure])
        logits = lm.step(greedy[:, i].contiguous(), states)
        tok = logits.float().argmax(1)
    seeded = lambda s: torch.Generator(device=dev).manual_seed(s)  # noqa: E731
    a, b, c = (lm.generate(ids, 12, temperature=1.0, generator=seeded(s))[0] for s in (1, 1, 2))
    assert torch.equal(a, b) and not torch.equal(a, c)
    allowed = torch.zeros(B, V, dtype=torch.bool)
    allowed[:, 5::7] = True
    pad = torch.zeros(B, -(-V // 32) * 32, dtype=torch.bool)
    pad[:, :V] = allowed
    mask = (pad.view(B, -1, 32).long() << torch.arange(32)).sum(-1).to(torch.int32).to(dev)
    out, _ = lm.generate(ids, 12, temperature=torch.tensor([0.0, 1.0], device=dev), mask=mask, repetition=1.2, presence=5.0)
    assert (out % 7 == 5).all() and all(len(set(row)) > 6 for row in out.tolist())  # the presence penalty spreads them
    assert lm.generate(ids, 0)[0].shape == (B, 0)


def test_generate_with_nothing_allowed(dev):
    """A sequence whose mask leaves nothing goes on with token -1, the other as without it."""
    V = 300
    lm = _lm(256, 64, 4, 32, 1, V, BF).to(dev)
    ids = torch.randint(0, V, (2, 5), generator=torch.Generator().manual_seed(1)).to(dev)
    mask = torch.full((2, -(-V // 32)), -1, dtype=torch.int32, device=dev)
    mask[0] = 0
    tokens, lp = lm.generate(ids, 6, mask=mask, presence=0.5)
    assert (tokens[0] == -1).all() and (lp[0] == -float("inf")).all()
    assert torch.equal(tokens[1], lm.generate(ids, 6, presence=0.5)[0][1])


def test_quantized_block_refuses_tangents(dev):
    from torch.autograd import forward_ad

    lm = hm.quantize_4bit(_lm(256, 64, 4, 32, 1, 100, BF).to(dev))
    blk = lm.backbone.layers[0]
    x = torch.randn(2, 32, 256, device=dev).to(BF)
    with forward_ad.dual_level(), torch.no_grad():
        d = forward_ad.make_dual(x, x.clone())
        for call in (lambda: blk(d), lambda: lm.backbone(d), lambda: lm.backbone.prefill(d),
                     lambda: blk.step(forward_ad.make_dual(x[:, 0].clone(), x[:, 1].clone()), blk.new_state(2, dev, BF))):
            with pytest.raises(RuntimeError, match="inference"):
                call()
        assert lm.backbone(x).shape == x.shape


@pytest.mark.parametrize("quantized", [False, True])
def test_fp32_blocks_under_bf16_autocast(dev, quantized):
    """Inference of an fp32 model in a bf16 autocast region: the blocks compute in their rows' type, as outside of it (a
    product in another type would hand the kernels around it what they read as fp32)."""
    _say("fp32 blocks under autocast", quantized)
    lm = _lm(256, 64, 4, 32, 2, 300, F32).to(dev)
    if quantized:
        hm.quantize_4bit(lm, 64)
    x = torch.randn(2, 70, 256, generator=torch.Generator().manual_seed(1)).to(dev)

    def run():
        y, states = lm.backbone.prefill(x[:, :40])
        return [lm.backbone(x), y, *(lm.backbone.step(x[:, 40 + i].contiguous(), states) for i in range(3)), lm.backbone.layers[0](x)[0]]

    with torch.no_grad():
        want = run()
        with torch.amp.autocast("cuda", dtype=BF):
            got = run()
    for a, b in zip(got, want):
        assert a.dtype == F32
        assert_close(a, b.cpu(), F32, "under autocast")


def test_a_forward_brings_each_weight_back_once(dev, monkeypatch):
    """The native path and the composition (with and without the folded LayerNorm): two weights a block, no more."""
    blk = hm.quantize_4bit(_lm(256, 64, 4, 32, 1, 50, BF).to(dev)).backbone.layers[0]
    calls, plain = [], hm.Weight4Bit.dequantize
    monkeypatch.setattr(hm.Weight4Bit, "dequantize", lambda self, dtype: calls.append(self.shape) or plain(self, dtype))
    x = torch.randn(1, 64, 256, device=dev).to(BF)
    shapes = [blk.in_proj.weight4.shape, blk.out_proj.weight4.shape]
    with torch.no_grad():
        for native in (True, False):
            if not native:
                monkeypatch.setattr(blk, "_native_ok", lambda x: False)
            for fused in (True, False):
                hm.set_fused_out_proj(blk, fused)
                calls.clear()
                blk(x)
                assert sorted(calls) == sorted(shapes), (native, fused)


@pytest.mark.parametrize("change", ["quantize", "move", "move a quantized"])
def test_recordings_outlive_the_weights_of_the_module(dev, change):
    """A model that gets other weights, and memory that is used again: earlier recordings replay on theirs."""
    from hdcmamba_amd.lm import _clone_state

    lm = _lm(256, 64, 4, 32, 2, 500, BF).to(dev)
    if change == "move a quantized":
        hm.quantize_4bit(lm)
    ids = torch.randint(0, 500, (2, 64), generator=torch.Generator().manual_seed(3)).to(dev)
    _, states = lm.prefill(ids)
    start = [_clone_state(st) for st in states]
    fg, dg = lm.capture_forward(ids), lm.capture_decode(states)
    want = fg(ids).clone(), dg.step(ids[:, 0]).clone()
    for a, b in zip(states, start):
        for name in ("conv", "h", "S_prev", "S_intra"):
            getattr(a, name).copy_(getattr(b, name))
    dg.pos.fill_(start[0].pos)
    torch.cuda.synchronize()
    sizes = [t.numel() for m in (lm, lm.backbone) for t in (*m.parameters(), *m.buffers())]
    if change == "quantize":
        hm.quantize_4bit(lm)
    else:
        lm.cpu().to(dev)
        with torch.no_grad():  # and other values, which a forward uses
            for p in (*lm.parameters(), *(m.scales for m in lm.modules() if isinstance(m, hm.Linear4Bit))):
                p.mul_(1.5)
            assert not torch.equal(lm(ids), want[0])
    junk = [torch.full((n,), float("nan"), device=dev, dtype=dt) for n in sizes for dt in (BF, F32) for _ in range(2)]
    torch.cuda.synchronize()
    assert torch.equal(fg(ids), want[0])
    assert torch.equal(dg.step(ids[:, 0]), want[1]) and len(junk) == 4 * len(sizes)


def test_out_proj_row_sums_are_finished_for_every_reader(dev):
    """An unquantised block's weight is written in place: two streams use it, the first one busy; then a recording is the
    first to use it, and an eager forward comes before the first replay."""
    blk, twin = (_lm(512, 64, 4, 32, 1, 50, BF).to(dev).backbone.layers[0] for _ in range(2))
    x = torch.randn(2, 64, 512, generator=torch.Generator().manual_seed(2)).to(BF).to(dev)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    with torch.no_grad():
        blk(x)
        assert blk._wsum is not None
        blk.out_proj.weight.mul_(-2)
        twin.out_proj.weight.mul_(-2)
        want = twin(x)[0]
        torch.cuda.synchronize()
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                if i == 0:
                    torch.cuda._sleep(20_000_000)
                got.append(blk(x)[0])
        torch.cuda.synchronize()
        assert torch.equal(got[0], want) and torch.equal(got[1], want)
        blk.out_proj.weight.mul_(4)
        twin.out_proj.weight.mul_(4)
        want = twin(x)[0]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = blk(x)[0]
        assert torch.equal(blk(x)[0], want)
        for _ in range(3):
            out.zero_()
            graph.replay()
            assert torch.equal(out, want)
            torch.cuda.synchronize()


def test_a_refused_weight_leaves_the_model_as_it_was(dev):
    lm = _lm(256, 64, 4, 32, 2, 50, BF).to(dev)
    ids = torch.randint(0, 50, (1, 32), device=dev)
    with torch.no_grad():
        want = lm(ids)
        weight = lm.backbone.layers[1].out_proj.weight
        kept = weight[3, 5].clone()
        weight[3, 5] = float("nan")
        with pytest.raises(ValueError, match="infinities"):
            hm.quantize_4bit(lm)
        weight[3, 5] = kept
        assert not any(isinstance(m, hm.Linear4Bit) for m in lm.modules()) and torch.equal(lm(ids), want)
        assert sum(isinstance(m, hm.Linear4Bit) for m in hm.quantize_4bit(lm).modules()) == 5


def test_quantized_step_without_the_folded_layer_norm(dev, monkeypatch):
    """set_fused_out_proj(False): the LayerNorm in a pass of its own, the same step within bf16."""
    from hdcmamba_amd import model

    eps, plain = [], model.linear_4bit
    monkeypatch.setattr(model, "linear_4bit", lambda *a, norm_eps=None, **kw: eps.append(norm_eps) or plain(*a, norm_eps=norm_eps, **kw))
    blk = hm.quantize_4bit(_lm(256, 64, 4, 32, 1, 50, BF).to(dev)).backbone.layers[0]
    x = torch.randn(3, 256, generator=torch.Generator().manual_seed(1)).to(BF).to(dev)
    got = []
    with torch.no_grad():
        for fused in (True, False):
            hm.set_fused_out_proj(blk, fused)
            eps.clear()
            got.append(blk.step(x, blk.new_state(3, dev, BF)))
            assert eps == [None, 1e-5 if fused else None]
    assert_close_normwise(got[0], got[1].cpu(), BF, "step")


def test_recordings_are_made_on_the_models_device(dev, monkeypatch):
    """torch records on one stream of the process by default, which lies on the device that recorded first: the model's
    recordings name a stream of its own device."""
    plain, seen = torch.cuda.graph, []
    monkeypatch.setattr(torch.cuda, "graph", lambda g, stream=None: seen.append(stream) or plain(g, stream=stream))
    lm = _lm(256, 64, 4, 32, 1, 50, BF).to(dev)
    ids = torch.randint(0, 50, (1, 32), device=dev)
    lm.capture_forward(ids)
    lm.generate(ids, 3)
    assert len(seen) == 2 and all(s is not None and s.device == dev for s in seen)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_generate_on_another_device():
    lm, ids = _lm(256, 64, 4, 32, 1, 50, BF), torch.randint(0, 50, (2, 32))
    want = [t.cpu() for t in lm.to("cuda:0").generate(ids.to("cuda:0"), 5, presence=0.5)]
    got = [t.cpu() for t in lm.to("cuda:1").generate(ids.to("cuda:1"), 5, presence=0.5)]
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_prefill_of_a_quantized_model_in_training_mode(dev):
    """A prefill is inference whatever the module's mode."""
    lm = hm.quantize_4bit(_lm(256, 64, 4, 32, 1, 50, BF).to(dev))
    ids = torch.randint(0, 50, (1, 40), device=dev)
    want = lm.prefill(ids)[0]
    assert torch.equal(lm.train().prefill(ids)[0], want)


@pytest.mark.parametrize("quantized", [False, True])
def test_a_recording_replays_while_the_model_is_elsewhere(dev, quantized):
    lm = _lm(512, 64, 4, 32, 1, 100, BF).to(dev)
    if quantized:
        hm.quantize_4bit(lm)
    ids = torch.randint(0, 100, (2, 64), device=dev)
    fg, dg = lm.capture_forward(ids), lm.capture_decode(lm.prefill(ids)[1])
    want = fg(ids).clone()
    lm.cpu()
    assert torch.equal(fg(ids), want) and dg.step(ids[:, 0]).isfinite().all()
    lm.to(dev)
    assert torch.equal(fg(ids), want)


@pytest.mark.parametrize("quantized", [False, True])
def test_models_made_under_inference_mode(dev, quantized):
    """Construction, rounding, forward, generation and recordings under inference mode, and the forward outside of it; an
    in-place write, which such tensors do not count, is seen."""
    with torch.inference_mode():
        lm = _lm(256, 64, 4, 32, 2, 300, BF).to(dev)
        if quantized:
            hm.quantize_4bit(lm)
        ids = torch.randint(0, 300, (2, 64), device=dev)
        want = lm(ids)
        fg = lm.capture_forward(ids)
        assert torch.equal(fg(ids), want)
        assert lm.generate(ids, 4, temperature=0.7, presence=0.5)[0].shape == (2, 4)
        out = lm.backbone.layers[0].out_proj
        write = out.scales if quantized else out.weight
        write.mul_(2)
        changed = lm(ids)
        assert not torch.equal(changed, want)
        write.mul_(0.5)
        assert torch.equal(lm(ids), want)
    with torch.no_grad():
        assert torch.equal(lm(ids), want)
