"""Calls around the token rows, the gradients' norm and clipping that the operators' own tests leave out: ids outside the
vocabulary through the whole model, lookups that go past the kernels, gradients of every kind, and the largest lists."""
import copy

import pytest
import torch
import torch.nn as nn

import hdcmamba_amd as hm
from cfgs import reinit_block_

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float32


def _say(*a):
    print(*a, flush=True)


def gen(seed):
    return torch.Generator().manual_seed(seed)


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
