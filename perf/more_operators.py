"""The operators at the two ends of a training step of the HdcMamba framework: the lookup of token rows and its
gradient, and the global norm of all gradients with the clipping by it.

Each case is a plain dict; ``op`` names the operator:

  embed   hdcmamba_amd.embedding: rows of a weight by token id, times a scale; an id outside 0..V-1 gives zeros
  egrad   hdcmamba_amd.embedding_grad: the weight's gradient, for every token the sum of its positions' rows
  norm    hdcmamba_amd.grad_norm: the 2-norm over all tensors of a list
  clip    hdcmamba_amd.clip_grads_: a list of tensors scaled in place by min(1, max_norm / (norm + 1e-6)), the norm given
  step    hdcmamba_amd.clip_grad_norm_: both on the gradients of parameters, as a training step calls it

Gradients of a model lie one behind the other in a buffer for each type, as data-parallel training keeps them; the
list that the operators get holds the views of the single parameters.

With ``own`` false, ``run`` computes everything in elementary torch operations in 32 bits, long sums in 64.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _embed(dtype, B, L, D, V, scale=1.0, ids="int64", padded=0.0):
    """padded: the share of positions behind the sequences' ends, whose id is -1."""
    return dict(op="embed", dtype=dtype, B=B, L=L, D=D, V=V, scale=scale, ids=ids, padded=padded)


def _egrad(dtype, B, L, D, V, scale=1.0, padding_idx=-1, padded=0.0):
    """padded: the share of positions behind the sequences' ends: id 0, their gradient zero.  padding_idx -1: none."""
    return dict(op="egrad", dtype=dtype, B=B, L=L, D=D, V=V, scale=scale, padding_idx=padding_idx, padded=padded)


def _model(op, dtype, layers, d_model, d_state, heads, V, norm=0.5):
    """dtype "mixed": matrices in bf16, the rest in fp32.  norm: about that of the gradients; the limit is 1."""
    return dict(op=op, dtype=dtype, layers=layers, d_model=d_model, d_state=d_state, heads=heads, V=V, norm=norm)


def listed():
    return [
        # one token for each of sixteen sequences, d_model 2048: a decode step's lookup
        dict(_embed("bf16", 16, 1, 2048, 50304), name="embed_step"),
        # a right-padded batch of two sequences, fp32, rows scaled by sqrt(d_model), 32-bit ids
        dict(_embed("fp32", 2, 3001, 768, 50277, scale=768 ** 0.5, ids="int32", padded=0.2), name="embed_ragged"),
        # the long sequence of the 24-layer model
        dict(_embed("bf16", 1, 32768, 1024, 50304), name="embed_long"),
        # a small model's step
        dict(_egrad("bf16", 2, 192, 256, 1024), name="egrad_small"),
        # a model of characters: every token's sum has hundreds of rows
        dict(_egrad("fp32", 64, 256, 512, 65), name="egrad_chars"),
        # the training step of the 24-layer model on its long sequence
        dict(_egrad("bf16", 1, 32768, 1024, 50304), name="egrad_long"),
        # a large right-padded batch of the d_model 2048 model without a padding index: a quarter of all positions is one token
        dict(_egrad("bf16", 16, 8192, 2048, 50304, padded=0.25), name="egrad_padded"),
        # a two-layer model in fp32: two dozen small tensors
        dict(_model("norm", "fp32", 2, 256, 64, 4, 1024), name="norm_small"),
        # the 42-layer, d_model 2048 model in bf16: 10^9 elements in 420 tensors
        dict(_model("norm", "bf16", 42, 2048, 128, 32, 50277), name="norm_1b"),
        # two-layer model, a norm over several ranks a little above the limit
        dict(_model("clip", "fp32", 2, 256, 64, 4, 1024, norm=1.0005), name="clip_small"),
        # the same for the 24-layer model with fp32 gradients
        dict(_model("clip", "fp32", 24, 1024, 128, 16, 50304, norm=1.0005), name="clip_long"),
        # the 24-layer model's bf16 gradients in a step whose norm is within the limit, as most steps' are
        dict(_model("step", "bf16", 24, 1024, 128, 16, 50304), name="step_long"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "egrad", "egrad", "egrad", "norm", "clip", "step"])
    if op in ("embed", "egrad"):
        D, V, B = _log_int(rng, 32, 2304), _log_int(rng, 65, 131072), _log_int(rng, 1, 16)
        if rng.random() < 0.7:  # most widths are whole vectors
            D = max(32, D // 32 * 32)
        L = max(1, min(_log_int(rng, 1, 131072), 131072 * 2048 // max(D, 512)) // B)
        dtype, scale = rng.choice(["bf16", "bf16", "fp32"]), rng.choice([1.0, 1.0, D ** 0.5])
        padded = rng.choice([0.0, 0.0, round(rng.uniform(0.02, 0.5), 2)])
        V = min(V, 50304 * 2048 // D)
        if dtype == "fp32":
            L, V = max(1, L // 2), max(65, V // 2)
        if op == "embed":
            return _embed(dtype, B, L, D, V, scale, rng.choice(["int64", "int32"]), padded)
        return _egrad(dtype, B, L, D, V, scale, rng.choice([-1, -1, 0, V - 1]), padded)
    d, V = 64 * _log_int(rng, 1, 32), _log_int(rng, 65, 65536)
    ds, dtype = rng.choice([16, 64, 128]), rng.choice(["bf16", "fp32", "mixed"])
    most = 1_900_000_000 // ((4 if dtype == "fp32" else 2) * (2 if op == "clip" else 1)) - V * d
    layers = max(1, min(_log_int(rng, 1, 48), most // (5 * d * d + 4 * ds * d + 13 * d)))
    # a norm above the limit is drawn where it is given: a step's second pass would find its gradients clipped already
    norm = 0.5 if op != "clip" else 1.0005 if dtype == "fp32" else 1.02
    return _model(op, dtype, layers, d, ds, max(1, d // rng.choice([32, 64, 64, 128])), V, norm)


# ------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _tokens(g, V, *shape):
    """Token ids as text has them: the k-th most frequent about 1/k as often as the first."""
    u = torch.rand(*shape, generator=g, device=DEV, dtype=torch.float64)
    return (torch.exp(u * math.log(V + 1)).long() - 1).clamp_(0, V - 1)


def _behind_ends(g, c):
    """[B, L], true behind the end of each sequence: from none to twice the share of positions."""
    ends = c["L"] * (1 - 2 * c["padded"] * torch.rand(c["B"], 1, generator=g, device=DEV)).clamp_(min=0)
    return torch.arange(c["L"], device=DEV) >= ends.ceil()


def _embed_inputs(c, seed):
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    ids = _tokens(g, c["V"], c["B"], c["L"])
    if c["padded"]:
        ids = ids.masked_fill(_behind_ends(g, c), -1)
    weight = torch.empty(c["V"], c["D"], device=DEV, dtype=dt).normal_(0, 0.04, generator=g)
    return dict(ids=ids.to(torch.int32) if c["ids"] == "int32" else ids, weight=weight, scale=c["scale"])


def _egrad_inputs(c, seed):
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    ids = _tokens(g, c["V"], c["B"], c["L"])
    grad = torch.empty(c["B"], c["L"], c["D"], device=DEV, dtype=dt).normal_(0, 1e-3, generator=g)
    if c["padded"]:
        behind = _behind_ends(g, c)
        ids = ids.masked_fill(behind, 0)
        grad.masked_fill_(behind[:, :, None], 0)
    return dict(ids=ids, grad=grad, V=c["V"], scale=c["scale"], padding_idx=None if c["padding_idx"] < 0 else c["padding_idx"])


def _shapes(c):
    """The shapes of the parameters that have a gradient: embedding, layers, the two final norms."""
    d, ds = c["d_model"], c["d_state"]
    layer = [(d,), (d,), (d, 1, 4), (d,), (3 * ds + 4 * d, d), (3 * ds + 4 * d,), (ds,), (d, ds + d), (d,), (d,)]
    return [(c["V"], d)] + layer * c["layers"] + [(d,)] * 4


def _places(c):
    """(type, shape, first element in the type's buffer) of every parameter, at multiples of 8 elements; the buffers' lengths."""
    ends, at = {}, []
    for shape in _shapes(c):
        kind = c["dtype"] if c["dtype"] != "mixed" else "bf16" if len(shape) == 2 else "fp32"
        begin = ends.get(kind, 0)
        at.append((kind, shape, begin))
        ends[kind] = begin + -(-math.prod(shape) // 8) * 8
    return at, ends


def _model_inputs(c, seed):
    g = _gen(seed)
    places, ends = _places(c)
    count = sum(math.prod(shape) for _, shape, _ in places)
    share = 0.5 if c["op"] == "clip" else c["norm"]  # where the norm is given these are one rank's gradients
    flat = {k: torch.empty(n, device=DEV, dtype=DTYPES[k]).normal_(0, share / count ** 0.5, generator=g) for k, n in ends.items()}
    grads = []
    for kind, shape, begin in places:
        n = math.prod(shape)
        grads.append(flat[kind][begin:begin + n].view(shape))
        if n % 8:  # what lies between the parameters is zero
            flat[kind][begin + n:begin + n + 8 - n % 8] = 0
    return dict(flat=[flat[k] for k in sorted(flat)], grads=grads, norm=torch.tensor(c["norm"], device=DEV))


_INPUTS = {"embed": _embed_inputs, "egrad": _egrad_inputs, "norm": _model_inputs, "clip": _model_inputs, "step": _model_inputs}


def prepare(case, seed):
    state = dict(_INPUTS[case["op"]](case, seed), op=case["op"])
    if case["op"] == "step":  # the parameters whose gradients these are
        state["params"] = [torch.nn.Parameter(torch.zeros_like(t)) for t in state["grads"]]
        for p, t in zip(state["params"], state["grads"]):
            p.grad = t
    return state


# ------------------------------------------------------------------------------- plain forms
def _plain_embed(s):
    ids, w = s["ids"].long(), s["weight"]
    there = (ids >= 0) & (ids < w.shape[0])
    rows = w[torch.where(there, ids, 0)].float() * s["scale"]
    return torch.where(there[..., None], rows, 0.0).to(w.dtype)


def _plain_egrad(s):
    grad, V = s["grad"].flatten(0, 1), s["V"]
    ids = s["ids"].flatten()
    if s["padding_idx"] is not None:
        ids = torch.where(ids == s["padding_idx"], V, ids)  # a row that is dropped
    # a frequent token's sum has thousands of rows: in 64 bits where the result keeps 24
    total = torch.zeros(V + 1, grad.shape[1], device=DEV, dtype=torch.float64 if grad.dtype == torch.float32 else torch.float32)
    total.index_add_(0, ids, grad.to(total.dtype))
    return (total[:V] * s["scale"]).to(grad.dtype)


def _plain_norm(s):
    squares = [t.float().square().sum(dtype=torch.float64) for t in s["flat"]]
    return torch.stack(squares).sum().sqrt().float()


def _plain_clip(s, norm):
    factor = (1.0 / (norm + 1e-6)).clamp(max=1.0)
    return [t.copy_(t.float() * factor) for t in s["flat"]]


# ------------------------------------------------------------------------------- the calls
def run(state):
    s, op = state, state["op"]
    if not own:
        if op == "embed":
            return _plain_embed(s)
        if op == "egrad":
            return _plain_egrad(s)
        if op == "clip":
            return _plain_clip(s, s["norm"])
        norm = _plain_norm(s)
        return norm if op == "norm" else (norm, _plain_clip(s, norm))
    import hdcmamba_amd as hm

    if op == "embed":
        return hm.embedding(s["ids"], s["weight"], scale=s["scale"])
    if op == "egrad":
        return hm.embedding_grad(s["ids"], s["grad"], s["V"], scale=s["scale"], padding_idx=s["padding_idx"])
    if op == "norm":
        return hm.grad_norm(s["grads"])
    if op == "clip":
        hm.clip_grads_(s["grads"], 1.0, s["norm"])
        return s["flat"]
    return hm.clip_grad_norm_(s["params"], 1.0), s["flat"]


# ------------------------------------------------------------------------------- work and exact values
def _distinct(c):
    """How many rows of the weight the ids are expected to name."""
    k = torch.arange(1, c["V"] + 1, dtype=torch.float64)
    p = torch.log1p(1 / k) / math.log(c["V"] + 1)
    return float((1 - (1 - p) ** (c["B"] * c["L"] * (1 - c["padded"]))).sum())


def work(case):
    c = case
    if c["op"] in ("embed", "egrad"):
        T, D, e = c["B"] * c["L"], c["D"], DTYPES[c["dtype"]].itemsize
        if c["op"] == "embed":
            return {"bytes": _distinct(c) * D * e + T * D * e + T * (4 if c["ids"] == "int32" else 8), "flops": 1.0 * T * D}
        return {"bytes": T * D * e + c["V"] * D * e + 8.0 * T, "flops": 1.0 * (T + c["V"]) * D}
    places, _ = _places(c)
    size = sum(math.prod(shape) * DTYPES[kind].itemsize for kind, shape, _ in places)
    count = sum(math.prod(shape) for _, shape, _ in places)
    if c["op"] == "norm":
        return {"bytes": size, "flops": 2.0 * count}
    if c["op"] == "clip":
        return {"bytes": 2.0 * size, "flops": 1.0 * count}
    clipped = c["norm"] > 1
    return {"bytes": size * (2.0 if clipped else 1.0), "flops": count * (3.0 if clipped else 2.0)}


def _exact_embed(c, s):
    ids, w = s["ids"].flatten().long(), s["weight"].double()
    out = torch.zeros(ids.numel(), c["D"], device=DEV, dtype=torch.float64)
    named = ((ids >= 0) & (ids < c["V"])).nonzero()[:, 0]
    out[named] = w.index_select(0, ids[named]) * c["scale"]
    return out.view(c["B"], c["L"], c["D"])


def _exact_egrad(c, s):
    """Positions in the order of their tokens, a part of the columns at a time: each token's sum is a segment's."""
    ids, grad = s["ids"].flatten(), s["grad"].flatten(0, 1)
    order = torch.argsort(ids, stable=True)
    lengths = torch.bincount(ids, minlength=c["V"])
    parts = [torch.segment_reduce(grad[:, k:k + 256][order].double(), "sum", lengths=lengths, axis=0, initial=0)
             for k in range(0, c["D"], 256)]
    out = torch.cat(parts, 1) * c["scale"]
    if s["padding_idx"] is not None:
        out[s["padding_idx"]] = 0
    return out


def _exact_norm(s):
    return torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(t.double()) for t in s["grads"]]))


def exact(case, seed):
    s = _INPUTS[case["op"]](case, seed)
    if case["op"] == "embed":
        return _exact_embed(case, s)
    if case["op"] == "egrad":
        return _exact_egrad(case, s)
    if case["op"] == "norm":
        return _exact_norm(s)
    norm = s["norm"].double() if case["op"] == "clip" else _exact_norm(s)
    scaled = [t.double() * min(1.0, 1 / (float(norm) + 1e-6)) for t in s["flat"]]
    return scaled if case["op"] == "clip" else (norm, scaled)
