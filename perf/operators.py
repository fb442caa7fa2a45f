"""The decode-side operators of the HdcMamba framework: what a program that generates text calls per step.

Each case is a plain dict; ``op`` names the operator:

  linear    hdcmamba_amd.linear_4bit: rows of activations times a 4-bit weight with group scales
  process   hdcmamba_amd.process_logits: repetition, frequency and presence penalties, a bias and a
            grammar mask on a batch of logits
  select    hdcmamba_amd.select_tokens: the same, then temperature, noise, the largest value's index
            and its log-probability, without writing the processed logits
  history   hdcmamba_amd.fill_token_history: which tokens a sequence holds, from its prompt and output

Weights are w[n, k] = scale[n, g] (code[n, k] - zero[n, g]) with codes 0..15 and g = k // group; without
zero points the zero is 8.  A token history is an int16 per (sequence, token): the sign bit is set for
tokens of the prompt, the low 15 bits count the token in the output (up to 32767).

With ``own`` false, ``run`` computes everything in elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _linear(dtype, M, K, N, group, zeros=False, bias=False, residual=False, scales="bf16"):
    return dict(op="linear", dtype=dtype, M=M, K=K, N=N, group=group, zeros=zeros, bias=bias, residual=residual,
                scales=scales)


def _logits(op, dtype, B, V, penalties=True, bias="", mask=True, sampled=False):
    """bias: "" none, "shared" one row for all sequences (fp32), "rows" one per sequence (the logits' type)."""
    case = dict(op=op, dtype=dtype, B=B, V=V, penalties=penalties, bias=bias, mask=mask)
    return dict(case, sampled=sampled) if op == "select" else case


def _history(B, V, prompt, output):
    return dict(op="history", B=B, V=V, prompt=prompt, output=output)


def listed():
    return [
        # one sequence generating: out_proj of a d_model 1024 layer (d_state 128) with the residual
        dict(_linear("bf16", 1, 1152, 1024, 128, residual=True), name="linear_one"),
        # an fp32 model of d_model 768 (d_state 64), three sequences: in_proj, with zero points
        dict(_linear("fp32", 3, 768, 3264, 64, zeros=True, bias=True, scales="fp32"), name="linear_fp32"),
        # batched generation, d_model 2048: in_proj of a layer
        dict(_linear("bf16", 16, 2048, 8576, 128, bias=True), name="linear_in_b16"),
        # the head of that model, the step's largest product
        dict(_linear("bf16", 16, 2048, 50304, 128), name="linear_head_b16"),
        # a larger batch on the head of a d_model 768 model with the default vocabulary, small groups with zero points
        dict(_linear("bf16", 33, 768, 50277, 32, zeros=True), name="linear_head_ragged"),
        # a short prompt's rows at once (or a large batch): in_proj, d_model 2048
        dict(_linear("bf16", 128, 2048, 8576, 128, bias=True), name="linear_in_m128"),
        # one sequence, repetition and count penalties only
        dict(_logits("process", "bf16", 1, 50304, mask=False), name="process_one"),
        # a serving batch over the default vocabulary (odd rows): penalties, a shared bias, a grammar mask each
        dict(_logits("process", "bf16", 64, 50277, bias="shared"), name="process_b64"),
        # greedy choice under a grammar for the batch of 16
        dict(_logits("select", "bf16", 16, 50304), name="select_greedy"),
        # sampling for a large batch in fp32, biases of each sequence's own
        dict(_logits("select", "fp32", 128, 50304, bias="rows", mask=False, sampled=True), name="select_b128"),
        # a short prompt joins the batch
        dict(_history(1, 50304, 200, 0), name="history_one"),
        # sixteen long prompts with half-done outputs (the tests' 8192 and 256 tokens)
        dict(_history(16, 50304, 8192, 256), name="history_b16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "process", "select", "history"])
    if op == "linear":
        K, N = _log_int(rng, 64, 2304), _log_int(rng, 64, 50304)
        if rng.random() < 0.6:  # most widths are whole groups
            K = max(64, K // 64 * 64)
        M = min(_log_int(rng, 1, 128), max(1, 128 * 2048 * 8576 // (K * N)))
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        return _linear(dtype, M, K, N, rng.choice([32, 64, 128, 128]), zeros=rng.random() < 0.5, bias=rng.random() < 0.5,
                       residual=rng.random() < 0.3, scales=rng.choice(["bf16", "fp32"]))
    V = _log_int(rng, 500, 131072)
    if op == "history":
        B = min(_log_int(rng, 1, 64), 64 * 50304 // V)
        prompt = _log_int(rng, 1, 16384)
        return _history(B, V, prompt, rng.choice([0, 1, _log_int(rng, 2, 2048)]))
    B = min(_log_int(rng, 1, 128), 64 * 50304 // V)
    return _logits(op, rng.choice(["bf16", "fp32"]), B, V, penalties=rng.random() < 0.8, bias=rng.choice(["", "shared", "rows"]),
                   mask=rng.random() < 0.6, sampled=rng.random() < 0.5)


# ------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _uniform(g, lo, hi, *shape):
    return lo + (hi - lo) * torch.rand(*shape, generator=g, device=DEV)


def _tokens(g, V, *shape):
    """Token ids with a few frequent ones, as text has."""
    return (torch.rand(*shape, generator=g, device=DEV) ** 3 * V).long().clamp_(max=V - 1)


def _linear_inputs(c, seed):
    g = _gen(seed)
    dt, sdt = DTYPES[c["dtype"]], DTYPES[c["scales"]]
    M, K, N = c["M"], c["K"], c["N"]
    groups = -(-K // c["group"])
    # what rounding normal weights to steps of 0.4 of their deviation gives
    codes = (_randn(g, N, K) * 2.5 + 8).round_().clamp_(0, 15).to(torch.uint8)
    scales = (_uniform(g, 0.6, 1.4, N, groups) * 0.008).to(sdt)
    zeros = torch.randint(5, 12, (N, groups), generator=g, device=DEV, dtype=torch.uint8) if c["zeros"] else None
    return dict(x=_randn(g, M, K).to(dt), codes=codes, scales=scales, zeros=zeros,
                bias=_randn(g, N).to(dt) if c["bias"] else None,
                residual=_randn(g, M, N).to(dt) if c["residual"] else None)


def _logits_inputs(c, seed):
    g = _gen(seed)
    dt = DTYPES[c["dtype"]]
    B, V = c["B"], c["V"]
    s = dict(logits=(_randn(g, B, V) * 3).to(dt), history=None, repetition=None, frequency=None, presence=None, bias=None,
             mask=None, temperature=None, noise=None)
    if c["penalties"]:
        count = torch.zeros(B, V, device=DEV, dtype=torch.int32)
        ids = _tokens(g, V, B, 256)
        count.scatter_add_(1, ids, torch.ones_like(ids, dtype=torch.int32))
        count.scatter_(1, _tokens(g, V, B, 1024), -32768)  # a prompt token (its count here is 0)
        s["history"] = count.to(torch.int16)
        s["repetition"] = _uniform(g, 1.0, 1.5, B)
        s["frequency"] = _uniform(g, 0.0, 0.5, B)
        s["presence"] = _uniform(g, -0.2, 0.5, B)
    if c["bias"] == "shared":
        s["bias"] = _randn(g, V)
    elif c["bias"] == "rows":
        s["bias"] = _randn(g, B, V).to(dt)
    if c["mask"]:  # from a few allowed tokens to nearly all of them
        words = -(-V // 32)
        keep = torch.rand(B, 1, generator=g, device=DEV) ** 2 * 0.95 + 0.01
        bits = torch.rand(B, words * 32, generator=g, device=DEV) < keep
        weights = torch.ones(32, device=DEV, dtype=torch.int64) << torch.arange(32, device=DEV)
        s["mask"] = (bits.view(B, words, 32).long() * weights).sum(-1).to(torch.int32)
    if c.get("sampled"):
        s["temperature"] = _uniform(g, 0.3, 1.3, B)
        u = torch.rand(B, V, generator=g, device=DEV).clamp_(1e-20, 1 - 1e-7)
        s["noise"] = -torch.log(-torch.log(u))
    return s


def _history_inputs(c, seed):
    g = _gen(seed)
    B, V = c["B"], c["V"]
    s = dict(table=torch.zeros(B, V, device=DEV, dtype=torch.int16), prompt=_tokens(g, V, B, c["prompt"]),
             output=_tokens(g, V, B, c["output"]))
    for name in ("prompt", "output"):  # right-padded rows of several lengths
        n = c[name]
        s[name + "_lengths"] = torch.randint(n // 2, n + 1, (B,), generator=g, device=DEV)
    return s


_INPUTS = {"linear": _linear_inputs, "process": _logits_inputs, "select": _logits_inputs, "history": _history_inputs}


def prepare(case, seed):
    state = dict(_INPUTS[case["op"]](case, seed), op=case["op"])
    if case["op"] == "linear":
        state["group"] = case["group"]
        if own:  # the weight laid out once, as a loaded model keeps it
            from hdcmamba_amd import Weight4Bit

            state["weight"] = Weight4Bit.from_codes(state["codes"], state["scales"], state["zeros"], case["group"])
    return state


# ------------------------------------------------------------------------------- plain forms
def _plain_linear(s):
    K, group = s["codes"].shape[1], s["group"]
    per_k = lambda t: t.float().repeat_interleave(group, 1)[:, :K]  # noqa: E731
    zero = per_k(s["zeros"]) if s["zeros"] is not None else 8.0
    w = (s["codes"].float() - zero) * per_k(s["scales"])
    y = s["x"].float() @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _plain_processed(s):
    z = s["logits"].float()
    if s["history"] is not None:
        h = s["history"].int()
        count = (h & 0x7FFF).float()
        r = s["repetition"][:, None]
        z = torch.where(h != 0, torch.where(z > 0, z / r, z * r), z)
        z = z - s["frequency"][:, None] * count
        z = z - s["presence"][:, None] * (count > 0).float()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    if s["mask"] is not None:
        at = torch.arange(z.shape[1], device=z.device)
        allowed = (s["mask"][:, at // 32] >> (at % 32).int()) & 1
        z = torch.where(allowed != 0, z, float("-inf"))
    return z


def _plain_select(s):
    z = _plain_processed(s)
    V = z.shape[1]
    if s["temperature"] is not None:
        z = z / s["temperature"][:, None]
    v = z if s["noise"] is None else z + s["noise"]
    at = torch.arange(V, device=z.device)
    token = torch.where(v == v.amax(1, keepdim=True), at, V).amin(1)
    top = z.amax(1, keepdim=True)
    lse = (z - top).exp().sum(1).log() + top[:, 0]
    logprob = z.gather(1, token[:, None])[:, 0] - lse
    empty = top[:, 0] == float("-inf")
    return torch.where(empty, -1, token), torch.where(empty, float("-inf"), logprob)


def _plain_history(s):
    B, V = s["table"].shape
    n = {k: torch.arange(s[k].shape[1], device=s[k].device) < s[k + "_lengths"][:, None] for k in ("prompt", "output")}
    count = torch.zeros(B, V + 1, device=s["table"].device, dtype=torch.int32)
    count.scatter_add_(1, torch.where(n["output"], s["output"], V), torch.ones_like(s["output"], dtype=torch.int32))
    seen = torch.zeros(B, V + 1, device=s["table"].device, dtype=torch.bool)
    seen.scatter_(1, torch.where(n["prompt"], s["prompt"], V), True)
    table = count[:, :V].clamp(max=32767) - 32768 * seen[:, :V].int()
    return s["table"].copy_(table)


# ------------------------------------------------------------------------------- the calls
def run(state):
    s, op = state, state["op"]
    if not own:
        plain = {"linear": _plain_linear, "select": _plain_select, "history": _plain_history}
        return plain[op](s) if op in plain else _plain_processed(s).to(s["logits"].dtype)
    import hdcmamba_amd as hm

    if op == "linear":
        return hm.linear_4bit(s["x"], s["weight"], bias=s["bias"], residual=s["residual"])
    if op == "history":
        return hm.fill_token_history(s["table"], s["prompt"], s["prompt_lengths"], s["output"], s["output_lengths"])
    controls = {k: s[k] for k in ("history", "repetition", "frequency", "presence", "bias", "mask")}
    if op == "process":
        return hm.process_logits(s["logits"], **controls)
    return hm.select_tokens(s["logits"], temperature=s["temperature"], noise=s["noise"], **controls)


# ------------------------------------------------------------------------------- work and exact values
def work(case):
    c = case
    if c["op"] == "linear":
        M, K, N, e = c["M"], c["K"], c["N"], DTYPES[c["dtype"]].itemsize
        groups = N * -(-K // c["group"])
        read = N * K / 2 + groups * (DTYPES[c["scales"]].itemsize + (1 if c["zeros"] else 0)) + M * K * e
        read += (N * e if c["bias"] else 0) + (M * N * e if c["residual"] else 0)
        return {"bytes": read + M * N * e, "flops": 2.0 * M * N * K}
    B, V = c["B"], c["V"]
    if c["op"] == "history":
        return {"bytes": 2.0 * B * V + 8.0 * B * (c["prompt"] + c["output"] + 2), "flops": 1.0 * B * (c["prompt"] + c["output"])}
    e = DTYPES[c["dtype"]].itemsize
    read = B * V * e + (2 * B * V + 12 * B if c["penalties"] else 0) + (4 * B * -(-V // 32) if c["mask"] else 0)
    read += {"": 0, "shared": 4 * V, "rows": B * V * e}[c["bias"]]
    flops = B * V * (7.0 if c["penalties"] else 1.0)
    if c["op"] == "process":
        return {"bytes": read + B * V * e, "flops": flops}
    return {"bytes": read + (4 * B * V + 4 * B if c["sampled"] else 0) + 12 * B, "flops": flops + 5.0 * B * V}


def _exact_linear(c, s):
    x, q = s["x"].double(), s["codes"].double()
    y = torch.zeros(c["M"], c["N"], device=x.device, dtype=torch.float64)
    for i, k in enumerate(range(0, c["K"], c["group"])):
        part = x[:, k:k + c["group"]] @ q[:, k:k + c["group"]].t()
        zero = s["zeros"][:, i].double() if c["zeros"] else 8.0
        y += s["scales"][:, i].double() * (part - zero * x[:, k:k + c["group"]].sum(1, keepdim=True))
    for more in ("bias", "residual"):
        if s[more] is not None:
            y += s[more].double()
    return y


def _exact_processed(c, s):
    z = s["logits"].double()
    if c["penalties"]:
        h = s["history"].long() & 0xFFFF
        count = h % 32768
        factor = torch.where(z > 0, 1 / s["repetition"].double()[:, None], s["repetition"].double()[:, None])
        z = z * torch.where(h > 0, factor, 1.0)
        z -= s["frequency"].double()[:, None] * count + s["presence"].double()[:, None] * count.clamp(max=1)
    if s["bias"] is not None:
        z = z + s["bias"].double()
    if c["mask"]:
        shifts = torch.arange(32, device=z.device)
        bits = ((s["mask"].long()[:, :, None] >> shifts) & 1).flatten(1)[:, :c["V"]]
        z = z.masked_fill(bits == 0, float("-inf"))
    return z


def _exact_select(c, s):
    z = _exact_processed(c, s)
    if c["sampled"]:
        z = z / s["temperature"].double()[:, None]
    v = z + s["noise"].double() if c["sampled"] else z
    order = torch.sort(v, dim=1, descending=True, stable=True).indices  # equal values keep their order
    token = order[:, 0]
    logprob = z.log_softmax(1).gather(1, token[:, None])[:, 0]
    empty = (z == float("-inf")).all(1)
    return token.masked_fill(empty, -1), logprob.masked_fill(empty, float("-inf"))


def _exact_history(c, s):
    rows = []
    for b in range(c["B"]):
        seen = torch.bincount(s["prompt"][b, :int(s["prompt_lengths"][b])], minlength=c["V"])
        count = torch.bincount(s["output"][b, :int(s["output_lengths"][b])], minlength=c["V"])
        rows.append(count.clamp(max=32767) - 32768 * (seen > 0).long())
    return torch.stack(rows).to(torch.int16)


def exact(case, seed):
    s = _INPUTS[case["op"]](case, seed)
    if case["op"] == "process":
        return _exact_processed(case, s)
    return {"linear": _exact_linear, "select": _exact_select, "history": _exact_history}[case["op"]](case, s)
