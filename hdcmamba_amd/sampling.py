"""From logits to the next tokens on the GPU (csrc/logits.hip): penalties for repeated tokens, biases
and grammar masks on a batch of logits, the choice of the next token, and the token history that the
penalties read.  The reference's generate (train.py:139-151) samples from the plain softmax in torch.

Controls, shared by process_logits and select_tokens.  For logit l of token v of a sequence, in fp32
and in this order:

  repetition  l / repetition if l > 0, else l * repetition, for tokens of the prompt or the output
  frequency   l - frequency * count if count > 0, count = how often the output holds the token
  presence    l - presence if count > 0
  bias        l + bias[v]
  mask        -inf unless bit v % 32 of mask word v // 32 is set

An infinite ``frequency`` or ``presence`` bans the output's tokens.

``repetition`` (> 0), ``frequency`` and ``presence`` are numbers or tensors of one value per
sequence and need ``history``, an int16 table [B, V] (new_token_history): the sign bit marks the
prompt's tokens, the low 15 bits count the token in the output (at most 32767).  ``bias`` is [V] or
[B, V] (float32 or bfloat16), ``mask`` int32 [ceil(V / 32)] or [B, ceil(V / 32)].  No gradient: a
tensor among all these that needs one, or carries a tangent, is refused.
"""
from __future__ import annotations

import torch

from . import _ops

__all__ = ["process_logits", "select_tokens", "new_token_history", "fill_token_history", "append_tokens"]


def process_logits(logits, history=None, repetition=None, frequency=None, presence=None, bias=None, mask=None, out=None):
    """logits [B, V] (float32 or bfloat16) under the controls, rounded once to their type; ``out`` may be
    ``logits``."""
    return _ops.native().process_logits(logits, (history, repetition, frequency, presence, bias, mask), out)


def select_tokens(logits, history=None, repetition=None, frequency=None, presence=None, bias=None, mask=None,
                  temperature=None, noise=None):
    """The next token of every sequence from logits [B, V] under the controls, which are not written:
    (tokens int64 [B], log-probabilities float32 [B]).

    With t = processed / temperature, the token is the lowest index of the largest t + noise and its
    log-probability that of softmax(t); with ``noise`` [B, V] float32 drawn from the standard Gumbel
    distribution (-log(-log(u)), u uniform in (0, 1)) it is a sample of softmax(t).  ``temperature`` is a
    number or one per sequence (1 by default); one that is not above 0 makes a greedy choice, without
    noise, from t = processed.  -inf and NaN are never chosen: a sequence with nothing else gets token -1
    and -inf.  A NaN or +inf among the allowed logits makes the log-probability NaN."""
    return _ops.native().select_tokens(logits, (history, repetition, frequency, presence, bias, mask), temperature, noise)


def new_token_history(batch, vocab, device="cuda"):
    """An empty history table [batch, vocab] int16 (rows padded to 16 bytes)."""
    return torch.zeros(batch, -(-vocab // 8) * 8, dtype=torch.int16, device=device)[:, :vocab]


def fill_token_history(table, prompt=None, prompt_lengths=None, output=None, output_lengths=None):
    """Write all of ``table`` [B, V] from the token ids of prompts [B, P] and outputs [B, O]; ``*_lengths``
    [B]: how many of a row's ids count (right-padded batches).  Ids outside 0..V-1 are passed over.
    Returns the table."""
    return _ops.native().fill_token_history(table, prompt, prompt_lengths, output, output_lengths)


def append_tokens(table, tokens, lengths=None):
    """Count output tokens [B] or [B, T] (``lengths`` [B]: how many of a row) in ``table``, in place; ids
    outside 0..V-1 (a token -1 of select_tokens) are passed over.  Returns the table."""
    return _ops.native().append_tokens(table, tokens, lengths)
