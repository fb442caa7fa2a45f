"""hdcmamba_amd: the HdcMamba block forward on MI355X (gfx950) HIP kernels.

Public names match the reference package (hdcmamba/__init__.py:1-13).
"""
from .model import (
    BlockState,
    FusedNormConv1dFunction,
    HdcMamba9v3Block,
    HdcMamba9v3Model,
    fused_norm_conv1d_trainable,
    quantize_4bit,
    set_differentiable_mixer,
    set_fused_out_proj,
    set_fused_step_front,
)
from .lm import DecodeGraph, ForwardGraph, HdcMambaLM
from .quant4 import Linear4Bit, Weight4Bit, linear_4bit
from .sampling import append_tokens, fill_token_history, new_token_history, process_logits, select_tokens

__all__ = [
    "HdcMamba9v3Block",
    "HdcMamba9v3Model",
    "FusedNormConv1dFunction",
    "fused_norm_conv1d_trainable",
    "HdcMambaLM",
    "BlockState",
    "DecodeGraph",
    "ForwardGraph",
    "set_differentiable_mixer",
    "set_fused_out_proj",
    "set_fused_step_front",
    "Weight4Bit",
    "Linear4Bit",
    "quantize_4bit",
    "linear_4bit",
    "process_logits",
    "select_tokens",
    "new_token_history",
    "fill_token_history",
    "append_tokens",
]
