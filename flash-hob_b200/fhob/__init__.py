"""B200-native double-backward flash attention behind the reference's entry
point (``from fhog import flash_bwdbwd`` becomes ``from fhob import flash_bwdbwd``),
and the twice-differentiable operators that a layer has around it."""
from .autograd import attention, attention_backward
from .layer import RotaryPositions, layer_norm, layer_norm_backward, layer_norm_bwdbwd, layer_norm_forward, rotary
from .ops import attention_forward, flash_bwdbwd, produce_L, release_cached_memory, run_passes
from . import torch_op  # registers torch.ops.fhob.bwdbwd

__all__ = ["flash_bwdbwd", "produce_L", "attention_forward", "attention_backward", "attention", "run_passes",
           "release_cached_memory", "rotary", "RotaryPositions", "layer_norm", "layer_norm_forward", "layer_norm_backward",
           "layer_norm_bwdbwd"]
