"""B200-native Evoformer attention (pair-bias + residue-mask flash attention).

Public surface:
    EvoformerAttention            autograd.Function, drop-in for the reference class
    EvoformerAttentionTrueLayout  same op with genuine head-axis semantics
    GatedEvoformerAttention       the op followed by ``sigmoid(gate) *``, fused into the kernel
    evoformer_attention           DS4Sci-style ``attn(Q, K, V, [mask, pair_bias])``; options for the
                                  ``[B, R, R, H]`` bias layout, the gate and the mask-bias gradient
    layer_norm                    layer norm with its backward, rows read where they lie
    relative_position_bias        a learned pair bias by buckets of residue distance
    pair_bias_projection          the pair representation, normalised and projected to a pair bias in one pass
"""
from .attention import (EvoformerAttention, EvoformerAttentionTrueLayout, GatedEvoformerAttention,
                        check_device_status, evoformer_attention, force_generic)
from .inputs import layer_norm, pair_bias_projection, relative_position_bias

__all__ = ["EvoformerAttention", "EvoformerAttentionTrueLayout", "GatedEvoformerAttention",
           "evoformer_attention", "check_device_status", "force_generic",
           "layer_norm", "relative_position_bias", "pair_bias_projection"]
