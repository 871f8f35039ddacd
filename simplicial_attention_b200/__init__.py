"""B200-native sliding-window causal 2-simplicial attention (forward + backward).

Drop-in for the sliding path of lucidrains/simplicial-attention:
``SlidingWindowTwoSimplicialMHA``, ``sliding_two_simplicial_attn`` and
``SlidingTwoSimplicialAttention`` keep the reference's signatures and run on
hand-written sm_100a CUDA kernels behind the C ABI of ``include/sa2.h``.  So do the parts
of a language model around its attention layers: ``token_embedding``, ``qk_norm_rotary``,
``distillation_loss`` and ``sample_tokens``.
"""
from .attention import (
    BackwardCall,
    SlidingTwoSimplicialAttention,
    check_device,
    device_status,
    sa2_backward,
    sa2_forward,
    sliding_two_simplicial_attn,
    sliding_two_simplicial_attn_with_lse,
)
from .distill import distillation_loss, distillation_loss_and_grad
from .embedding import token_embedding
from .host import HostPipeline
from .mha import HigherOrderAttention, SlidingWindowTwoSimplicialMHA
from .rotary import qk_norm_rotary, rotary_frequencies
from .sampling import sample_tokens

__all__ = [
    "SlidingTwoSimplicialAttention",
    "sliding_two_simplicial_attn",
    "sliding_two_simplicial_attn_with_lse",
    "sa2_forward",
    "sa2_backward",
    "device_status",
    "check_device",
    "BackwardCall",
    "HostPipeline",
    "HigherOrderAttention",
    "SlidingWindowTwoSimplicialMHA",
    "token_embedding",
    "rotary_frequencies",
    "qk_norm_rotary",
    "distillation_loss",
    "distillation_loss_and_grad",
    "sample_tokens",
]
