"""RMSNorm of the query and key heads and the rotary position embedding, in one pass.

The reference runs them one after the other: RMSNorm on q.view(-1, head_dim) and k.view(-1, head_dim)
(python/sglang/srt/layers/layernorm.py), then RotaryEmbedding.forward on the result
(python/sglang/srt/layers/rotary_embedding.py).  qk_norm_rope_store_kv_fp8 in layers/quantization/kv_cache.py writes the
keys and values into a quantised cache in the same pass.  No gradient passes through; what is written in place counts as
modified for autograd.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _lib


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: Optional[torch.Tensor], cos_sin_cache: Optional[torch.Tensor],
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, norm_eps: float = 1e-6,
                 is_neox: bool = True, q_out: Optional[torch.Tensor] = None,
                 k_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """q [T, num_q_heads, head_dim] and k [T, num_kv_heads, head_dim] (bf16 / fp16, e.g. views of a packed qkv output) ->
    (q_out, k_out), new contiguous tensors unless given; q_out may be q itself and k_out k itself; other overlaps are refused.

    Every head is normalised with its weight [head_dim] (None: not), then its first cos_sin_cache.shape[1] elements are rotated
    by row positions[t] of cos_sin_cache [max_position, rotary_dim] (fp32, cosines | sines; None: no rotation): pairs
    (i, i + rotary_dim / 2), or (2 i, 2 i + 1) with is_neox=False.  All in fp32, rounded once.  A token with a negative position
    is padding (also without a table): its rows of q_out and k_out stay as they are.  A position that the table lacks gives NaN.
    head_dim and rotary_dim are multiples of 16, head_dim at most 256; token and head strides multiples of 8 elements."""
    return _lib.host().head_rows("qk_norm_rope", q, k, None, positions, cos_sin_cache, q_weight, k_weight, norm_eps, is_neox,
                                 q_out, k_out, True, None, None, None, None, None)
