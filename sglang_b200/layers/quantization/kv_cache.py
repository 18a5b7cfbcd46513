"""A paged key/value cache in e4m3 with one fp32 scale for each token and head: written and read back.

  k_cache, v_cache   [num_pages, page_size, num_kv_heads, head_dim] float8_e4m3fn
  k_scale, v_scale   [num_pages, page_size, num_kv_heads] float32

Any page, token and head strides (multiples of 16 elements in the codes), so a pool with another order of dimensions is passed
as a permuted view.  Slot s is place s % page_size of page s // page_size.  The codes and scales of a token are those that
sglang_per_token_group_quant_fp8 with group_size = head_dim gives, special values included: a NaN does not count for the scale and
gets the code of -448, so that it reads back as minus the head's largest finite magnitude (a head of NaN alone as -1e-10); an
infinity makes the scale infinite and reads back as minus infinity, the rest of its head as NaN.  No gradient passes through;
what is written counts as modified for autograd.

The reference keeps FP8 keys and values with one scale for the whole layer (python/sglang/srt/layers/quantization/kv_cache.py,
MHATokenToKVPool.set_kv_buffer in python/sglang/srt/mem_cache/memory_pool.py); a scale for each token and head needs no
calibration.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ... import _lib


def store_kv_fp8(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                 v_scale: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantises k and v [T, num_kv_heads, head_dim] (bf16 / fp16) into the cache slots slots [T] (int32 / int64).  A slot
    outside the cache (-1 for padding) is skipped; the slots of one call have to be distinct (not checked).  The caches and scales
    share no memory with one another or with what is read, except that v_cache and v_scale may be k_cache and k_scale where v
    is k."""
    _lib.host().head_rows("store_kv_fp8", None, k, v, None, None, None, None, 0.0, True, None, None, False, k_cache, v_cache,
                          k_scale, v_scale, slots)


def qk_norm_rope_store_kv_fp8(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: Optional[torch.Tensor],
                              cos_sin_cache: Optional[torch.Tensor], k_cache: torch.Tensor, v_cache: torch.Tensor,
                              k_scale: torch.Tensor, v_scale: torch.Tensor, slots: torch.Tensor,
                              q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                              norm_eps: float = 1e-6, is_neox: bool = True, q_out: Optional[torch.Tensor] = None,
                              k_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """qk_norm_rope (layers/rotary_embedding.py) and store_kv_fp8 of the rotated keys and of v, one pass over the qkv output.
    Returns q_out (new and contiguous unless given; may be q itself).  The keys are quantised from fp32, without a rounding to
    16 bits in between; k_out, if given, receives them in k's type as well.  A token with a negative position is padding:
    nothing of it is written, whatever its slot.  What is written shares no memory with anything else, q_out being q and k_out
    being k apart."""
    return _lib.host().head_rows("qk_norm_rope_store_kv_fp8", q, k, v, positions, cos_sin_cache, q_weight, k_weight, norm_eps,
                                 is_neox, q_out, k_out, False, k_cache, v_cache, k_scale, v_scale, slots)[0]


def load_kv_fp8(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                page_table: torch.Tensor, kv_indptr: torch.Tensor, num_tokens: int, kv_start: Optional[torch.Tensor] = None,
                out_dtype: torch.dtype = torch.bfloat16, k_out: Optional[torch.Tensor] = None,
                v_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The cached keys and values of a batch, packed: two [num_tokens, num_kv_heads, head_dim] tensors of out_dtype (new unless
    given).  Rows kv_indptr[b] ... kv_indptr[b + 1] - 1 (int32 [batch + 1], on the device) are tokens kv_start[b] ... (int32
    [batch]; None: from 0) of sequence b, whose pages are page_table[b] (int32 [batch, max_pages]).  num_tokens is what the
    host knows kv_indptr[batch] to be, or more: rows behind the last sequence are left as they were.  A token whose page is
    missing from the table or the cache reads as NaN.  k_out and v_out share no memory with one another or with what is read."""
    return _lib.host().load_kv(k_cache, v_cache, k_scale, v_scale, page_table, kv_indptr, kv_start, num_tokens, out_dtype,
                               k_out, v_out)
