"""Low-rank adapters of many requests beside a shared projection.

  out[t] = base_output[t] + scalings[a] * (x[t] A[a]^T) B[a]^T,   a = the adapter of token t (or none)

base_output is what the projection gave, e.g. Fp8LinearMethod.apply.  A projection that is several in one (qkv, gate_up) has
one low-rank product per slice: lora_a holds the slices' A one below the other, and output_sizes says which columns of the
output belong to which.  Adapters live in buffers of a common largest rank R, lora_a [num_adapters, num_slices * R, K] and
lora_b [num_adapters, N, R], slice s of A in rows s * R ... ; what lies behind an adapter's own rank is not used.
No gradient passes through any of this; what is written in place counts as modified for autograd.

The reference's counterparts: LoRABatchInfo, sgemm_lora_a_fwd, sgemm_lora_b_fwd, qkv_lora_b_fwd and gate_up_lora_b_fwd
(python/sglang/srt/lora/triton_ops, lora/layers.py).
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from .. import _lib


class LoRABatch:
    """Which adapter each token of a batch uses, grouped for the kernels.  Made once per batch of tokens, for every projection
    of every layer; nothing is read on the host.

    token_adapters  int32 [num_tokens]: index into the adapter buffers; anything outside them (-1) means none
    lora_ranks      int32 [num_adapters]: each adapter's rank; 0 means that the buffer is empty
    scalings        fp32 [num_adapters]

    The kernels are chosen by the numbers of tokens and of adapter buffers, in use or not: 8191 tokens of one adapter (K = 8192,
    N = 10240, rank 64) take 111 us with 8 buffers and 321 with 512, where they count as a small batch."""

    def __init__(self, token_adapters: torch.Tensor, lora_ranks: torch.Tensor, scalings: torch.Tensor) -> None:
        self.token_adapters, self.lora_ranks, self.scalings = token_adapters, lora_ranks, scalings
        self.plan = _lib.host().lora_plan(token_adapters, lora_ranks, None)
        self.num_adapters = lora_ranks.shape[0]

    @classmethod
    def from_segments(cls, weight_indices: torch.Tensor, seg_lens: torch.Tensor, num_tokens: int, lora_ranks: torch.Tensor,
                      scalings: torch.Tensor) -> "LoRABatch":
        """Request i, with adapter weight_indices[i], holds the next seg_lens[i] tokens of num_tokens; tokens behind the last
        request (a padded batch) have no adapter."""
        # a search instead of repeat_interleave, which needs num_tokens to be the exact sum and asserts it on the device (40 us
        # back to back against 22, device time 12 against 9, for 32 requests of 4096 tokens; once for a batch)
        request = torch.searchsorted(seg_lens.cumsum(0), torch.arange(num_tokens, device=seg_lens.device), right=True)
        ids = torch.nn.functional.pad(weight_indices.to(torch.int32), (0, 1), value=-1)[request]
        return cls(ids, lora_ranks, scalings)

    def update(self) -> None:
        """Groups again after token_adapters or lora_ranks have been written in place (the next replay of a captured graph, of
        which this call may be a part).  Their lengths stay."""
        if self.lora_ranks.shape[0] != self.num_adapters:
            raise RuntimeError(f"the batch was made for {self.num_adapters} adapters, not {self.lora_ranks.shape[0]}")
        _lib.host().lora_plan(self.token_adapters, self.lora_ranks, self.plan)


def lora_shrink(x: torch.Tensor, lora_a: torch.Tensor, batch: LoRABatch, num_slices: int = 1) -> torch.Tensor:
    """h [num_tokens, num_slices * R] = x A^T, each token with its adapter's A; fp32 sums, rounded once to x's type.  Zero behind
    an adapter's rank and for tokens without one; not scaled."""
    return _lib.host().lora(None, x, None, lora_a, None, batch.plan, batch.num_adapters, batch.scalings, None, num_slices, None)


def lora_expand(h: torch.Tensor, lora_b: torch.Tensor, batch: LoRABatch, base_output: Optional[torch.Tensor] = None,
                output_sizes: Optional[Sequence[int]] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """base_output + scalings * h B^T, slice by slice; see apply_lora for base_output, output_sizes and out."""
    if out is None:
        out = base_output
    sizes = None if output_sizes is None else tuple(output_sizes)
    return _lib.host().lora(base_output, None, h, None, lora_b, batch.plan, batch.num_adapters, batch.scalings, sizes, 1, out)


def apply_lora(base_output: Optional[torch.Tensor], x: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
               batch: LoRABatch, output_sizes: Optional[Sequence[int]] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Adds the adapters' part for x [num_tokens, K] to base_output [num_tokens, N], in place unless `out` is given; None counts
    as zeros and gives a new tensor.  The result shares memory with neither x nor, unless it is base_output itself, base_output.
    output_sizes: the columns of each slice (None: one slice).  bf16 or fp16 throughout; K, R and the slices' sizes are multiples
    of 8, R <= 256, at most 8 slices.  The sums are fp32; x A^T, unscaled, is rounded to x's type in between (in fp16 it must
    stay below 65504), the result once.  The order of the sums, which is the same in every run, depends on the sizes, the number
    of tokens among them."""
    if out is None:
        out = base_output
    sizes = None if output_sizes is None else tuple(output_sizes)
    return _lib.host().lora(base_output, x, None, lora_a, lora_b, batch.plan, batch.num_adapters, batch.scalings, sizes, 1, out)
