"""Causal varlen attention with a sliding window and sinks: the first keys of a sequence stay visible to all its queries.

The reference has no operator for it; it stands next to sliding_window_attention, whose call it takes without max_seqlen.  Its
single-token form is paged_attention_decode with window_size and num_sinks.
"""
from typing import Optional

import torch

from .. import _lib


def sink_window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, window_size: int, num_sinks: int,
                          sm_scale: Optional[float] = None) -> torch.Tensor:
    """q [total, Hq, d], k/v [total, Hkv, d] (self-attention: one cu_seqlens, int32 [batch + 1]); key j of a sequence is visible to its
    query i iff j <= i and (i - j <= window_size or j < num_sinks).  cu_seqlens ascends from 0; a sequence that ends behind the rows ends with them,
    and one that starts outside of them is none (either sets device status 2).

    bfloat16 or float16, head_dim 64 or 128, Hq / Hkv a power of two of at most 16 (NotImplementedError otherwise).  Differentiable in q, k
    and v.  Rows behind the last sequence (a padded batch) may hold anything: they reach no other row, and their output and gradients are
    zero.  A value that is not finite reaches the rows that see it and no others.

    Where an input requires gradients the forward keeps its probabilities in two 16-bit parts, and a second tensor of the output's size until
    the backward pass (what the output's rounding took away); without gradients it keeps one part: 2.2e-3 of 64 bits instead of 1.66e-3 in
    bfloat16, an eighth of that in float16, and in fewer microseconds.  So the two calls differ in their last bits.  dK and dV of the sinks, and of
    all keys where the batch is short or its heads few, are sums over several thread blocks whose last bits depend on their order.
    """
    return _lib.host().sink_window_attention(q, k, v, cu_seqlens, int(window_size), int(num_sinks), sm_scale)
