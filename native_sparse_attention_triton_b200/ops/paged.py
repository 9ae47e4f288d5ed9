"""A paged key-value cache: rows appended, attended to by one token per sequence, and cut down to the ones attention has used most.

k_pages and v_pages are [num_pages, page_size, num_kv_heads, head_dim], bfloat16 or float16, head_dim 64 or 128, any page_size and any strides of
multiples of 8 elements with contiguous head_dim (slices of a larger cache, pages with their heads outermost).  Row j of sequence b is slot
j % page_size of page block_table[b, j // page_size]; block_table is int32 [batch, max_pages], its entries behind a sequence's rows are not
read, and sequences may share pages that are only read.  seqlens is int32 [batch].  Everything is read on the device: no call waits for the
GPU, and all of them can be captured in a CUDA graph.  A page number outside the cache or a length beyond block_table sets device status 2
(native_sparse_attention_triton_b200.device_status()); such rows are neither read nor written.

The reference has no paged cache; these operators stand next to its single-token operators on contiguous caches (ops/decode.py).
"""
from typing import Optional, Tuple

import torch

from .. import _lib


def paged_kv_append(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, seqlens: torch.Tensor, k: torch.Tensor,
                    v: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Writes k, v [rows, num_kv_heads, head_dim] behind the seqlens[b] rows that each sequence holds: rows cu_seqlens[b] to
    cu_seqlens[b + 1] (a prompt), or one row per sequence without cu_seqlens (a decode step).

    The pages are written in place and must be in block_table already, those that are written by one sequence alone; k and v may be rows of the
    cache itself, as they are before the call.  Returns the lengths
    after that, a new int32 [batch]; rows beyond max_pages * page_size are dropped (device status 2).
    """
    return _lib.host().paged_kv_append(k_pages, v_pages, block_table, seqlens, k, v, cu_seqlens)


def paged_attention_decode(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, seqlens: torch.Tensor,
                           sm_scale: Optional[float] = None, window_size: Optional[int] = None, num_sinks: int = 0,
                           weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One query token per sequence, at the position of the last of its seqlens[b] rows, attends to the cache.

    q [batch, num_q_heads, head_dim], at most 16 query heads per key/value head; row j is visible iff window_size is None, or
    seqlens[b] - 1 - j <= window_size, or j < num_sinks: what the query sees in sink_window_attention.  A sequence without rows gets zeros.
    weights float32 [batch, num_kv_heads, max_pages * page_size or more]: the probabilities that each visible row receives, summed over
    the query heads of its key/value head, are added in place (paged_kv_evict goes by them); other entries are left as they are.
    They take scratch of 4 bytes for each query head and row of the table (with a window: for the rows that it and the sinks reach into), of which
    up to 64 MiB a stream are kept for the next call.
    Values that are not finite reach what the definition makes depend on them: a head whose logits hold NaN has no output, and adds NaN to the
    weights of the rows it sees.  Not differentiable.
    """
    return _lib.host().paged_attention_decode(q, k_pages, v_pages, block_table, seqlens, sm_scale,
                                              None if window_size is None else int(window_size), int(num_sinks), weights)


def paged_kv_evict(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, seqlens: torch.Tensor, weights: torch.Tensor,
                   new_block_table: torch.Tensor, budget: int, num_sinks: int, num_recent: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Keeps at most `budget` rows of every sequence, for each key/value head its own: the first num_sinks, the last num_recent, and the
    rest of the budget by the largest weights of the rows between (equal ones: the lower row; NaN counts as the smallest).

    The kept rows are written, in their order, to the pages of new_block_table (int32 [batch, max_new_pages], with room for min(budget,
    capacity) rows; pages that hold no row of these sequences).  The old pages keep what they hold and are the caller's to free.  Call it for the
    sequences that are over the budget: one that is not is copied whole.

    Returns (seqlens int32 [batch], weights like the ones given, with zeros behind the kept rows, kept int32 [batch, num_kv_heads, budget]:
    the old row of each kept one, -1 behind them).
    """
    return _lib.host().paged_kv_evict(k_pages, v_pages, block_table, seqlens, weights, new_block_table, int(budget), int(num_sinks),
                                      int(num_recent))
