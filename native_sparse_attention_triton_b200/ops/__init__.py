"""The operator namespace: the nine names of the reference's ``native_sparse_attention.ops``, the steps its layer leaves to other
code (sliding-window attention, the gated sum of the branches, rotary embedding), sliding-window attention with sinks, and the paged
key-value cache."""
from .compress import avgpool_compress, linear_compress, weightedpool_compress
from .compressed_attention import compressed_attention
from .decode import compressed_attention_decode, flash_attention_decode, topk_sparse_attention_decode
from .flash_attention import flash_attention_varlen
from .gate_combine import gate_combine
from .paged import paged_attention_decode, paged_kv_append, paged_kv_evict
from .rope import rope
from .sink_window import sink_window_attention
from .sliding_window import sliding_window_attention
from .topk_sparse_attention import topk_sparse_attention
from .utils import get_compressed_seqlens

__all__ = [
    "avgpool_compress",
    "weightedpool_compress",
    "linear_compress",
    "flash_attention_varlen",
    "sliding_window_attention",
    "sink_window_attention",
    "gate_combine",
    "rope",
    "compressed_attention",
    "topk_sparse_attention",
    "flash_attention_decode",
    "compressed_attention_decode",
    "topk_sparse_attention_decode",
    "paged_kv_append",
    "paged_attention_decode",
    "paged_kv_evict",
    "get_compressed_seqlens",
]
