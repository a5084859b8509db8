"""B200-native (sm_100a) small-q paged-KV attention for MTP / speculative decoding.

Public API:
  small_q_attention(query, key_cache, value_cache, block_tables, seq_lens, page_size, max_seq_len=0)
  small_q_attention_partial(...) -> (O, LSE)   shard form for a split sequence
  merge_partials(parts_o, parts_lse)           log-sum-exp merge of shards
  cache_append(new_k, new_v, k_cache, v_cache, block_tables, seq_lens)
                                               write the draft tokens' K/V into their pages
  small_q_attention_scaled(query, k_cache, v_cache, k_scales, v_scales, ...)
  cache_append_scaled(new_k, new_v, k_cache, v_cache, k_scales, v_scales, ...)
                                               an FP8 cache with one scale per page and KV head
  accumulate_attention_weights(query, k_cache, block_tables, seq_lens, lse, scores, 16)
  cache_evict(k_cache, v_cache, scores, block_tables, seq_lens, budget)
                                               eviction by accumulated attention weight
  PagedMTPAttention(device).plan(...).run(...)  planned, CUDA-graph-capturable step
  cuda.forward_v0 ... forward_v5               upstream-compatible entry points

All compute runs in the in-tree C-ABI library ``_lib/libsqa_b200.so``; there is
no CPU fallback.
"""

from .cache import cache_append  # noqa: F401
from .eviction import accumulate_attention_weights, cache_evict  # noqa: F401
from .scaled import cache_append_scaled, small_q_attention_scaled  # noqa: F401
from .wrapper import PagedMTPAttention  # noqa: F401
from .attention import (  # noqa: F401
    merge_partials,
    read_device_status,
    selected_kernel,
    small_q_attention,
    small_q_attention_partial,
    workspace_bytes,
)

__all__ = [
    "small_q_attention",
    "small_q_attention_partial",
    "merge_partials",
    "workspace_bytes",
    "read_device_status",
    "selected_kernel",
    "cache_append",
    "small_q_attention_scaled",
    "cache_append_scaled",
    "accumulate_attention_weights",
    "cache_evict",
    "PagedMTPAttention",
]
