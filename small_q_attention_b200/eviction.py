"""Eviction from the paged cache by accumulated attention weight.

Every cached token has a score per KV head, ``scores`` fp32 ``[num_pages, Hkv, 16]`` in
the order of the cache's pages, 16-byte aligned for ``cache_evict``.  ``accumulate_attention_weights`` adds a step's attention
weights to them, ``cache_evict`` keeps the tokens of the highest scores within a
budget and compacts them in place.  Both take 16-bit caches and block-scaled FP8-E4M3
caches.  Neither has an upstream counterpart.
"""

from __future__ import annotations

from . import _native
from .attention import _cuda_available, _layout_code


def accumulate_attention_weights(query, key_cache, block_tables, seq_lens, lse, scores, page_size: int,
                                 max_seq_len: int = 0, *, key_scales=None, mask_lens=None, num_ctas: int = 0,
                                 check: bool = False, kv_layout: str = "NHD", sm_scale: float | None = None,
                                 min_seq_len: int = 0):
    """Add the step's attention weights to the cached tokens' scores, in place; returns ``scores``.

    The weight of token ``t`` for KV head ``h`` is the sum over the rows (``q_len`` draft tokens x 4
    query heads) that see it of ``exp(sm_scale * q.k_t - lse[row])``, with ``lse`` ``[batch, q_len, Hq]``
    from the step's attention (``small_q_attention_partial`` or ``small_q_attention_scaled``
    with ``return_lse``; same ``query``, cache and ``sm_scale``).  The last ``q_len``
    tokens of a sequence are new in this step: their scores are set to their weight, whatever
    their slots held; the earlier ones are added to.  Slots behind the tokens held are left.
    A shard of a longer sequence passes its ``mask_lens`` as it does to the attention (the whole
    length less the shard's offset), which also tells which of its tokens, if any, are new, and
    the merged log-sum-exp of all shards (``merge_partials`` with ``return_lse``), not its own.
    ``key_scales`` belong to an FP8-E4M3 cache.  Pages must not be shared between sequences.
    ``check=True`` synchronises and raises as ``small_q_attention`` does.
    """
    if not _cuda_available():
        raise RuntimeError("CUDA is required for the attention-weight kernel")
    try:
        _native.torch_ext().accumulate_weights(query, key_cache, key_scales, block_tables, seq_lens, lse, scores,
                                               page_size, mask_lens, max_seq_len, num_ctas, check,
                                               _layout_code(kv_layout), 0.0 if sm_scale is None else sm_scale,
                                               min_seq_len)
    except TypeError as e:  # a non-tensor where a tensor belongs (pybind11's argument check)
        raise ValueError(f"all inputs must be CUDA tensors ({e})") from None
    return scores


def cache_evict(key_cache, value_cache, scores, block_tables, seq_lens, budget: int, *, recent: int = 0,
                sinks: int = 0, key_scales=None, value_scales=None, new_lens=None, kept=None, check: bool = False,
                kv_layout: str = "NHD"):
    """Cut every sequence longer than ``budget`` to ``budget`` tokens per KV head, in place;
    returns ``(new_lens, kept)``.

    A head keeps the sequence's first ``sinks`` tokens, its last ``recent`` ones and, of the others,
    the ``budget - sinks - recent`` of the highest score (NaN counts as the lowest; equal scores:
    the earlier token).  Kept tokens move, in order, to positions ``0 .. budget - 1`` of the sequence's
    own pages: K, V and scores; the pages behind are free afterwards.  Every page of a
    block-scaled cache that is written gets the smallest power-of-two scale for the values it
    now holds.  Sequences of at most ``budget`` tokens are left as they are.

    ``new_lens`` (int32, shaped like ``seq_lens``, memory of its own) is ``min(seq_lens, budget)``;
    ``kept`` (int32 ``[batch, Hkv, budget]``) holds the position each target came from, -1 behind
    the last.  Pages must not be shared between sequences or listed twice.  With ``check=True``
    the call synchronises and raises ``ValueError`` for a negative length or one beyond the page
    table and ``IndexError`` for a page id outside the cache; those sequences are left, the others
    are cut, and a ``new_lens`` that was passed in holds every sequence's length.
    """
    if not _cuda_available():
        raise RuntimeError("CUDA is required for the cache-eviction kernel")
    try:
        return _native.torch_ext().cache_evict(key_cache, value_cache, scores, block_tables, seq_lens, budget, recent,
                                               sinks, key_scales, value_scales, new_lens, kept, check,
                                               _layout_code(kv_layout))
    except TypeError as e:
        raise ValueError(f"all inputs must be CUDA tensors ({e})") from None
