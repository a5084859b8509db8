"""A block-scaled 8-bit cache: the append that fills it and the attention that reads it.

The caches are FP8-E4M3 pages with one fp32 scale per page (16 tokens) and KV head,
K and V apart: a cached element stands for ``scale * e4m3``.  ``key_scales`` and
``value_scales`` are ``[num_pages, Hkv]``; a row may be further apart than ``Hkv``
(a view of a bigger array).  Next to ``small_q_attention`` over FP8 caches, which takes
one scale for a whole cache, a scale per page follows the values' magnitude from token
block to token block and head to head.  Neither operator has an upstream counterpart.
"""

from __future__ import annotations

from . import _native
from .attention import _cuda_available, _layout_code


def cache_append_scaled(new_keys, new_values, key_cache, value_cache, key_scales, value_scales, block_tables,
                        seq_lens, *, check: bool = False, kv_layout: str = "NHD"):
    """Quantise ``new_keys`` / ``new_values`` ``[batch, q_len, Hkv, 128]`` (FP16 or BF16)
    into the paged FP8-E4M3 caches and their scales, in place; returns
    ``(key_cache, value_cache, key_scales, value_scales)``.

    The tokens and slots are those of ``cache_append``: token ``qi`` of sequence ``b`` is
    position ``seq_lens[b] - q_len + qi`` (``seq_lens`` is the length after the append); any
    ``q_len >= 1``, so prompts too.  Per touched page and head, K and V apart: ``need`` is the
    smallest power of two (``2**-100`` at least) that brings the page's finite new values
    within ``448 * need``; a page whose first slot is new gets ``need`` as its scale, any other
    the larger of ``need`` and its old scale, and where the scale grew its older tokens are
    stored again at the new one.  Powers of two move only the older values' exponents, so
    a growing scale rounds them again only below E4M3's smallest normal value.  Values are
    rounded to nearest even and saturate at ``448 * scale``; NaN stays NaN.  Slots behind
    the last new token keep their bytes.

    Errors of the contract raise ``ValueError`` before launch.  With ``check=True`` the call
    synchronises and raises ``ValueError`` for ``seq_lens < q_len`` or lengths beyond the page
    table (those sequences are skipped) and ``IndexError`` for a page id outside the cache
    (those pages are skipped).  A page may be named once per call.
    """
    if not _cuda_available():
        raise RuntimeError("CUDA is required for the cache-append kernel")
    try:
        _native.torch_ext().append_scaled(new_keys, new_values, key_cache, value_cache, key_scales, value_scales,
                                          block_tables, seq_lens, check, _layout_code(kv_layout))
    except TypeError as e:  # a non-tensor where a tensor belongs (pybind11's argument check)
        raise ValueError(f"all inputs must be CUDA tensors ({e})") from None
    return key_cache, value_cache, key_scales, value_scales


def small_q_attention_scaled(query, key_cache, value_cache, key_scales, value_scales, block_tables, seq_lens,
                             page_size: int, max_seq_len: int = 0, *, out=None, out_lse=None, return_lse: bool = False,
                             mask_lens=None, workspace=None, num_ctas: int = 0, check: bool = False,
                             kv_layout: str = "NHD", sm_scale: float | None = None, out_scale: float = 1.0,
                             min_seq_len: int = 0, cluster: int = 0):
    """``small_q_attention`` over a block-scaled FP8-E4M3 cache.

    ``query`` is FP16 or BF16; K is ``key_scales * key_cache`` and V ``value_scales *
    value_cache`` per page and head.  Value scales must lie in ``[0, 2**30]`` (those below ``2**-60``,
    an all-zero page's among them, count as ``2**-60``); key scales must be finite.  Returns the rows in
    the query's type (or into ``out``, which may also be fp32: the rows before their rounding, for
    :func:`merge_partials`), and with ``return_lse`` also the
    fp32 natural-log log-sum-exp ``[batch, q_len, Hq]`` (-inf for a row that sees no token), which
    :func:`accumulate_attention_weights` takes.  Probabilities keep 13 bits, and tokens down to ``2**-29`` of a
    row's largest ``p * value scale`` count.  The other arguments are those of
    ``small_q_attention`` and ``small_q_attention_partial``; ``cluster`` is 0 or 1 (1: near-uniform
    bounds do not make every segment split evenly).

    Without ``workspace``, eager calls share one per (device, stream) and calls under CUDA-graph
    capture take one from the graph's own memory pool.
    """
    if not _cuda_available():
        raise RuntimeError("CUDA is required for the small-q attention kernel")
    try:
        o, lse = _native.torch_ext().forward_scaled(
            query, key_cache, value_cache, key_scales, value_scales, block_tables, seq_lens, page_size, mask_lens,
            max_seq_len, out, out_lse, return_lse, workspace, num_ctas, check, _layout_code(kv_layout),
            0.0 if sm_scale is None else sm_scale, out_scale, min_seq_len, cluster)
    except TypeError as e:
        raise ValueError(f"all inputs must be CUDA tensors ({e})") from None
    return (o, lse) if return_lse else o
