"""CPU oracle for the small-q paged attention path (test infrastructure only).

Imported only by ``tests/``, ``__graft_entry__.smoke()`` and the CPU-baseline
legs of ``bench.py``; the product package never imports it.
"""

from .cache_append import cache_append_reference  # noqa: F401
from .paged_mtp_attention import (  # noqa: F401
    merge_partials,
    paged_mtp_attention_partial,
    paged_mtp_attention_reference,
)
from .scaled_cache import (  # noqa: F401
    append_scaled_reference,
    attention_scaled_reference,
    evict_reference,
    page_scale,
    round_e4m3,
    weights_reference,
)
