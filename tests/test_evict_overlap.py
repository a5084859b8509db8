"""The eviction's results must not share memory with what its CTAs still read (C ABI, no GPU: every call ends in a check)."""

import ctypes

import pytest

from tests.test_oracle_scaled import _evict_args, lib  # noqa: F401

APART = dict(seq_lens=65536, block_tables=131072, new_lens=1 << 20, kept=2 << 20)


@pytest.mark.parametrize("kw", [
    dict(new_lens=65536), dict(new_lens=65540), dict(new_lens=65532), dict(new_lens=131072 + 4 * 2 * 32 - 4), dict(new_lens=131068),
    dict(kept=65540), dict(kept=65536 - 4 * 2 * 8 * 100 + 4), dict(kept=131072 + 4 * 2 * 32 - 4), dict(kept=(1 << 20) + 4),
    dict(kept=(1 << 20) - 4 * 2 * 8 * 100 + 4)])
def test_overlaps_are_refused(lib, kw):  # noqa: F811
    assert lib.sqa_cache_evict(ctypes.byref(_evict_args(**{**APART, **kw})), None, None) == 1



@pytest.mark.gpu
def test_neighbours_in_one_allocation_are_not():
    import torch

    from tests.test_gpu_eviction import assert_evicted, evict, evict_case, gpu

    c = evict_case([200, 100], 2, torch.float16, seed=1)
    g = gpu(c)
    base = torch.zeros(2 * 2 * 64 + 4, dtype=torch.int32, device="cuda")
    base[:2] = g["seq_lens"]
    lens, new, kept = base[:2], base[2:4], base[4:].view(2, 2, 64)
    import small_q_attention_b200 as sqa

    evict(sqa, dict(g, seq_lens=lens), 64, recent=3, new_lens=new, kept=kept, check=True)
    assert lens.tolist() == [200, 100]
    assert_evicted(g, c, new, kept, 64, recent=3)
    for bad in (base[1:3], base[:2]):
        with pytest.raises(ValueError):
            evict(sqa, dict(g, seq_lens=lens), 64, recent=3, new_lens=bad)
    with pytest.raises(ValueError):
        evict(sqa, dict(g, seq_lens=base[5:7]), 64, recent=3, new_lens=new, kept=kept)
