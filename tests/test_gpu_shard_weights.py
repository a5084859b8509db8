"""Attention weights of a sequence that is cut into shards: every shard adds to what its tokens had, and only the step's own
tokens are set, wherever the cut lies.  Bounds as in test_gpu_eviction.
"""

import pytest
import torch

from tests.test_gpu_eviction import assert_weights, gpu, weight_case
from tests.test_gpu_scaled import F8

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sqa():
    if not torch.cuda.is_available() or F8 is None:
        pytest.skip("needs a CUDA device and torch.float8_e4m3fn")
    import small_q_attention_b200 as m

    return m


@pytest.mark.parametrize("scaled", [False, True], ids=["16bit", "e4m3"])
@pytest.mark.parametrize("q_len,n,cuts", [(4, 700, (20,)), (4, 690, (43,)), (1, 700, (20, 40)), (16, 4100, (100, 256)),
                                          (8, 2050, (127, 128)), (3, 16, ())])
def test_shards_do_what_the_whole_does(sqa, q_len, n, cuts, scaled):
    """Cuts before, inside (43 pages of 690 tokens: two of the four new tokens on either side) and at the end of the new
    tokens; pages and scores stay where they are, a shard's table is a part of the whole one."""
    c = weight_case(q_len, [n], 2, torch.float16, scaled, seed=q_len)
    g = gpu(c)
    pages = (n + 15) // 16
    for lo, hi in zip((0, *cuts), (*cuts, pages)):
        held, mask = min(n, 16 * hi) - 16 * lo, n - 16 * lo
        sqa.accumulate_attention_weights(
            g["query"], g["k"], g["table"][:, lo:hi].contiguous(), torch.tensor([held], dtype=torch.int32).cuda(), g["lse"],
            g["scores"], 16, key_scales=g["ks"], mask_lens=torch.tensor([mask], dtype=torch.int32).cuda())
    assert_weights(g["scores"], c)


@pytest.mark.parametrize("scaled", [False, True], ids=["16bit", "e4m3"])
def test_a_shard_may_hold_fewer_tokens_than_the_step(sqa, scaled):
    """check=True reports a length below q_len of a whole sequence, not of a shard."""
    c = weight_case(4, [690], 2, torch.float16, scaled, seed=6)
    g = gpu(c)
    two, mask = (torch.tensor([2], dtype=torch.int32).cuda() for _ in range(2))
    last = g["table"][:, 43:44].contiguous()
    call = lambda **kw: sqa.accumulate_attention_weights(  # noqa: E731
        g["query"], g["k"], last, two, g["lse"], g["scores"], 16, key_scales=g["ks"], check=True, **kw)
    call(mask_lens=mask)
    with pytest.raises(ValueError, match="at least q_len"):
        call()
    if scaled:
        attend = lambda **kw: sqa.small_q_attention_scaled(  # noqa: E731
            g["query"], g["k"], g["v"], g["ks"], g["vs"], last, two, 16, check=True, **kw)
        for hints in (dict(), dict(num_ctas=3)):  # both schedules
            attend(mask_lens=mask, **hints)
            with pytest.raises(ValueError, match="at least q_len"):
                attend(**hints)


def test_shards_with_their_merged_log_sum_exp(sqa):
    """The step as shards run it: fp32 rows and log-sum-exps, their merge, then the weights; they sum to the rows."""
    c = weight_case(4, [1000], 2, torch.float16, True, seed=5)
    g = gpu(c)
    g["scores"].zero_()
    shards = []
    for lo, hi in ((0, 30), (30, 63)):
        lens = torch.tensor([min(1000, 16 * hi) - 16 * lo], dtype=torch.int32).cuda()
        shards.append((g["table"][:, lo:hi].contiguous(), lens, torch.tensor([1000 - 16 * lo], dtype=torch.int32).cuda()))
    parts = [sqa.small_q_attention_scaled(g["query"], g["k"], g["v"], g["ks"], g["vs"], t, n, 16, mask_lens=m, return_lse=True,
                                          out=torch.empty(g["query"].shape, device="cuda")) for t, n, m in shards]
    _, lse = sqa.merge_partials(torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts]), return_lse=True)
    for t, n, m in shards:
        sqa.accumulate_attention_weights(g["query"], g["k"], t, n, lse, g["scores"], 16, key_scales=g["ks"], mask_lens=m)
    total = g["scores"].double().sum(dim=(0, 2))
    assert torch.allclose(total, torch.full_like(total, 16.0), rtol=1e-4)
