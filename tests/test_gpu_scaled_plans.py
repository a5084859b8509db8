"""Which split the block-scaled attention takes by itself must not change its results: numbers of segments on both sides of
one and two waves of CTAs, at lengths on both sides of the limits, against calls with a forced split.
"""

import pytest
import torch

from tests.test_gpu_scaled import F8, assert_within, attend, reference, scaled_case, to_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sqa():
    if not torch.cuda.is_available() or F8 is None:
        pytest.skip("needs a CUDA device and torch.float8_e4m3fn")
    import small_q_attention_b200 as m

    return m


@pytest.mark.parametrize("longest", [640, 656, 1024, 1040])
@pytest.mark.parametrize("q_len,dtype", [(1, torch.bfloat16), (2, torch.float16), (4, torch.float16), (6, torch.bfloat16), (12, torch.float16)])
@pytest.mark.parametrize("batch", [74, 75, 148, 149])
def test_automatic_splits(sqa, batch, q_len, dtype, longest):
    """batch x 2 heads: 148, 150, 296 and 298 segments on a GPU of 148 SMs."""
    g = torch.Generator().manual_seed(batch)
    lens = torch.randint(q_len, longest + 1, (batch,), generator=g).tolist()
    lens[0], lens[-1], lens[batch // 2] = longest, q_len, 0
    c = scaled_case(q_len, lens, hkv=2, dtype=dtype, seed=q_len)
    gpu = to_gpu(c)
    out, lse = attend(sqa, gpu, max_seq_len=longest)
    split, split_lse = attend(sqa, gpu, max_seq_len=longest, num_ctas=100)
    some = [0, 1, batch // 2, batch // 2 + 1, batch - 1]  # the oracle's share
    part = dict(c, query=c["query"][some], table=c["table"][some], seq_lens=c["seq_lens"][some], lens=[lens[i] for i in some])
    assert_within(out[some], lse[some], reference(part), dtype)
    assert_within(split[some], split_lse[some], reference(part), dtype)
    # one rounding of the output to each side, and P's 2^-13 relative to what it weighs (|v| up to about 5 here)
    eps = torch.finfo(dtype).eps
    assert ((out.float() - split.float()).abs() <= eps * out.float().abs() + 2.0 ** -11 * 5).all()
    assert torch.equal(torch.isneginf(lse), torch.isneginf(split_lse))
