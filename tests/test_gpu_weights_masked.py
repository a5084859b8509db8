"""Tokens that a sequence holds and no row sees (mask_lens below seq_lens): whatever their K and scales hold, their weight is zero.
"""

import math

import pytest
import torch

from tests.test_gpu_eviction import accumulate, assert_weights, gpu, weight_case
from tests.test_gpu_scaled import F8

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sqa():
    if not torch.cuda.is_available() or F8 is None:
        pytest.skip("needs a CUDA device and torch.float8_e4m3fn")
    import small_q_attention_b200 as m

    return m


@pytest.mark.parametrize("scaled", [False, True], ids=["16bit", "e4m3"])
@pytest.mark.parametrize("q_len", [1, 2, 3, 5, 7, 9, 13, 16])
def test_nan_in_tokens_that_no_row_sees(sqa, q_len, scaled):
    """Every query length: the kernel's row groups hold 8, 16, 32 or 64 rows, of which the step fills 4 q_len."""
    lens = [100, 700, 33]
    c = weight_case(q_len, lens, 2, torch.float16, scaled, seed=q_len)
    mask = [80, 650, 32]
    for b, (n, m) in enumerate(zip(lens, mask)):
        for t in range(m, n):  # all rows see t < m at most
            page, slot = int(c["table"][b, t // 16]), t % 16
            if scaled:
                c["k"].view(torch.uint8)[page, slot] = 0x7F
                if t // 16 > (m - 1) // 16:
                    c["ks"][page] = math.nan if t // 16 % 2 else math.inf
            else:
                c["k"][page, slot] = math.nan if t % 2 else math.inf
            c["scores"][page, :, slot] = math.nan
    clean = dict(c, k=c["k"].clone(), ks=None if c["ks"] is None else c["ks"].nan_to_num(1.0, 1.0))
    if scaled:
        clean["k"].view(torch.uint8)[c["k"].view(torch.uint8) == 0x7F] = 0
    else:
        clean["k"] = c["k"].nan_to_num(0.0, 0.0, 0.0)
    for kw in (dict(), dict(num_ctas=2)):
        got = accumulate(sqa, gpu(c), mask_lens=torch.tensor(mask, dtype=torch.int32).cuda(), **kw)
        for b, (n, m) in enumerate(zip(lens, mask)):
            for t in range(m, n):
                assert (got[int(c["table"][b, t // 16]), :, t % 16] == 0).all(), (b, t)
        pages = {int(p) for b, n in enumerate(lens) for p in c["table"][b, : (n + 15) // 16]}
        behind = [p for p in range(len(c["scores"])) if p not in pages]
        assert_weights(got, dict(clean, scores=clean["scores"]), mask_lens=mask)
        assert torch.equal(got[behind].cpu(), c["scores"][behind])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("q_len", [1, 2, 3, 5, 7, 9, 13, 16])
def test_attention_ignores_them_too(sqa, q_len, dtype):
    """K, V and both scales of pages that lie behind the mask and within the lengths: the output's bits do not change."""
    from tests.test_gpu_scaled import attend, scaled_case, to_gpu

    lens, mask = [300, 700, 33], [80, 650, 32]
    c = scaled_case(q_len, lens, hkv=2, dtype=dtype, seed=q_len)
    masks = torch.tensor(mask, dtype=torch.int32).cuda()
    want = [attend(sqa, to_gpu(c), mask_lens=masks, num_ctas=n) for n in (0, 2)]
    for b, (n, m) in enumerate(zip(lens, mask)):
        for t in range(m, n):
            page, slot = int(c["table"][b, t // 16]), t % 16
            for side in "kv":
                c[side].view(torch.uint8)[page, slot] = 0x7F if t % 3 else 0xFF
                if t // 16 > (m - 1) // 16:
                    c[side + "s"][page] = math.nan if t // 16 % 2 else math.inf
    for (o, lse), n in zip(want, (0, 2)):
        got, got_lse = attend(sqa, to_gpu(c), mask_lens=masks, num_ctas=n)
        assert torch.equal(got, o) and torch.equal(got_lse, lse) and o.isfinite().all()
