"""The planned wrapper's runs with scores and its evictions: errors come before anything has changed that they should
have kept, and memory that a captured graph uses stays.
"""

import pytest
import torch

from tests.test_gpu_scaled import F8
from tests.test_gpu_scaled_loop import BATCH, HKV, Q, WIDTH, fresh, on_gpu, step_inputs

pytestmark = pytest.mark.gpu
SCALED = pytest.mark.parametrize("scaled", [True, False], ids=["e4m3", "16bit"])


@pytest.fixture(scope="module")
def sqa():
    if not torch.cuda.is_available() or F8 is None:
        pytest.skip("needs a CUDA device and torch.float8_e4m3fn")
    import small_q_attention_b200 as m

    return m


def planned(sqa, g, scaled, batch=BATCH, **kw):
    return sqa.PagedMTPAttention(torch.device("cuda", 0)).plan(batch, Q, HKV, g["k"].shape[0], WIDTH, 190,
                                                               block_scaled=scaled, **kw)


def lengths(*n):
    return torch.tensor(n, dtype=torch.int32).cuda()


def scales(g):
    return dict(key_scales=g["ks"], value_scales=g["vs"])


@SCALED
def test_checked_run_with_scores_reports_bad_metadata(sqa, scaled):
    """A length below q_len, one beyond the table and a bad page raise as without scores, and no score has changed."""
    g = on_gpu(fresh(scaled, torch.float16))
    query = step_inputs(1, Q, torch.float16)[0].cuda()
    attn = planned(sqa, g, scaled)
    before = g["scores"].clone()
    bad = g["table"].clone()
    bad[1, 1] = 10 ** 6
    for table, lens, error in ((g["table"], lengths(100, Q - 1, 150), ValueError), (g["table"], lengths(100, 37, 0), ValueError),
                               (g["table"], lengths(100, 37, 16 * WIDTH + 1), ValueError), (bad, lengths(100, 37, 150), IndexError)):
        for s in (None, g["scores"]):
            with pytest.raises(error):
                attn.run(query, g["k"], g["v"], table, lens, scores=s, check=True, **scales(g))
            assert torch.equal(g["scores"], before)
    attn.run(query, g["k"], g["v"], g["table"], lengths(100, Q, 150), scores=g["scores"], check=True, **scales(g))
    assert not torch.equal(g["scores"], before)
