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


def bytes_of(g):
    return [g[k].view(torch.uint8).clone() for k in ("k", "v", "scores")]


def test_scores_of_a_single_scale_fp8_plan_are_refused_before_the_step(sqa):
    g = on_gpu(fresh(True, torch.float16))
    query, *new = [x.cuda() for x in step_inputs(1, Q, torch.float16)]
    attn = planned(sqa, g, False, cache_dtype=F8)
    before, out = bytes_of(g), torch.full_like(query, 7.0)
    lens = lengths(100, 37, 150)
    new8 = [x.clamp(-448, 448).to(F8) for x in new]
    with pytest.raises(ValueError, match="block_scaled"):
        attn.run(query, g["k"], g["v"], g["table"], lens, out=out, append_keys=new8[0], append_values=new8[1], scores=g["scores"])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, bytes_of(g))) and (out == 7.0).all()
    attn.run(query, g["k"], g["v"], g["table"], lens, out=out, append_keys=new8[0], append_values=new8[1], check=True)
    assert not (out == 7.0).any()


@SCALED
def test_scores_of_the_wrong_kind_are_refused_before_the_step(sqa, scaled):
    g = on_gpu(fresh(scaled, torch.float16))
    query, *new = [x.cuda() for x in step_inputs(1, Q, torch.float16)]
    attn = planned(sqa, g, scaled)
    before, out = bytes_of(g), torch.full_like(query, 7.0)
    for s in (g["scores"][:-1], g["scores"].double(), g["scores"].cpu(), g["scores"].transpose(0, 1), g["scores"][..., :8], 3):
        with pytest.raises(ValueError, match="scores"):
            attn.run(query, g["k"], g["v"], g["table"], lengths(100, 37, 150), out=out, append_keys=new[0], append_values=new[1],
                     scores=s, **scales(g))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, bytes_of(g))) and (out == 7.0).all()


@SCALED
def test_graph_outlives_a_larger_plan(sqa, scaled):
    """A graph captured on a small plan replays after larger plans have outgrown its memory and the allocator
    has given out everything that was freed."""
    g, h, other = (on_gpu(fresh(scaled, torch.float16)) for _ in range(3))
    lens = lengths(100, 37, 150)
    query = step_inputs(1, Q, torch.float16)[0].cuda()
    attn = planned(sqa, g, scaled, batch=1)
    attn.run(query[:1], other["k"], other["v"], other["table"][:1], lens[:1], scores=other["scores"], **scales(other))  # warm up
    torch.cuda.synchronize()
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(query[:1])
    with torch.cuda.graph(graph):
        attn.run(query[:1], g["k"], g["v"], g["table"][:1], lens[:1], out=out, scores=g["scores"], **scales(g))
    used = [x.data_ptr() for x in (attn.workspace, attn._lse, attn._rows) if x is not None]
    attn.plan(BATCH, Q, HKV, g["k"].shape[0], WIDTH, 190, block_scaled=scaled, num_ctas=2000)  # a larger workspace
    attn.run(query, other["k"], other["v"], other["table"], lens, scores=other["scores"], **scales(other))
    assert attn.workspace.data_ptr() != used[0] and attn._lse.data_ptr() != used[1]
    torch.cuda.synchronize()
    taken = [torch.full((n,), 0xA5, dtype=torch.uint8, device="cuda") for n in (512, 4096, 1 << 16, 1 << 18, 1 << 20) for _ in range(64)]
    assert not {x.data_ptr() for x in taken} & set(used)
    attn.plan(1, Q, HKV, g["k"].shape[0], WIDTH, 190, block_scaled=scaled)
    want = attn.run(query[:1], h["k"], h["v"], h["table"][:1], lens[:1], scores=h["scores"], **scales(h))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(g["scores"], h["scores"])
    assert all((x == 0xA5).all() for x in taken)


def test_block_scaled_plan_hands_on_its_cluster_option(sqa, monkeypatch):
    """cluster=1 turns the even split off in the plan and in the run alike: with a workspace for one, not the other."""
    import small_q_attention_b200.wrapper as w

    g = on_gpu(fresh(True, torch.float16))
    query = step_inputs(1, Q, torch.float16)[0].cuda()
    seen = []
    call = w.small_q_attention_scaled
    monkeypatch.setattr(w, "small_q_attention_scaled", lambda *a, **kw: (seen.append(kw.get("cluster")), call(*a, **kw))[1])
    outs = [planned(sqa, g, True, min_seq_len=180, cluster=c).run(query, g["k"], g["v"], g["table"], lengths(190, 185, 180),
                                                                  check=True, **scales(g)) for c in (0, 1)]
    assert seen == [0, 1]
    assert torch.allclose(outs[0].float(), outs[1].float(), rtol=2e-3, atol=1e-3)
    with pytest.raises(ValueError, match="cluster"):
        call(query, g["k"], g["v"], g["ks"], g["vs"], g["table"], lengths(190, 185, 180), 16, cluster=2)


@SCALED
def test_checked_eviction_that_raises_leaves_lengths_and_caches_in_step(sqa, scaled):
    """One bad page: that sequence is left, the others are cut, and the lengths say so although the call raised."""
    g, h = on_gpu(fresh(scaled, torch.float16)), on_gpu(fresh(scaled, torch.float16))
    attn = planned(sqa, g, scaled)
    bad = g["table"].clone()
    bad[1, 2] = 10 ** 6
    lens = lengths(150, 120, 40)
    with pytest.raises(IndexError):
        attn.evict(g["k"], g["v"], g["scores"], bad, lens, 64, recent=8, sinks=2, check=True, **scales(g))
    assert lens.tolist() == [64, 120, 40]
    new, _ = sqa.cache_evict(h["k"], h["v"], h["scores"], bad, lengths(150, 120, 40), 64, recent=8, sinks=2, **scales(h))
    assert new.tolist() == [64, 120, 40] and all(torch.equal(a, b) for a, b in zip(bytes_of(g), bytes_of(h)))
    for kw in (dict(recent=65), dict(sinks=-1), dict(key_scales=3)):  # refused before the launch
        with pytest.raises(ValueError):
            attn.evict(g["k"], g["v"], g["scores"], g["table"], lens, 64, **{**scales(g), **kw})
    assert lens.tolist() == [64, 120, 40] and all(torch.equal(a, b) for a, b in zip(bytes_of(g), bytes_of(h)))
    with pytest.raises(ValueError):
        attn.evict(g["k"], g["v"], g["scores"], g["table"], None, 64, **scales(g))
