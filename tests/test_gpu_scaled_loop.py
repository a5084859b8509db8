"""Append, attention, attention weights and eviction together, as a serving loop runs them:
several steps of drafts of which some are accepted, against the 64-bit oracle at each step,
eagerly, through the planned wrapper and as one captured graph.
"""

import numpy as np
import pytest
import torch

from oracle import append_scaled_reference, attention_scaled_reference, evict_reference, weights_reference
from tests.test_gpu_eviction import assert_weights
from tests.test_gpu_scaled import F8, assert_within

pytestmark = pytest.mark.gpu
BATCH, Q, HKV, WIDTH, BUDGET, RECENT, SINKS = 3, 4, 2, 12, 96, 24, 2


@pytest.fixture(scope="module")
def sqa():
    if not torch.cuda.is_available() or F8 is None:
        pytest.skip("needs a CUDA device and torch.float8_e4m3fn")
    import small_q_attention_b200 as m

    return m


def fresh(scaled, dtype):
    """An empty cache whose pages hold whatever was there before."""
    g = torch.Generator().manual_seed(1)
    pool = BATCH * WIDTH + 4
    s = dict(table=torch.randperm(pool, generator=g)[: BATCH * WIDTH].to(torch.int32).view(BATCH, WIDTH),
             scores=torch.rand(pool, HKV, 16, generator=g))
    for side in "kv":
        x = torch.randn(pool, 16, HKV, 128, generator=g)
        s[side] = x.clamp(-448, 448).to(F8) if scaled else x.to(dtype)
        s[side + "s"] = torch.rand(pool, HKV, generator=g) if scaled else None
    return s


def step_inputs(step, q_len, dtype):
    g = torch.Generator().manual_seed(100 + step)
    grow = 1.0 + 0.2 * step  # scales have to follow
    new = [(grow * torch.randn(BATCH, q_len, HKV, 128, generator=g)).to(dtype) for _ in range(2)]
    return (1.5 * torch.randn(BATCH, q_len, 4 * HKV, 128, generator=g)).to(dtype), *new


def on_gpu(s):
    return {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in s.items()}


def num(x):
    return None if x is None else x.double().cpu().numpy()


def expected_append(before, new, lens):
    if before["ks"] is not None:
        return append_scaled_reference(num(new[0]), num(new[1]), num(before["k"]), num(before["v"]), num(before["ks"]),
                                       num(before["vs"]), before["table"].numpy(), lens)
    from oracle import cache_append_reference

    k, v = cache_append_reference(new[0].float(), new[1].float(), before["k"].float(), before["v"].float(),
                                  before["table"], np.array(lens))
    return k.astype(np.float64), v.astype(np.float64), None, None


@pytest.mark.parametrize("scaled", [True, False], ids=["e4m3", "16bit"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_decoding_with_eviction(sqa, dtype, scaled):
    g = on_gpu(fresh(scaled, dtype))
    held = [0] * BATCH  # committed tokens of each sequence
    rng = np.random.default_rng(3)
    evictions = 0
    for step in range(9):
        q_len = 45 if step == 0 else Q  # a prompt, then drafts
        query, *new = step_inputs(step, q_len, dtype)
        lens = [n + q_len for n in held]
        seq = torch.tensor(lens, dtype=torch.int32).cuda()
        before = {k: (v.cpu() if isinstance(v, torch.Tensor) else v) for k, v in g.items()}
        append = sqa.cache_append_scaled if scaled else sqa.cache_append
        scales = (g["ks"], g["vs"]) if scaled else ()
        append(new[0].cuda(), new[1].cuda(), g["k"], g["v"], *scales, g["table"], seq, check=True)
        want = expected_append(before, new, lens)
        for name, x in zip(("k", "v", "ks", "vs"), want):
            assert x is None or np.array_equal(num(g[name]), x), (step, name)
        if step:  # the prompt's attention is another kernel's work; its scores start at zero here
            q = query.cuda()
            if scaled:
                out, lse = sqa.small_q_attention_scaled(q, g["k"], g["v"], g["ks"], g["vs"], g["table"], seq, 16,
                                                        return_lse=True, check=True)
            else:
                out, lse = sqa.small_q_attention_partial(q, g["k"], g["v"], g["table"], seq, 16, check=True)
                out = out.to(dtype)
            ones = np.ones((g["k"].shape[0], HKV))
            ref = attention_scaled_reference(num(query), num(g["k"]), num(g["v"]), num(g["ks"]) if scaled else ones,
                                             num(g["vs"]) if scaled else ones, before["table"].numpy(), lens)
            if scaled:
                assert_within(out, lse, ref, dtype)
            else:
                # this kernel rounds P and its output to 16 bits: half a step of each, relative to what
                # they carry (2^-8 of a value of 6 in bf16 is 0.023: no fixed bound would do); 2^-12 for its fp32 sums
                half = torch.finfo(dtype).eps / 2
                assert (np.abs(num(out) - ref[0]) <= half * np.abs(ref[0]) + (half + 2.0 ** -12) * ref[2]["abs"] + 1e-6).all()
            c = dict(query=query, k=g["k"].cpu(), ks=None if not scaled else g["ks"].cpu(), table=before["table"],
                     seq_lens=torch.tensor(lens), lse=lse.cpu(), scores=before["scores"], q_len=Q)
            sqa.accumulate_attention_weights(q, g["k"], g["table"], seq, lse, g["scores"], 16, key_scales=g["ks"], check=True)
            assert_weights(g["scores"], c)
            held = [n - int(r) for n, r in zip(lens, rng.integers(0, Q, BATCH))]  # the last drafts are rejected
        else:
            g["scores"].zero_()
            held = lens
        if step % 3 == 2:
            budget = 40 + step
            seq = torch.tensor(held, dtype=torch.int32).cuda()
            before = {k: (v.cpu() if isinstance(v, torch.Tensor) else v) for k, v in g.items()}
            new_lens, kept = sqa.cache_evict(g["k"], g["v"], g["scores"], g["table"], seq, budget, recent=RECENT, sinks=SINKS,
                                             key_scales=g["ks"], value_scales=g["vs"], check=True)
            k, v, sc, ks, vs, ln, kp = evict_reference(num(before["k"]), num(before["v"]), before["scores"].numpy(),
                                                       before["table"].numpy(), held, budget, recent=RECENT, sinks=SINKS,
                                                       ks=num(before["ks"]), vs=num(before["vs"]))
            assert np.array_equal(kept.cpu().numpy(), kp) and np.array_equal(new_lens.cpu().numpy(), ln)
            assert np.array_equal(num(g["k"]), k) and np.array_equal(num(g["v"]), v)
            assert np.array_equal(g["scores"].cpu().numpy(), sc)
            assert ks is None or (np.array_equal(num(g["ks"]), ks) and np.array_equal(num(g["vs"]), vs))
            evictions += int(any(n > budget for n in held))
            held = ln.tolist()
    assert evictions


@pytest.mark.parametrize("scaled", [True, False], ids=["e4m3", "16bit"])
def test_wrapper_step_is_the_operators_and_captures(sqa, scaled):
    """run(scores=...) and evict() of the planned wrapper do what the operators do, and a captured step
    replays on new inputs."""
    dtype = torch.float16
    g, h = on_gpu(fresh(scaled, dtype)), on_gpu(fresh(scaled, dtype))
    lens = torch.tensor([100, 37, 150], dtype=torch.int32).cuda()
    attn = sqa.PagedMTPAttention(torch.device("cuda", 0)).plan(BATCH, Q, HKV, g["k"].shape[0], WIDTH, 190, block_scaled=scaled)
    query, *new = [x.cuda() for x in step_inputs(1, Q, dtype)]
    out = torch.empty_like(query)
    kw = dict(out=out, append_keys=new[0], append_values=new[1])
    run = lambda s, **k: attn.run(query, s["k"], s["v"], s["table"], lens, key_scales=s["ks"], value_scales=s["vs"],  # noqa: E731
                                  scores=s["scores"], **kw, **k)
    run(on_gpu(fresh(scaled, dtype)))  # warm up
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(g)
    for step in (1, 2):
        for x, y in zip((query, *new), step_inputs(step, Q, dtype)):
            x.copy_(y)
        graph.replay()
        if scaled:
            sqa.cache_append_scaled(new[0], new[1], h["k"], h["v"], h["ks"], h["vs"], h["table"], lens)
            want, lse = sqa.small_q_attention_scaled(query, h["k"], h["v"], h["ks"], h["vs"], h["table"], lens, 16, 190,
                                                     return_lse=True)
        else:
            sqa.cache_append(new[0], new[1], h["k"], h["v"], h["table"], lens)
            want, lse = sqa.small_q_attention_partial(query, h["k"], h["v"], h["table"], lens, 16, max_seq_len=190)
            want = want.to(dtype)
        sqa.accumulate_attention_weights(query, h["k"], h["table"], lens, lse, h["scores"], 16, 190, key_scales=h["ks"])
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(g["scores"], h["scores"])
        assert torch.equal(g["k"].view(torch.uint8), h["k"].view(torch.uint8))
        lens += 4
    scales = dict(key_scales=g["ks"], value_scales=g["vs"])
    kept = attn.evict(g["k"], g["v"], g["scores"], g["table"], lens, 64, recent=8, sinks=2, check=True, **scales)
    assert lens.tolist() == [64, 45, 64] and kept.shape == (BATCH, HKV, 64) and (kept[1, :, 45:] == -1).all()
    with pytest.raises(ValueError, match="block_scaled"):
        attn.run(query, g["k"], g["v"], g["table"], lens, **({} if scaled else dict(key_scales=1, value_scales=1)))


@pytest.mark.parametrize("scaled", [True, False], ids=["e4m3", "16bit"])
def test_wrapper_graph_outlives_a_smaller_plan(sqa, scaled):
    """A graph captured with scores keeps its memory when the object is planned again and run eagerly."""
    dtype = torch.float16
    g, h, other = (on_gpu(fresh(scaled, dtype)) for _ in range(3))
    lens = torch.tensor([100, 37, 150], dtype=torch.int32).cuda()
    query = step_inputs(1, Q, dtype)[0].cuda()
    attn = sqa.PagedMTPAttention(torch.device("cuda", 0))
    plan = lambda n: attn.plan(n, Q, HKV, g["k"].shape[0], WIDTH, 190, block_scaled=scaled)  # noqa: E731
    scales = lambda s: dict(key_scales=s["ks"], value_scales=s["vs"])  # noqa: E731
    out = torch.empty_like(query)
    plan(BATCH)
    attn.run(query, other["k"], other["v"], other["table"], lens, scores=other["scores"], **scales(other))  # warm up
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attn.run(query, g["k"], g["v"], g["table"], lens, out=out, scores=g["scores"], **scales(g))
    kept = attn._lse.data_ptr()
    plan(1)
    attn.run(query[:1], other["k"], other["v"], other["table"][:1], lens[:1], scores=other["scores"], **scales(other))
    plan(BATCH)
    want = attn.run(query, h["k"], h["v"], h["table"], lens, scores=h["scores"], **scales(h))
    assert attn._lse.data_ptr() == kept
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(g["scores"], h["scores"])


def test_wrapper_plan_refusals(sqa):
    attn = sqa.PagedMTPAttention(torch.device("cuda", 0))
    with pytest.raises(RuntimeError, match="plan"):
        attn.evict(None, None, None, None, None, 4)
    with pytest.raises(ValueError, match="one kernel"):
        attn.plan(BATCH, Q, HKV, 40, WIDTH, block_scaled=True, cluster=4)
    with pytest.raises(ValueError, match="one kernel"):
        sqa.PagedMTPAttention(torch.device("cuda", 0), kernel=1).plan(BATCH, Q, HKV, 40, WIDTH, block_scaled=True)
