"""Attention weights and eviction on the GPU against the 64-bit oracle.

Eviction is exact (selection, moves, scores, scales).  A weight is a sum of rows of
exp(x - lse): x is a sum of at most 3 x 128 products in fp32, off by at most 384 * 2^-24 *
sum |q k|, the exponential adds 2^-22, the sum of the rows and the addition to the old score 2^-24 per
term, all relative to the sum of positive terms.
"""

import math

import numpy as np
import pytest
import torch

from oracle import attention_scaled_reference, evict_reference, weights_reference
from tests.test_gpu_scaled import F8, scaled_case, to_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sqa():
    if not torch.cuda.is_available() or F8 is None:
        pytest.skip("needs a CUDA device and torch.float8_e4m3fn")
    import small_q_attention_b200 as m

    return m


def weight_case(q_len, lens, hkv, dtype, scaled, seed, **kw):
    c = scaled_case(q_len, lens, hkv=hkv, dtype=dtype, seed=seed, spread=0.3, **kw)
    if not scaled:
        for side in "kv":
            c[side] = (c[side].float() * c[side + "s"][:, None, :, None]).to(dtype)
            c[side + "s"] = None
    g = torch.Generator().manual_seed(seed)
    c["scores"] = torch.rand(c["k"].shape[0], hkv, 16, generator=g)
    ones = np.ones((c["k"].shape[0], hkv))
    ks, vs = (ones if c[s] is None else c[s].double().numpy() for s in ("ks", "vs"))
    _, lse, _ = attention_scaled_reference(c["query"].double().numpy(), c["k"].double().numpy(), c["v"].double().numpy(),
                                           ks, vs, c["table"].numpy(), c["seq_lens"].tolist())
    c["lse"] = torch.from_numpy(lse).float()
    return c


def gpu(c, layout="NHD"):
    if c["k"].dtype == F8:
        return to_gpu(c, layout)
    g = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in c.items()}
    if layout == "HND":
        for side in "kv":
            g[side] = g[side].permute(0, 2, 1, 3).contiguous()
    return g


def accumulate(sqa, g, layout="NHD", **kw):
    return sqa.accumulate_attention_weights(g["query"], g["k"], g["table"], g["seq_lens"], g["lse"], g["scores"], 16,
                                            key_scales=g["ks"], kv_layout=layout, **kw)


def assert_weights(got, c, **kw):
    want, dot = weights_reference(c["query"].double().numpy(), c["k"].double().numpy(),
                                  None if c["ks"] is None else c["ks"].double().numpy(), c["table"].numpy(),
                                  c["seq_lens"].tolist(), c["lse"].numpy(), c["scores"].numpy(), **kw)
    rel = 384 * 2.0 ** -24 * dot + 2.0 ** -22 + (4 * c["q_len"] + 1) * 2.0 ** -24
    # lse is an input, but x - lse is rounded: half a step of the larger of the two, at most dot here
    rel += 2 * 2.0 ** -24 * (dot + 20)
    got = got.double().cpu().numpy()
    err = np.abs(got - want)
    assert (err <= rel * np.abs(want) + 1e-37).all(), f"worst {np.max(err / (rel * np.abs(want) + 1e-37)):.2f} of the bound"


CASES = [(1, [1], 1), (1, [0, 1, 17, 500], 4), (2, [33, 2, 1024], 8), (3, [3, 128, 129, 127, 1000], 2),
         (8, [2048, 8, 9, 300], 2), (9, [9, 640], 3), (16, [16, 31, 4096], 2), (4, [8192], 4)]


@pytest.mark.parametrize("scaled", [False, True], ids=["16bit", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("q_len,lens,hkv", CASES, ids=[f"q{q}-n{len(l)}-kv{max(l)}" for q, l, _ in CASES])
def test_weights(sqa, q_len, lens, hkv, dtype, scaled):
    c = weight_case(q_len, lens, hkv, dtype, scaled, seed=q_len + len(lens))
    layout = "HND" if q_len % 2 else "NHD"
    got = accumulate(sqa, gpu(c, layout), layout)
    assert_weights(got, c)


@pytest.mark.parametrize("scaled", [False, True], ids=["16bit", "e4m3"])
def test_weights_masks_and_garbage(sqa, scaled):
    """Shards, sm_scale, NaN in slots that no row sees and in the scores of new tokens, rows
    without tokens, splits and wrong length bounds."""
    c = weight_case(4, [37, 700, 16], 2, torch.float16, scaled, seed=3)
    mask = [37, 702, 14]
    for b, n in enumerate(c["lens"]):
        if n % 16:
            c["k"].view(torch.uint8)[c["table"][b, n // 16], n % 16:] = 0x7F
        c["scores"][c["table"][b, (n - 1) // 16], :, (n - 1) % 16] = math.nan  # a new token's slot
    c["lse"][1, 0, 0] = -math.inf  # counts nothing
    for kw in (dict(), dict(num_ctas=3), dict(num_ctas=200), dict(max_seq_len=20, min_seq_len=20)):
        got = accumulate(sqa, gpu(c), mask_lens=torch.tensor(mask, dtype=torch.int32).cuda(), sm_scale=0.07, **kw)
        assert_weights(got, c, mask_lens=mask, sm_scale=0.07)


@pytest.mark.parametrize("scaled", [False, True], ids=["16bit", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("q_len", [1, 4, 8, 9, 16])
def test_weights_many_blocks_a_cta(sqa, q_len, dtype, scaled):
    """Few CTAs over long sequences: every slot and ring position is used again and again."""
    c = weight_case(q_len, [5003, 700, 2600], 1, dtype, scaled, seed=q_len)
    for num_ctas in (1, 2):
        assert_weights(accumulate(sqa, gpu(c), num_ctas=num_ctas, check=True), c)


def test_weights_sum_to_the_rows(sqa):
    """With the attention's own log-sum-exp, the new weights of a step sum to the number of rows."""
    c = weight_case(4, [1000, 33, 4], 2, torch.bfloat16, True, seed=4)
    g = gpu(c)
    _, lse = sqa.small_q_attention_scaled(g["query"], g["k"], g["v"], g["ks"], g["vs"], g["table"], g["seq_lens"], 16,
                                          return_lse=True)
    g["lse"], g["scores"] = lse, torch.zeros_like(g["scores"])
    total = accumulate(sqa, g, check=True).double().sum(dim=(0, 2))
    assert torch.allclose(total, torch.full_like(total, 3 * 16.0), rtol=1e-4)


def test_weights_bad_metadata_and_refusals(sqa):
    c = weight_case(4, [40, 100], 2, torch.float16, False, seed=5)
    g = gpu(c)
    bad = dict(g, table=g["table"].clone(), scores=g["scores"].clone())
    bad["table"][0, 1] = 10 ** 6
    with pytest.raises(IndexError):
        accumulate(sqa, bad, check=True)
    good = accumulate(sqa, dict(g, scores=g["scores"].clone()))
    pages = [int(p) for p in c["table"][1, :7]]
    assert torch.equal(bad["scores"][pages], good[pages])  # the other sequence is done
    with pytest.raises(ValueError, match="at least q_len"):
        accumulate(sqa, dict(g, seq_lens=torch.tensor([3, 100], dtype=torch.int32, device="cuda"), scores=g["scores"].clone()),
                   check=True)
    with pytest.raises(ValueError, match="exceeds"):
        accumulate(sqa, dict(g, seq_lens=torch.tensor([40, 2000], dtype=torch.int32, device="cuda"), scores=g["scores"].clone()),
                   check=True)
    with pytest.raises(ValueError, match="key_scales"):
        accumulate(sqa, dict(g, ks=torch.ones(g["k"].shape[0], 2, device="cuda")))
    with pytest.raises(ValueError, match="key_scales"):
        accumulate(sqa, dict(g, k=g["k"].to(F8)))
    with pytest.raises(ValueError, match="lse"):
        accumulate(sqa, dict(g, lse=g["lse"].half()))
    with pytest.raises(ValueError, match="scores"):
        accumulate(sqa, dict(g, scores=g["scores"][:-1]))
    with pytest.raises(ValueError):
        accumulate(sqa, dict(g, lse=3))


# ------------------------------------------------------------------ eviction
def evict_case(lens, hkv, dtype, seed, ties=False, width=None):
    c = scaled_case(1, lens, hkv=hkv, seed=seed, width=width)
    g = torch.Generator().manual_seed(seed)
    if dtype != F8:
        for side in "kv":
            c[side] = c[side].float().to(dtype)
            c[side + "s"] = None
    c["scores"] = torch.rand(c["k"].shape[0], hkv, 16, generator=g) ** 4
    if ties:
        c["scores"] = torch.round(c["scores"] * 3) / 3
    return c


def evict(sqa, g, budget, layout="NHD", **kw):
    return sqa.cache_evict(g["k"], g["v"], g["scores"], g["table"], g["seq_lens"], budget, key_scales=g["ks"],
                           value_scales=g["vs"], kv_layout=layout, **kw)


def assert_evicted(g, c, lens, kept, budget, layout="NHD", **kw):
    num = lambda x: None if x is None else x.double().numpy()  # noqa: E731
    want = evict_reference(num(c["k"]), num(c["v"]), c["scores"].numpy(), c["table"].numpy(), c["seq_lens"].tolist(), budget,
                           ks=num(c["ks"]), vs=num(c["vs"]), **kw)
    assert np.array_equal(lens.cpu().numpy(), want[5])
    assert np.array_equal(kept.cpu().numpy(), want[6])
    assert np.array_equal(g["scores"].cpu().numpy(), want[2].astype(np.float32), equal_nan=True)
    for side, values, scales in (("k", want[0], want[3]), ("v", want[1], want[4])):
        got = g[side].double().cpu().numpy()
        got = got.transpose(0, 2, 1, 3) if layout == "HND" else got
        if scales is not None:
            assert np.array_equal(g[side + "s"].double().cpu().numpy(), scales)
        assert np.array_equal(got, values, equal_nan=True)


EVICT = [([1], 1, 1, 0, 0), ([2, 1, 0], 1, 2, 0, 1), ([40, 17, 16, 15], 16, 3, 4, 2), ([100, 33], 17, 1, 0, 0),
         ([1000, 999, 20], 64, 2, 64, 0), ([1000], 65, 2, 0, 65), ([513, 700], 512, 8, 100, 4), ([4096], 1000, 1, 100, 4),
         ([300] * 40, 40, 1, 8, 1), ([129, 5000], 128, 4, 1, 1), ([2050, 2048, 2049], 2048, 2, 500, 0)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, F8], ids=["fp16", "bf16", "e4m3"])
@pytest.mark.parametrize("lens,budget,hkv,recent,sinks", EVICT,
                         ids=[f"n{len(e[0])}-kv{max(e[0])}-to{e[1]}-r{e[3]}-s{e[4]}" for e in EVICT])
def test_evict(sqa, lens, budget, hkv, recent, sinks, dtype):
    c = evict_case(lens, hkv, dtype, seed=budget)
    layout = "HND" if budget % 2 else "NHD"
    g = gpu(c, layout)
    new, kept = evict(sqa, g, budget, layout, recent=recent, sinks=sinks, check=True)
    assert_evicted(g, c, new, kept, budget, layout, recent=recent, sinks=sinks)


@pytest.mark.parametrize("dtype", [torch.float16, F8], ids=["fp16", "e4m3"])
def test_evict_ties_and_odd_scores(sqa, dtype):
    """Many equal scores; NaN, infinities, negative values and both zeros; all equal."""
    c = evict_case([900, 450, 300], 2, dtype, seed=1, ties=True)
    flat = c["scores"].view(-1)
    g = torch.Generator().manual_seed(3)
    at = torch.randperm(flat.numel(), generator=g)
    for k, x in enumerate((math.nan, math.inf, -math.inf, -0.0, 0.0, -1e-40, 1e-40, -2.0)):
        flat[at[k * 60:(k + 1) * 60]] = x
    c["scores"][c["table"][2, :19].long()] = 0.25
    for budget, recent, sinks in ((200, 20, 3), (290, 0, 0), (37, 37, 0)):
        gg = gpu(c)
        new, kept = evict(sqa, gg, budget, recent=recent, sinks=sinks)
        assert_evicted(gg, c, new, kept, budget, recent=recent, sinks=sinks)


def test_evict_long_sequence_past_the_key_buffer(sqa):
    """Slices longer than the keys that shared memory holds (40 segments of one CTA each would be needed
    for a single-CTA slice: here 8 CTAs of 16384 and more positions)."""
    c = evict_case([140000], 1, F8, seed=2)
    g = gpu(c)
    new, kept = evict(sqa, g, 5000, recent=1000, sinks=4)
    assert_evicted(g, c, new, kept, 5000, recent=1000, sinks=4)


def test_evict_many_segments(sqa):
    """More segments than CTAs fit at once: clusters of every size down to one CTA."""
    for batch, hkv in ((10, 8), (30, 8), (90, 8)):
        c = evict_case([60 + b for b in range(batch)], hkv, torch.float16, seed=batch)
        g = gpu(c)
        new, kept = evict(sqa, g, 50, recent=10, sinks=1)
        assert_evicted(g, c, new, kept, 50, recent=10, sinks=1)


def test_evict_again_and_again(sqa):
    """The compacted cache is a cache: scores and positions carry over to the next eviction."""
    c = evict_case([700, 650], 2, F8, seed=5)
    for budget in (600, 599, 300, 31):
        g = gpu(c)
        new, kept = evict(sqa, g, budget, recent=min(20, budget), sinks=1)
        assert_evicted(g, c, new, kept, budget, recent=min(20, budget), sinks=1)
        c.update({k: g[k].cpu() for k in ("k", "v", "ks", "vs", "scores")}, seq_lens=new.cpu())


@pytest.mark.parametrize("dtype", [torch.float16, F8], ids=["16bit", "e4m3"])
def test_evict_slices_of_unequal_work(sqa, dtype):
    """CTAs of a cluster whose slices hold nothing or one score exchange their ranges at once, before the
    others may have read theirs; the call runs back to back, so that clusters start at every moment."""
    c = evict_case([65, 300, 66], 2, dtype, seed=11)
    for _ in range(20):
        g = gpu(c)
        new, kept = evict(sqa, g, 64, recent=32, sinks=30)
        assert_evicted(g, c, new, kept, 64, recent=32, sinks=30)


@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 15, 2 ** 31 - 16])
def test_lengths_near_the_end_of_int32(sqa, length):
    """Rounded up to pages, they pass 32 bits: too long all the same, never short."""
    c = evict_case([100, 90], 2, F8, seed=12)
    c["seq_lens"] = torch.tensor([length, 90], dtype=torch.int32)
    g = gpu(c)
    with pytest.raises(ValueError, match="exceeds"):
        evict(sqa, g, 32, check=True)
    g = gpu(c)
    new, kept = evict(sqa, g, 32)
    assert_evicted(g, c, new, kept, 32)


def test_evict_bad_metadata(sqa):
    """Bad sequences are left, whole; the others are cut."""
    c = evict_case([100, 90, 80, 70, 60], 2, F8, seed=6)
    c["seq_lens"] = torch.tensor([100, -3, 16 * c["table"].shape[1] + 1, 70, 60], dtype=torch.int32)
    c["table"][3, 4] = 10 ** 6
    c["table"][4, 3] = -1  # its last page
    g = gpu(c)
    with pytest.raises((ValueError, IndexError)):
        evict(sqa, g, 32, check=True)
    g = gpu(c)
    new, kept = evict(sqa, g, 32)
    assert_evicted(g, c, new, kept, 32)
    # a bad page id behind the sequence does not matter, nor one of a sequence that is left anyway
    c["table"][0, 7] = 10 ** 6
    c["seq_lens"][4] = 30
    g = gpu(c)
    new, kept = evict(sqa, g, 32)
    c["table"][4, 3] = 0
    assert_evicted(g, c, new, kept, 32)


def test_evict_strided_pool_outputs_and_refusals(sqa):
    c = evict_case([200, 100], 4, F8, seed=7)
    g = gpu(c)
    pool = torch.stack([g["k"].view(torch.uint8), g["v"].view(torch.uint8)], dim=1).contiguous().view(F8)
    scales = torch.stack([g["ks"], g["vs"]], dim=1).contiguous()
    g2 = dict(g, k=pool[:, 0], v=pool[:, 1], ks=scales[:, 0], vs=scales[:, 1])
    lens, kept = torch.empty_like(g["seq_lens"]), torch.empty(2, 4, 64, dtype=torch.int32, device="cuda")
    got = evict(sqa, g2, 64, recent=3, new_lens=lens, kept=kept, check=True)
    assert got[0].data_ptr() == lens.data_ptr() and got[1].data_ptr() == kept.data_ptr()
    assert_evicted(g2, c, lens, kept, 64, recent=3)
    for kw in (dict(budget=0), dict(budget=4, recent=5), dict(budget=4, recent=2, sinks=3), dict(budget=4, sinks=-1),
               dict(budget=4, recent=-1), dict(budget=4, new_lens=g["seq_lens"]), dict(budget=4, kept=kept)):
        with pytest.raises(ValueError):
            evict(sqa, g, kw.pop("budget"), **kw)
    with pytest.raises(ValueError, match="scales"):
        sqa.cache_evict(g["k"], g["v"], g["scores"], g["table"], g["seq_lens"], 4)
    with pytest.raises(ValueError, match="scores"):
        evict(sqa, dict(g, scores=g["scores"].double()), 4)
    with pytest.raises(ValueError):
        evict(sqa, dict(g, scores="x"), 4)


def test_evict_in_a_graph(sqa):
    c = evict_case([500, 300], 2, torch.float16, seed=8)
    g = gpu(c)
    evict(sqa, gpu(c), 100)  # warm up
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new, kept = evict(sqa, g, 100, recent=7, sinks=2)
    graph.replay()
    torch.cuda.synchronize()
    assert_evicted(g, c, new, kept, 100, recent=7, sinks=2)
