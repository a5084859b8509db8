"""The block-scaled e4m3 cache on the GPU: append and attention against the 64-bit oracle.

The append is exact.  Attention's bound, per output element, with x the scaled scores,
p the probabilities and V the dequantised values:

* the output's own rounding: eps / 2 of its type, relative;
* a score is a sum of at most 3 x 128 products in fp32 (the query enters as at most
  three exact parts): off by at most 384 * 2^-24 * sum |q k|, and so is log2's input;
  the exponential adds 2^-22: relative error d of p, once in the numerator, once in the sum;
* p enters the second product with at least 12 significant bits for fp16 queries (2^-12) and 8
  for bf16 (2^-8 counts twice the rounding of 2^-9), relative, and values below 2^-18
  (bf16; 2^-22 for fp16) of a row's largest p |v| may be lost, each token at most once.
"""

import math

import numpy as np
import pytest
import torch

from oracle import append_scaled_reference, attention_scaled_reference, merge_partials

pytestmark = pytest.mark.gpu
F8 = getattr(torch, "float8_e4m3fn", None)


@pytest.fixture(scope="module")
def sqa():
    if not torch.cuda.is_available() or F8 is None:
        pytest.skip("needs a CUDA device and torch.float8_e4m3fn")
    import small_q_attention_b200 as m

    return m


def scaled_case(q_len, lens, *, hkv=8, dtype=torch.float16, seed=0, extra=5, spread=1.0, width=None):
    """Inputs on the CPU: pages of every magnitude, distinct pages in random order."""
    g = torch.Generator().manual_seed(seed)
    pages = [max(1, (n + 15) // 16) for n in lens]
    pool = sum(pages) + extra
    ids = torch.randperm(pool, generator=g).to(torch.int32)
    width = width or max(pages) + 1
    table = torch.full((len(lens), width), int(ids[-1]), dtype=torch.int32)
    cur = 0
    for b, n in enumerate(pages):
        table[b, :n] = ids[cur:cur + n]
        cur += n
    c = dict(lens=list(lens), q_len=q_len, hkv=hkv, table=table, seq_lens=torch.tensor(lens, dtype=torch.int32),
             query=torch.randn(len(lens), q_len, 4 * hkv, 128, generator=g).to(dtype))
    for side in "kv":
        x = torch.randn(pool, 16, hkv, 128, generator=g)
        c[side] = (x * 100).clamp(-448, 448).to(F8)
        c[side + "s"] = 0.01 * torch.exp(spread * torch.randn(pool, hkv, generator=g))
    return c


def to_gpu(c, layout="NHD"):
    g = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in c.items()}
    if layout == "HND":
        for side in "kv":
            g[side] = g[side].view(torch.uint8).permute(0, 2, 1, 3).contiguous().view(F8)
    return g


def attend(sqa, g, layout="NHD", **kw):
    return sqa.small_q_attention_scaled(g["query"], g["k"], g["v"], g["ks"], g["vs"], g["table"], g["seq_lens"], 16,
                                        kv_layout=layout, return_lse=True, **kw)


def reference(c, **kw):
    return attention_scaled_reference(c["query"].double().numpy(), c["k"].double().numpy(), c["v"].double().numpy(),
                                      c["ks"].double().numpy(), c["vs"].double().numpy(), c["table"].numpy(),
                                      c["seq_lens"].tolist(), **kw)


def assert_within(out, lse, want, query_dtype):
    ref, ref_lse, spread = want
    bf = query_dtype == torch.bfloat16
    d = 2 * (384 * 2.0 ** -24 * spread["dot"] + 2.0 ** -22)
    part, lost = (2.0 ** -8, 2.0 ** -18) if bf else (2.0 ** -12, 2.0 ** -22)
    n = 8192  # tokens of the longest case
    rounding = torch.finfo(out.dtype).eps / 2
    tol = rounding * np.abs(ref) + (d[..., None] + part) * spread["abs"] + (n * lost * spread["top"])[..., None] + 1e-30
    if out.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half a subnormal step
    err = np.abs(out.double().cpu().numpy() - ref)
    assert np.isfinite(err).all()
    assert (err <= tol).all(), f"{(err > tol).sum()} elements out of bounds, worst {np.max(err / tol):.2f} of it"
    got = lse.double().cpu().numpy()
    seen = np.isfinite(ref_lse)
    assert np.array_equal(np.isneginf(got), ~seen)
    # log of a sum whose terms are off by d, and the fp32 result's rounding
    assert (np.abs(got - np.where(seen, ref_lse, 0))[seen] <= (d + 2.0 ** -21 * (1 + np.abs(ref_lse)))[seen]).all()


CASES = [(1, [1], 1), (1, [0, 1, 17, 500], 4), (2, [33, 2, 1024], 8), (3, [3, 128, 129, 127, 1000], 2),
         (4, [4, 16, 17, 1000, 2048], 8), (5, [5, 4095, 63], 1), (8, [2048, 8, 9, 300], 2), (9, [9, 640], 3),
         (12, [12, 200, 777], 2), (16, [16, 31, 4096], 4), (4, [8192, 8191], 8)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("q_len,lens,hkv", CASES, ids=[f"q{q}-n{len(l)}-kv{max(l)}-h{h}" for q, l, h in CASES])
def test_attention(sqa, q_len, lens, hkv, dtype):
    c = scaled_case(q_len, lens, hkv=hkv, dtype=dtype, seed=q_len * 31 + len(lens))
    layout = "HND" if q_len % 2 else "NHD"
    out, lse = attend(sqa, to_gpu(c, layout), layout)
    assert out.dtype == dtype
    assert_within(out, lse, reference(c), dtype)


@pytest.mark.parametrize("num_ctas", [1, 2, 3, 7, 64, 333])
def test_attention_splits(sqa, num_ctas):
    c = scaled_case(4, [40, 700, 16, 0, 1500, 8], hkv=2, seed=7)
    g = to_gpu(c)
    out, lse = attend(sqa, g, num_ctas=num_ctas)
    assert_within(out, lse, reference(c), torch.float16)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("q_len", [1, 3, 6, 8, 9, 16])
def test_attention_many_blocks_a_cta(sqa, q_len, dtype):
    """Few CTAs over long sequences: every slot, buffer and ring position is used again and again."""
    c = scaled_case(q_len, [5003, 700, 2600], hkv=1, dtype=dtype, seed=q_len)
    g, want = to_gpu(c), reference(c)
    for num_ctas in (1, 2):
        out, lse = attend(sqa, g, num_ctas=num_ctas, check=True)
        assert_within(out, lse, want, dtype)


@pytest.mark.parametrize("q_len,batch", [(1, 1), (4, 1), (4, 3), (16, 1), (16, 2)])
def test_attention_length_hints(sqa, q_len, batch):
    """Right whatever the bounds say: tight, loose and wrong ones."""
    c = scaled_case(q_len, [4000 + 10 * b for b in range(batch)], hkv=8, seed=batch)
    g, want = to_gpu(c), reference(c)
    for hints in (dict(max_seq_len=4000 + 10 * (batch - 1), min_seq_len=4000), dict(max_seq_len=1 << 20), dict(max_seq_len=16),
                  dict(max_seq_len=100, min_seq_len=100)):
        out, lse = attend(sqa, g, **hints)
        assert_within(out, lse, want, torch.float16)


def test_attention_scale_ranges(sqa):
    """Scales across many powers of two, zero scales, an outlier page."""
    c = scaled_case(3, [500, 100, 260], hkv=2, seed=3, spread=3.0)
    c["vs"][c["table"][0, 3]] = 0.0
    c["ks"][c["table"][0, 5]] = 0.0
    c["vs"][c["table"][1]] = 0.0  # a sequence of zeros
    c["vs"][c["table"][2, 2]] *= 1e4
    out, lse = attend(sqa, to_gpu(c))
    assert_within(out, lse, reference(c), torch.float16)
    assert (out[1] == 0).all()


def test_attention_peaked_and_flat_rows(sqa):
    """A first token that takes most of the weight and thousands that share the rest; and
    queries of very different size in one call."""
    c = scaled_case(4, [8192, 4000], hkv=1, seed=5, spread=0.0)
    c["query"][:, 0] = 0.0  # flat: the mean of all values
    c["query"][:, 1] *= 20.0  # nearly one-hot
    c["query"][:, 2] *= 2.0 ** -9
    first = c["table"][:, 0].long()
    k = c["k"].float()
    k[first, 0, 0] = (40 * c["query"][:, 3, 0].float()).clamp(-448, 448)
    c["k"] = k.to(F8)
    out, lse = attend(sqa, to_gpu(c))
    assert_within(out, lse, reference(c), torch.float16)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("step", [0.001, 0.01, 0.05, 0.2])
def test_attention_creeping_maximum(sqa, step, dtype):
    """Scores that rise from token to token, so that a row's running base is passed by any amount up
    to where it is raised, with value scales just under and just over powers of two."""
    n = 4096
    c = scaled_case(2, [n, n // 2 + 5], hkv=2, dtype=dtype, seed=11, spread=0.0)
    c["query"][:] = 0.0
    c["query"][..., 0] = 1.0
    c["query"][:, 1, ::2, 0] = -1.0  # falls for some rows
    k = torch.zeros_like(c["k"].float())
    for b, row in enumerate(c["table"]):
        for t in range(c["lens"][b]):
            k[row[t // 16], t % 16, :, 0] = 16 + (t % 16) // 2  # within a page by e4m3's steps
    for b, row in enumerate(c["table"]):  # from page to page by the scale
        for j in range((c["lens"][b] + 15) // 16):
            c["ks"][row[j]] = step * 128 ** 0.5 * (16 * j + 8) / 20
    c["k"] = k.to(F8)
    c["vs"][:] = 1.99
    c["vs"][::3] = 1.01
    out, lse = attend(sqa, to_gpu(c))
    assert_within(out, lse, reference(c), dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_attention_ignores_what_a_row_does_not_see(sqa, dtype):
    """NaN bytes and NaN or infinite scales behind the sequence and in other sequences' pages, and
    NaN in draft tokens' K and V that earlier drafts do not see."""
    c = scaled_case(4, [37, 50, 16, 129], hkv=2, dtype=dtype, seed=5)
    want = reference(c)
    k8, v8 = c["k"].view(torch.uint8), c["v"].view(torch.uint8)
    used = set()
    for b, n in enumerate(c["lens"]):
        used |= set(c["table"][b, : (n + 15) // 16].tolist())
        if n % 16:
            k8[c["table"][b, n // 16], n % 16:] = 0x7F
            v8[c["table"][b, n // 16], n % 16:] = 0xFF
    for page in set(range(len(k8))) - used:
        k8[page] = v8[page] = 0x7F
        c["ks"][page], c["vs"][page] = math.nan, math.inf
    out, lse = attend(sqa, to_gpu(c))
    assert_within(out, lse, want, dtype)
    for b, n in enumerate(c["lens"]):  # the last draft: rows 0..2 do not see it
        k8[c["table"][b, (n - 1) // 16], (n - 1) % 16] = 0x7F
        v8[c["table"][b, (n - 1) // 16], (n - 1) % 16, :, 5] = 0x7F
    out, lse = attend(sqa, to_gpu(c))
    assert_within(out[:, :3], lse[:, :3], (want[0][:, :3], want[1][:, :3], {k: v[:, :3] for k, v in want[2].items()}), dtype)
    assert out[:, 3].isnan().all()


def test_attention_nan_value_reaches_only_rows_that_see_it(sqa):
    c = scaled_case(4, [37, 131], hkv=1, seed=6)
    want = reference(c)[0]
    for b, n in enumerate(c["lens"]):  # draft 2's V, dimension 5
        c["v"].view(torch.uint8)[c["table"][b, (n - 2) // 16], (n - 2) % 16, :, 5] = 0x7F
    out, _ = attend(sqa, to_gpu(c))
    assert out[:, 2:, :, 5].isnan().all()
    clean = out.clone()
    clean[:, 2:, :, 5] = 0
    assert not clean.isnan().any()
    assert np.allclose(out[:, :2].float().cpu().numpy(), want[:, :2], rtol=2e-3, atol=2e-2)


def test_attention_bad_queries_stay_in_their_row(sqa):
    c = scaled_case(2, [300, 40], hkv=2, seed=8)
    want = reference(c)
    c["query"][0, 0, 1, 3] = math.inf
    c["query"][0, 1, 6, 0] = math.nan
    c["query"][1, 0, 0] = math.nan
    out, lse = attend(sqa, to_gpu(c))
    bad = torch.zeros(out.shape[:3], dtype=torch.bool)
    bad[0, 0, 1] = bad[0, 1, 6] = bad[1, 0, 0] = True
    assert out.cpu()[bad].isnan().all() and lse.cpu()[bad].isnan().all()
    keep = (~bad).numpy()
    err = np.abs(out.double().cpu().numpy() - want[0])[keep]
    assert np.isfinite(err).all() and err.max() < 2e-2


def test_attention_scales_and_mask_lens(sqa):
    """sm_scale, out_scale, a shard of a longer sequence, fp32 rows, and the shards' merge."""
    c = scaled_case(4, [700], hkv=2, seed=9)
    whole = reference(c, sm_scale=0.05, out_scale=3.0)
    g = to_gpu(c)
    out, lse = attend(sqa, g, sm_scale=0.05, out_scale=3.0)
    assert_within(out, lse, whole, torch.float16)
    parts = []
    for lo, hi in ((0, 20), (20, 44)):  # pages of the two shards
        shard = dict(c, table=c["table"][:, lo:hi].contiguous(), seq_lens=torch.tensor([min(700, hi * 16) - lo * 16],
                                                                                       dtype=torch.int32))
        mask = torch.tensor([700 - lo * 16], dtype=torch.int32)
        gs = to_gpu(shard)
        o32 = torch.empty(c["query"].shape, dtype=torch.float32, device="cuda")
        o, l = attend(sqa, gs, mask_lens=mask.cuda(), sm_scale=0.05, out=o32)
        assert o is o32 or o.data_ptr() == o32.data_ptr()
        assert_within(o, l, reference(shard, mask_lens=mask.tolist(), sm_scale=0.05), torch.float16)
        parts.append((o, l))
    merged = sqa.merge_partials(torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts]))
    whole = reference(c, sm_scale=0.05)
    assert_within(merged, lse, whole, torch.float16)
    # a shard behind a row's last token: nothing is seen
    gs["seq_lens"].fill_(2)
    o, l = attend(sqa, gs, mask_lens=torch.tensor([1], dtype=torch.int32, device="cuda"))
    assert (o[:, :3] == 0).all() and torch.isneginf(l[:, :3]).all() and torch.isfinite(l[:, 3]).all()


def test_attention_strided_pools(sqa):
    """K and V interleaved per page in one pool, their scales too."""
    c = scaled_case(4, [100, 2000, 500], seed=12)
    g, want = to_gpu(c), reference(c)
    pool = torch.stack([g["k"].view(torch.uint8), g["v"].view(torch.uint8)], dim=1).contiguous().view(F8)
    scales = torch.stack([g["ks"], g["vs"]], dim=1).contiguous()
    g2 = dict(g, k=pool[:, 0], v=pool[:, 1], ks=scales[:, 0], vs=scales[:, 1])
    out, lse = attend(sqa, g2)
    assert_within(out, lse, want, torch.float16)


def test_attention_is_deterministic_and_graphs_do_not_share(sqa):
    c1, c2 = (scaled_case(4, [3000, 200, 70], hkv=4, seed=s) for s in (1, 2))
    g1, g2 = to_gpu(c1), to_gpu(c2)
    eager = [attend(sqa, g)[0].clone() for g in (g1, g2)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    s = torch.cuda.Stream()
    for g in (g1, g2):  # captured on one stream, replayed at the same time on two
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(attend(sqa, g)[0])
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, e) for o, e in zip(outs, eager))


def test_attention_compiled_and_from_two_threads(sqa):
    """The registered operator under torch.compile's tracing, and calls from two host threads on their
    own streams at once."""
    import threading

    cases = [scaled_case(4, [3000, 40], hkv=2, seed=s) for s in (1, 2)]
    gs = [to_gpu(c) for c in cases]
    want = [attend(sqa, g) for g in gs]
    f = lambda g: torch.ops.sqa_b200.small_q_attention_scaled(  # noqa: E731
        g["query"], g["k"], g["v"], g["ks"], g["vs"], g["table"], g["seq_lens"], 16)
    o, lse = f(gs[0])
    assert torch.equal(o, want[0][0]) and torch.equal(lse, want[0][1])
    torch.cuda.synchronize()
    bad = []

    def loop(g, w):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                o, lse = attend(sqa, g)
                torch.cuda.current_stream().synchronize()
                bad.append(not (torch.equal(o, w[0]) and torch.equal(lse, w[1])))

    threads = [threading.Thread(target=loop, args=(g, w)) for g, w in zip(gs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(bad) == 60 and not any(bad)


def test_attention_bad_metadata(sqa):
    c = scaled_case(4, [40, 100], hkv=2, seed=4)
    g = to_gpu(c)
    ok = attend(sqa, g, check=True)[0]
    bad = dict(g, table=g["table"].clone())
    bad["table"][0, 1] = 10 ** 6
    with pytest.raises(IndexError):
        attend(sqa, bad, check=True)
    bad["table"][0, 1] = -3
    with pytest.raises(IndexError):
        attend(sqa, bad, check=True)
    with pytest.raises(ValueError, match="at least q_len"):
        attend(sqa, dict(g, seq_lens=torch.tensor([3, 100], dtype=torch.int32, device="cuda")), check=True)
    with pytest.raises(ValueError, match="exceeds"):
        attend(sqa, dict(g, seq_lens=torch.tensor([40, 16 * g["table"].shape[1] + 1], dtype=torch.int32, device="cuda")), check=True)
    attend(sqa, dict(g, seq_lens=torch.tensor([40, -5], dtype=torch.int32, device="cuda")))
    torch.cuda.synchronize()
    again = attend(sqa, g)[0]
    assert torch.equal(ok, again)


def test_attention_refusals(sqa):
    g = to_gpu(scaled_case(2, [40], hkv=2, seed=4))
    with pytest.raises(ValueError, match="E4M3"):
        attend(sqa, dict(g, k=g["k"].to(torch.float16), v=g["v"].to(torch.float16)))
    with pytest.raises(ValueError, match="scales"):
        attend(sqa, dict(g, ks=g["ks"].half()))
    with pytest.raises(ValueError, match="scales"):
        attend(sqa, dict(g, vs=g["vs"][:-1]))
    with pytest.raises(ValueError, match="scales"):
        attend(sqa, dict(g, vs=g["vs"].t().contiguous().t()))
    with pytest.raises(ValueError, match="on the same device"):
        attend(sqa, dict(g, ks=g["ks"].cpu()))
    with pytest.raises(ValueError, match="out must be"):
        attend(sqa, g, out=torch.empty_like(g["query"], dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="workspace"):
        attend(sqa, g, workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError):
        attend(sqa, dict(g, query=None))


# ------------------------------------------------------------------ append
def append_case(q_len, lens, hkv, dtype, seed):
    c = scaled_case(q_len, lens, hkv=hkv, dtype=dtype, seed=seed)
    g = torch.Generator().manual_seed(seed + 100)
    for side in "kv":
        x = torch.randn(len(lens), q_len, hkv, 128, generator=g) * torch.exp(2 * torch.randn(len(lens), q_len, 1, 1, generator=g))
        c["new_" + side] = x.to(dtype)
        # half the pages hold powers of two, as the append itself leaves them
        c[side + "s"] = torch.where(torch.rand(c[side + "s"].shape, generator=g) < 0.5,
                                    torch.exp2(torch.round(torch.log2(c[side + "s"]))), c[side + "s"])
    return c


def append(sqa, g, layout="NHD", **kw):
    return sqa.cache_append_scaled(g["new_k"], g["new_v"], g["k"], g["v"], g["ks"], g["vs"], g["table"], g["seq_lens"],
                                   kv_layout=layout, **kw)


def assert_appended(g, c, layout="NHD"):
    with np.errstate(all="ignore"):
        want = append_scaled_reference(*(c[x].double().numpy() for x in ("new_k", "new_v", "k", "v", "ks", "vs")),
                                       c["table"].numpy(), c["seq_lens"].tolist())
    for side, values, scales in (("k", want[0], want[2]), ("v", want[1], want[3])):
        got = g[side].float().double().cpu().numpy()
        got = got.transpose(0, 2, 1, 3) if layout == "HND" else got
        assert np.array_equal(g[side + "s"].double().cpu().numpy(), scales)
        assert np.array_equal(got, values, equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("q_len,lens,hkv", [
    (1, [1, 16, 17, 1000, 15], 8), (2, [2, 15, 17, 33], 3), (4, [4, 20, 18, 64, 65], 2), (16, [16, 31, 32, 47], 4),
    (17, [17, 18, 33, 40], 1), (100, [100, 111, 112, 1000], 2), (1001, [1001, 1010], 1)])
def test_append(sqa, q_len, lens, hkv, dtype):
    c = append_case(q_len, lens, hkv, dtype, seed=q_len)
    layout = "HND" if q_len % 2 else "NHD"
    g = to_gpu(c, layout)
    append(sqa, g, layout, check=True)
    assert_appended(g, c, layout)


def test_append_step_by_step(sqa):
    """Token by token over three pages, with growing magnitudes: the cache and scales follow the
    oracle through every requantisation, and the values stay within half a step of the largest scale."""
    n, hkv = 40, 2
    c = append_case(1, [1], hkv, torch.float16, seed=2)
    c["table"] = torch.tensor([[2, 0, 4]], dtype=torch.int32)
    g = to_gpu(c)
    gen = torch.Generator().manual_seed(1)
    tokens = torch.randn(n, 2, 1, 1, hkv, 128, generator=gen).half() * torch.linspace(0.1, 4, n)[:, None, None, None, None, None].half()
    for t in range(n):
        for x in (c, g):
            x["new_k"], x["new_v"] = (tokens[t, i].to(g["k"].device if x is g else "cpu") for i in (0, 1))
            x["seq_lens"] = torch.tensor([t + 1], dtype=torch.int32, device=g["k"].device if x is g else "cpu")
        append(sqa, g, check=True)
        assert_appended(g, c)
        c.update({k: g[k].cpu() for k in ("k", "v", "ks", "vs")})
    k = c["k"].float() * c["ks"][:, None, :, None]
    for t in range(n):
        page, slot = int(c["table"][0, t // 16]), t % 16
        exact = tokens[t, 0, 0, 0].float()
        # half a step of 2^-4, and e4m3's subnormal step of 2^-9 at the page's final scale, once when it is
        # stored and once more when a growing scale pushes it there
        assert ((k[page, slot] - exact).abs() <= exact.abs() * 2 ** -4 + c["ks"][page][:, None] * 2 ** -9).all()


def test_append_special_values(sqa):
    c = append_case(4, [20, 4, 36], 2, torch.bfloat16, seed=3)
    c["new_k"][0, 1, 0, 3], c["new_k"][0, 2, 1, 4], c["new_v"][1, 0, 0, 0] = math.inf, math.nan, -math.inf
    c["new_v"][2] = 0.0
    c["new_k"][1] = 0.0  # a page of zeros: the smallest scale
    c["new_k"][2, 0, 0] = 3e38
    g = to_gpu(c)
    append(sqa, g, check=True)
    assert_appended(g, c)
    assert (g["ks"].cpu()[c["table"][1, 0]] == 2.0 ** -100).all()


def test_append_bad_metadata(sqa):
    c = append_case(4, [20, 40, 100], 2, torch.float16, seed=4)
    c["seq_lens"] = torch.tensor([3, 40, 16 * c["table"].shape[1] + 1], dtype=torch.int32)
    c["table"][1, 2] = 10 ** 6
    g = to_gpu(c)
    with pytest.raises((ValueError, IndexError)):
        append(sqa, g, check=True)
    assert_appended(g, c)  # the good pages of the second sequence are written, nothing else
    c["table"][1, 2] = -1
    g = to_gpu(c)
    append(sqa, g)
    torch.cuda.synchronize()
    assert_appended(g, c)


@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 15, 2 ** 31 - 16])
def test_lengths_near_the_end_of_int32(sqa, length):
    """Rounded up to pages, they pass 32 bits: too long all the same, never short."""
    c = append_case(4, [20, 40, 100], 2, torch.float16, seed=8)
    c["seq_lens"] = torch.tensor([20, length, 100], dtype=torch.int32)
    g = to_gpu(c)
    with pytest.raises(ValueError, match="exceeds"):
        append(sqa, g, check=True)
    assert_appended(g, c)
    a = scaled_case(4, [40, 100], hkv=2, seed=8)
    g = to_gpu(a)
    full = 16 * g["table"].shape[1]
    with pytest.raises(ValueError, match="exceeds"):
        attend(sqa, dict(g, seq_lens=torch.tensor([40, length], dtype=torch.int32, device="cuda")), check=True)
    ok = attend(sqa, g)[0]
    clamped = attend(sqa, dict(g, seq_lens=torch.tensor([40, length], dtype=torch.int32, device="cuda")))[0]
    torch.cuda.synchronize()
    assert full >= 100 and torch.equal(ok[0], clamped[0])


def test_append_strided_pool_and_refusals(sqa):
    c = append_case(6, [30, 6, 77], 4, torch.float16, seed=5)
    g = to_gpu(c)
    pool = torch.stack([g["k"].view(torch.uint8), g["v"].view(torch.uint8)], dim=1).contiguous().view(F8)
    scales = torch.stack([g["ks"], g["vs"]], dim=1).contiguous()
    g2 = dict(g, k=pool[:, 0], v=pool[:, 1], ks=scales[:, 0], vs=scales[:, 1])
    append(sqa, g2, check=True)
    assert_appended(g2, c)
    with pytest.raises(ValueError, match="FP16 or BF16"):
        append(sqa, dict(g, new_k=g["new_k"].float(), new_v=g["new_v"].float()))
    with pytest.raises(ValueError, match="E4M3"):
        append(sqa, dict(g, k=g["k"].half(), v=g["v"].half()))
    with pytest.raises(ValueError, match="contiguous"):
        append(sqa, dict(g, new_k=g["new_k"].transpose(0, 1), new_v=g["new_v"].transpose(0, 1)))
    with pytest.raises(ValueError, match="KV heads"):
        append(sqa, dict(g, new_k=g["new_k"][:, :, :2].contiguous(), new_v=g["new_v"][:, :, :2].contiguous()))
    with pytest.raises(ValueError, match="scales"):
        append(sqa, dict(g, ks=g["ks"].double()))
    with pytest.raises(ValueError):
        append(sqa, dict(g, new_k=[1]))


def test_append_then_attend_on_another_stream(sqa):
    c = append_case(4, [100, 40, 2049], 2, torch.float16, seed=6)
    g = to_gpu(c)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        append(sqa, g)
        out, lse = attend(sqa, g)
    torch.cuda.synchronize()
    assert_appended(g, c)
    held = dict(c, **{k: g[k].cpu() for k in ("k", "v", "ks", "vs")})
    assert_within(out, lse, reference(held), torch.float16)
