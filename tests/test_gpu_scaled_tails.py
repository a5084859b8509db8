"""Block-scaled attention over rows that a few tokens dominate: what the other tokens add up to must not be lost.

The bound counts the kernel's own steps.  A probability P (relative to the row's base) enters the value
product as p0 + p1 / 32 + p2 / 2^10 + p3 / 2^20 in e4m3:

* the first three parts leave at most 2^-13 of P, and below their smallest step at most 2^-20;
* the fourth holds what they leave to e4m3's half step, 2^-4 of it, or to half its own smallest step, 2^-30; the
  fp16 in which it is formed has its smallest half step at 2^-30 as well.

So |error| <= 2^-13 P + min(2^-4 P, 2^-24) + 2^-29, relative to P less the larger P is.  The largest P of a row is at
least 2^-1; where one token dominates a stream's first block it is 2^min(7, gap - 12), with the gap in bits to the
smallest of the maxima of that block's four runs of 32 tokens (2^4 where the token comes later).  To that come the
scores' own error (384 products in fp32, relative to sum |q k|), the exponential's 2^-22, both in the numerator
and in the sum, and the rounding of the output.
"""

import math

import numpy as np
import pytest
import torch

from tests.test_gpu_scaled import F8

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sqa():
    if not torch.cuda.is_available() or F8 is None:
        pytest.skip("needs a CUDA device and torch.float8_e4m3fn")
    import small_q_attention_b200 as m

    return m


def dominated(q_len, n, at, dtype, *, spread=1.0, vs=None, seed=0, low=11.0, high=16.5):
    """One sequence, one KV head: the tokens `at` score `low`..`high` nats (by row) above the mean of the others, whose
    V is positive while theirs is zero: the output is what the others add up to."""
    g = torch.Generator().manual_seed(seed)
    pages = (n + 15) // 16
    table = torch.randperm(pages + 2, generator=g)[:pages].to(torch.int32).view(1, pages)
    rows = 4 * q_len
    query = spread * torch.randn(1, q_len, 4, 128, generator=g)
    gaps = torch.linspace(low, high, rows).view(1, q_len, 4)
    query[..., 0] = gaps * 128 ** 0.5 / 7.0
    k = torch.randn(pages * 16, 1, 128, generator=g).clamp(-7, 7) * 64
    v = 200 + 100 * torch.rand(pages * 16, 1, 128, generator=g)
    k[..., 0] = 0
    for t in at:
        k[t], v[t] = 0, 0
        k[t, 0, 0] = 448  # 7 at the page scale
    c = dict(q_len=q_len, table=table, seq_lens=torch.tensor([n], dtype=torch.int32), query=query.to(dtype))
    scales = torch.full((pages,), 1 / 256.0) if vs is None else vs(pages)
    for side, x in (("k", k), ("v", v)):
        paged = torch.zeros(pages + 2, 16, 1, 128)
        paged[table[0].long()] = x.view(pages, 16, 1, 128)
        c[side] = paged.to(F8)
    c["ks"] = torch.full((pages + 2, 1), 1 / 64.0)
    c["vs"] = torch.ones(pages + 2, 1)
    c["vs"][table[0].long(), 0] = scales
    return c


def assert_tail(out, c, top):
    """`top(y, limit)`: log2 of the row's largest P, from its scores y (log2, value scales included)."""
    at = c["table"][0].long()
    n = int(c["seq_lens"][0])
    k = (c["k"].double()[at] * c["ks"].double()[at][:, None, :, None]).reshape(-1, 128)[:n].numpy()
    vs = c["vs"].double()[at].repeat_interleave(16, dim=0)[:n, 0].numpy()
    v8 = c["v"].double()[at].reshape(-1, 128)[:n].numpy()
    q = c["query"].double().numpy()
    for qi in range(c["q_len"]):
        for h in range(4):
            limit = n - c["q_len"] + qi + 1
            x = k[:limit] @ q[0, qi, h] * 128 ** -0.5
            p = np.exp(x - x.max())
            total = p.sum()
            ref = p @ (v8[:limit] * vs[:limit, None]) / total
            y = x / math.log(2) + np.log2(vs[:limit])
            big = np.exp2(y - y.max() + top(y, limit))
            off = 2.0 ** -13 + np.minimum(2.0 ** -4, 2.0 ** -24 / big) + 2.0 ** -29 / big
            d = 2 * (384 * 2.0 ** -24 * (np.abs(k[:limit]) @ np.abs(q[0, qi, h])).max() * 128 ** -0.5 + 2.0 ** -22)
            tol = (p * (off + d)) @ (np.abs(v8[:limit]) * vs[:limit, None]) / total
            eps = torch.finfo(out.dtype).eps / 2
            tol = tol + eps * np.abs(ref) + (2.0 ** -25 if out.dtype == torch.float16 else 0)
            err = np.abs(out[0, qi, h].double().cpu().numpy() - ref)
            assert (err <= tol).all(), f"row {qi},{h}: worst {np.max(err / tol):.2f} of the bound, output {ref.mean():.4g}"


def first_block(y, limit):
    warps = [y[i:i + 32].max() for i in range(0, 128, 32)]
    return min(7.0, max(-1.0, max(warps) - min(warps) - 12.0))


def attend(sqa, c, **kw):
    g = {k: x.cuda() if isinstance(x, torch.Tensor) else x for k, x in c.items()}
    return sqa.small_q_attention_scaled(g["query"], g["k"], g["v"], g["ks"], g["vs"], g["table"], g["seq_lens"], 16,
                                        check=True, **kw)


DTYPES = pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])


@DTYPES
@pytest.mark.parametrize("spread", [1.0, 0.0], ids=["spread", "flat"])
@pytest.mark.parametrize("q_len", [1, 2, 4, 8, 16])
def test_tail_under_a_dominant_first_token(sqa, q_len, spread, dtype):
    c = dominated(q_len, 32768, [0], dtype, spread=spread, seed=q_len)
    for num_ctas in (1, 0, 5):  # one CTA: every token beside the first one's base
        assert_tail(attend(sqa, c, num_ctas=num_ctas), c, first_block)


@DTYPES
@pytest.mark.parametrize("q_len", [4, 16])
def test_tail_under_a_dominant_token_that_comes_later(sqa, q_len, dtype):
    """The base is raised when it comes; the tail lies before and behind it."""
    c = dominated(q_len, 20003, [5000], dtype, seed=q_len)
    for num_ctas in (1, 0):
        assert_tail(attend(sqa, c, num_ctas=num_ctas), c, lambda y, limit: 0.0)


@DTYPES
@pytest.mark.parametrize("q_len", [2, 8])
def test_tail_under_dominant_tokens_in_every_run_of_a_block(sqa, q_len, dtype):
    """All four runs of 32 tokens of the first block hold one: its largest P is 2^-1, and the floor is the parts' own."""
    c = dominated(q_len, 32768, [0, 40, 70, 127], dtype, seed=q_len, low=10.0, high=14.0)
    assert_tail(attend(sqa, c, num_ctas=1), c, lambda y, limit: -1.0)


@DTYPES
def test_tail_beside_value_scales_of_other_sizes(sqa, dtype):
    """The largest P counts the value scale: the dominant token's page has a larger one than the tail's pages."""
    def scales(pages):
        s = torch.exp2(torch.randint(-9, -5, (pages,), generator=torch.Generator().manual_seed(1)).float())
        s[0] = 2.0 ** -4
        return s

    c = dominated(4, 16384, [0], dtype, vs=scales, seed=3, low=10.0, high=13.0)
    assert_tail(attend(sqa, c, num_ctas=1), c, lambda y, limit: -1.0)


@DTYPES
def test_fp32_rows_of_a_dominated_sequence(sqa, dtype):
    c = dominated(4, 32768, [0], dtype, seed=9)
    out = torch.empty(c["query"].shape, dtype=torch.float32, device="cuda")
    attend(sqa, c, num_ctas=1, out=out)
    assert_tail(out, c, first_block)


@pytest.mark.parametrize("q_len", [4, 8, 16])
def test_the_same_call_gives_the_same_bits(sqa, q_len):
    """bf16, many sequences and CTAs, the caches read again and again."""
    cs = [dominated(q_len, n, [0], torch.bfloat16, seed=n) for n in (8192, 3001)]
    for c in cs:
        want = attend(sqa, c).clone()
        for _ in range(10):
            assert torch.equal(attend(sqa, c), want)


@DTYPES
@pytest.mark.parametrize("q_len", [1, 4, 8, 16])
@pytest.mark.parametrize("largest", [2.0 ** 30, 1.0, 2.0 ** -20])
def test_pages_of_zeros_beside_the_largest_value_scale(sqa, q_len, largest, dtype):
    """Tokens whose values are zero (their pages' scale is the append's 2^-100, or 0) count in the denominator in full, 0 to
    20 bits below the one page that holds values at the largest scale allowed, and so do those of a small scale.

    Bounds.  A score less its base is fma(s, c, log2 scale - base), |values| below 128 over these 90 bits of scales
    and 20 of scores: two roundings of 2^-18 at most, the same for all tokens of one page.  The log-sum-exp adds
    one of 2^-19 (top + log2 sum, below 64), log2's own 2^-22, the exponential's 2^-22 and the product's half step of
    2^-20: ln 2 (2^-17 + 2^-19 + 2^-22) + 2^-22 + 2^-20 < 2^-16.4.  An output takes the first two in its
    numerator and in its sum, the exponential's, and the parts' 2^-13: (2^-13 + 2^-15) of it."""
    n = 4096
    g = torch.Generator().manual_seed(q_len)
    table = torch.randperm(n // 16, generator=g).to(torch.int32).view(1, -1)
    at = table[0].long()
    query = torch.zeros(1, q_len, 4, 128)
    query[..., 0] = torch.linspace(0, 20, 4 * q_len).view(1, q_len, 4) * math.log(2) * 128 ** 0.5 / 7
    k, v = torch.zeros(n // 16, 16, 1, 128), torch.zeros(n // 16, 16, 1, 128)
    k[at[37], :, 0, 0] = 448
    v[at[37]] = 200 + 100 * torch.rand(16, 1, 128, generator=g)
    v[at[90:95]] = 100
    vs = torch.full((n // 16, 1), 2.0 ** -100)
    vs[at[::3]] = 0.0
    vs[at[90:95]] = 2.0 ** -60
    vs[at[37]] = largest
    c = dict(q_len=q_len, table=table, seq_lens=torch.tensor([n], dtype=torch.int32), query=query.to(dtype), k=k.to(F8), v=v.to(F8),
             ks=torch.full((n // 16, 1), 1 / 64.0), vs=vs)
    for num_ctas in (0, 1):
        out = torch.empty(query.shape, device="cuda")
        out, lse = attend(sqa, c, num_ctas=num_ctas, out=out, return_lse=True)
        x = 7.0 * c["query"][..., 0].double() * 128 ** -0.5  # of the page's 16 tokens; the others' is 0
        seen = n - q_len + 1 + torch.arange(q_len)[:, None].double()
        total = 16 * torch.exp(x) + seen - 16
        want = (torch.exp(x) / total)[..., None] * largest * v[at[37], :, 0].to(F8).double().sum(dim=0)
        assert ((lse.cpu().double() - total.log()).abs() <= 2.0 ** -16.4).all()
        assert ((out.cpu().double() - want).abs() <= (2.0 ** -13 + 2.0 ** -15) * want).all()
