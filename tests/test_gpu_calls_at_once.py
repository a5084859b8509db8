"""The registered operators from several host threads on one stream, and inside a compiled step.  They run without Python's
lock, so the launches of two calls that share the stream's workspace must not come between one another.
"""

import threading

import pytest
import torch

from tests.test_gpu_scaled import F8, attend, scaled_case, to_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sqa():
    if not torch.cuda.is_available() or F8 is None:
        pytest.skip("needs a CUDA device and torch.float8_e4m3fn")
    import small_q_attention_b200 as m
    from small_q_attention_b200 import _native

    _native.torch_ext()
    return m


def scaled_op(g):
    return torch.ops.sqa_b200.small_q_attention_scaled(g["query"], g["k"], g["v"], g["ks"], g["vs"], g["table"], g["seq_lens"], 16)


def plain_op(g):
    return torch.ops.sqa_b200.small_q_attention(g["query"], g["k"], g["v"], g["table"], g["seq_lens"], 16)


def values(c, scaled):
    g = to_gpu(c)
    if not scaled:
        for side in "kv":
            g[side] = (g[side].float() * g[side + "s"][:, None, :, None]).half()
    return g


@pytest.mark.parametrize("scaled", [True, False], ids=["e4m3", "16bit"])
def test_threads_on_one_stream(sqa, scaled):
    """Two shapes that are split over many CTAs and merged; results are compared after the threads have ended."""
    op = scaled_op if scaled else lambda g: (plain_op(g),)
    gs = [values(scaled_case(4, lens, hkv=2, seed=i), scaled) for i, lens in enumerate(([5000, 300], [3001, 4000, 2222]))]
    want = [[x.clone() for x in op(g)] for g in gs]
    torch.cuda.synchronize()
    got, start = [[], []], threading.Barrier(2)

    def loop(i):
        start.wait()
        for _ in range(200):
            got[i].append(op(gs[i]))

    threads = [threading.Thread(target=loop, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for results, w in zip(got, want):
        assert len(results) == 200 and all(torch.equal(a, b) for r in results for a, b in zip(r, w))


def test_attention_compiles_without_a_graph_break(sqa):
    g = to_gpu(scaled_case(4, [3000, 40], hkv=2, seed=1))
    want, want_lse = attend(sqa, g)

    def step(query, k, v, ks, vs, table, lens):
        o, lse = torch.ops.sqa_b200.small_q_attention_scaled(query * 1.0, k, v, ks, vs, table, lens, 16)
        return o + 0.0, lse

    compiled = torch.compile(step, fullgraph=True, backend="aot_eager")
    for _ in range(2):
        o, lse = compiled(g["query"], g["k"], g["v"], g["ks"], g["vs"], g["table"], g["seq_lens"])
        assert torch.equal(o, want) and torch.equal(lse, want_lse)
