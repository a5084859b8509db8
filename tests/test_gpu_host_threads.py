"""Calls that are a host thread's first use of CUDA: every entry point works from a new thread."""

import ctypes
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

    return m


def in_a_new_thread(f):
    got = []

    def run():
        try:
            got.append(f())
        except Exception as e:  # reported by the caller
            got.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    torch.cuda.synchronize()
    if isinstance(got[0], Exception):
        raise got[0]
    return got[0]


@pytest.fixture(scope="module")
def case(sqa):
    g = to_gpu(scaled_case(4, [3000, 40], hkv=2, seed=1))
    g["k16"], g["v16"] = ((g[s].float() * g[s + "s"][:, None, :, None]).half() for s in "kv")
    g["scores"] = torch.zeros(g["k"].shape[0], 2, 16, device="cuda")
    return g


@pytest.mark.parametrize("kernel", [0, 1, 2])
def test_attention_over_16_bit_caches(sqa, case, kernel):
    call = lambda: sqa.small_q_attention(case["query"], case["k16"], case["v16"], case["table"], case["seq_lens"], 16, kernel=kernel)  # noqa: E731
    want = call()
    assert torch.equal(in_a_new_thread(call), want)


def test_partial_attention(sqa, case):
    call = lambda: sqa.small_q_attention_partial(case["query"], case["k16"], case["v16"], case["table"], case["seq_lens"], 16)  # noqa: E731
    want = call()
    assert all(torch.equal(a, b) for a, b in zip(in_a_new_thread(call), want))


def test_block_scaled_operators(sqa, case):
    want = attend(sqa, case)
    assert all(torch.equal(a, b) for a, b in zip(in_a_new_thread(lambda: attend(sqa, case)), want))
    weigh = lambda: sqa.accumulate_attention_weights(case["query"], case["k"], case["table"], case["seq_lens"], want[1],  # noqa: E731
                                                     case["scores"].clone(), 16, key_scales=case["ks"])
    assert torch.equal(in_a_new_thread(weigh), weigh())

    def evict():
        c = {k: x.clone() if isinstance(x, torch.Tensor) else x for k, x in case.items()}
        return sqa.cache_evict(c["k"], c["v"], c["scores"], c["table"], c["seq_lens"], 100, key_scales=c["ks"], value_scales=c["vs"])[1]

    assert torch.equal(in_a_new_thread(evict), evict())


def test_planned_step(sqa, case):
    attn = sqa.PagedMTPAttention(torch.device("cuda", 0)).plan(2, 4, 2, case["k"].shape[0], case["table"].shape[1])
    call = lambda: attn.run(case["query"], case["k16"], case["v16"], case["table"], case["seq_lens"], check=True)  # noqa: E731
    want = call()
    assert torch.equal(in_a_new_thread(call), want)


def test_c_abi(sqa, case):
    """The C entry alone, with everything allocated before: no other CUDA call of the thread comes first."""
    from small_q_attention_b200 import _native
    from small_q_attention_b200.attention import _fill_args

    lib = _native.library()
    out = torch.empty_like(case["query"])
    a = _fill_args(case["query"], case["k"], case["v"], case["table"], case["seq_lens"], None, 0, 0, 0, 0, "NHD", None, 1.0)
    a.out = out.data_ptr()
    s = _native.SqaScales(case["ks"].data_ptr(), case["vs"].data_ptr(), 0)
    st = ctypes.c_int(0)
    need = lib.sqa_scaled_workspace_bytes(ctypes.byref(a), 0, ctypes.byref(st))
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    code = in_a_new_thread(lambda: lib.sqa_forward_scaled(ctypes.byref(a), ctypes.byref(s), ws.data_ptr(), need, None))
    assert code == 0 and torch.equal(out, attend(sqa, case)[0])
