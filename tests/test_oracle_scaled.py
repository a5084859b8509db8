"""The oracle of the block-scaled cache and of eviction against hand-worked values, and
the refusals of the C ABI and the torch extension (no GPU: every call ends in a check)."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import (append_scaled_reference, attention_scaled_reference, evict_reference, page_scale, round_e4m3,
                    weights_reference)


def test_round_e4m3_is_torchs_rounding():
    x = torch.cat([torch.linspace(-470, 470, 4001), torch.linspace(-0.1, 0.1, 4001), torch.tensor([0.0, 2.0 ** -10])])
    want = x.clamp(-448, 448).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(round_e4m3(x.double().numpy()), want)
    assert np.isnan(round_e4m3(np.nan)) and round_e4m3(np.inf) == 448


@pytest.mark.parametrize("amax,scale", [(448.0, 1.0), (448.5, 2.0), (1.0, 2.0 ** -8), (0.0, 2.0 ** -100), (1.75, 2.0 ** -8),
                                        (1.7500001, 2.0 ** -7)])
def test_page_scale(amax, scale):
    assert page_scale(amax) == scale


def test_append_grows_a_scale_and_keeps_older_values():
    kc = np.zeros((2, 16, 1, 128))
    kc[1, :3] = 8.0  # three older tokens of page 1 stand for 8 * 0.5
    ks = np.array([[1.0], [0.5]])
    new = np.full((1, 2, 1, 128), 448.0)
    k, v, s, _ = append_scaled_reference(new, new, kc, kc, ks, ks, np.array([[1]]), [5])
    assert s[1, 0] == 1.0 and (k[1, :3] == 4.0).all() and (k[1, 3:5] == 448.0).all() and (k[1, 5:] == 0).all()
    # a page that starts with a new token forgets its old scale
    k, v, s, _ = append_scaled_reference(new[:, :1] * 0 + 1.0, new[:, :1], kc, kc, ks * 100, ks, np.array([[0, 1]]), [17])
    assert s[1, 0] == 2.0 ** -8 and (k[1, 0] == 256.0).all()


def test_attention_of_equal_scores_is_the_mean():
    q = np.zeros((1, 2, 4, 128))
    vc = np.zeros((1, 16, 1, 128))
    vc[0, :, 0, 0] = np.arange(16)
    out, lse, _ = attention_scaled_reference(q, vc, vc, np.ones((1, 1)), np.full((1, 1), 2.0), np.array([[0]]), [4])
    assert out[0, 1, 0, 0] == 2 * 1.5 and out[0, 0, 0, 0] == 2 * 1.0 and np.isclose(lse[0, 1, 0], np.log(4))
    scores, _ = weights_reference(q, vc, np.ones((1, 1)), np.array([[0]]), [4], lse, np.ones((1, 1, 16)))
    # tokens 0, 1 are older: 1 + 4 heads * (1/3 + 1/4); token 2 is seen by both rows, token 3 by the last
    assert np.allclose(scores[0, 0, :5], [1 + 7 / 3, 1 + 7 / 3, 7 / 3, 1.0, 1.0])


def test_evict_keeps_ends_and_best():
    kc = np.arange(2 * 16.0).reshape(2, 16, 1, 1) * np.ones(128)
    scores = np.zeros((2, 1, 16))
    scores[0, 0, [3, 5, 7]] = [1.0, np.nan, 1.0]
    k, v, s, _, _, lens, kept = evict_reference(kc, kc, scores, np.array([[0, 1]]), [20], 5, recent=2, sinks=1)
    assert kept[0, 0].tolist() == [0, 3, 7, 18, 19] and lens[0] == 5
    assert k[0, :5, 0, 0].tolist() == [0, 3, 7, 18, 19] and (k[0, 5:] == kc[0, 5:]).all()
    assert s[0, 0, :5].tolist() == [0, 1, 1, 0, 0]


# ------------------------------------------------------------------ refusals of the C ABI
@pytest.fixture(scope="module")
def lib():
    from small_q_attention_b200 import _native, build

    build.build()
    return _native.library()


def _args(**kw):
    from small_q_attention_b200._native import KV_FP8_E4M3, SqaArgs

    a = SqaArgs()
    a.query = a.key_cache = a.value_cache = a.block_tables = a.seq_lens = a.out = 256
    a.batch, a.q_len, a.num_q_heads, a.num_kv_heads = 4, 4, 32, 8
    a.head_dim, a.page_size, a.num_pages, a.max_pages, a.kv_dtype = 128, 16, 1024, 512, KV_FP8_E4M3
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _scales(key=256, value=256, stride=0):
    from small_q_attention_b200._native import SqaScales

    return SqaScales(key, value, stride)


@pytest.mark.parametrize("kw,code", [
    (dict(head_dim=64), 2), (dict(page_size=32), 2), (dict(num_q_heads=16), 2), (dict(q_len=17), 2), (dict(q_len=0), 1),
    (dict(kv_dtype=0), 1), (dict(kernel=2), 2), (dict(cluster=4), 2), (dict(batch=-1), 1), (dict(query=None), 1),
    (dict(key_cache=264), 1), (dict(out=None), 1), (dict(out_partial=256), 1), (dict(out_lse=258), 1),
    (dict(page_stride=24), 1), (dict(sm_scale=-1.0), 1),
])
def test_forward_scaled_refuses(lib, kw, code):
    assert lib.sqa_forward_scaled(ctypes.byref(_args(**kw)), ctypes.byref(_scales()), 256, 1 << 30, None) == code


def test_forward_scaled_refuses_scales_and_workspace(lib):
    a = _args()
    call = lambda s, ws=256, n=1 << 30: lib.sqa_forward_scaled(ctypes.byref(a), s, ws, n, None)  # noqa: E731
    assert call(None) == 1
    assert call(ctypes.byref(_scales(key=None))) == 1
    assert call(ctypes.byref(_scales(value=None))) == 1
    assert call(ctypes.byref(_scales(key=258))) == 1
    assert call(ctypes.byref(_scales(stride=4))) == 1
    assert call(ctypes.byref(_scales()), ws=None) in (1, 4)  # 4: no device to size the launch for
    assert lib.sqa_forward_scaled(None, ctypes.byref(_scales()), 256, 1 << 30, None) == 1


@pytest.mark.parametrize("kw,code", [(dict(query=None), 1), (dict(key_cache=264), 1), (dict(q_len=17), 2),
                                     (dict(kernel=1), 2), (dict(kv_dtype=0), 1), (dict(seq_lens=257), 1)])
def test_accumulate_refuses(lib, kw, code):
    a = _args(**kw)
    assert lib.sqa_accumulate_weights(ctypes.byref(a), 256, ctypes.byref(_scales()), 256, 256, None) == code


def test_accumulate_refuses_missing_arrays(lib):
    a = _args()
    s = ctypes.byref(_scales())
    assert lib.sqa_accumulate_weights(ctypes.byref(a), None, s, 256, 256, None) == 1
    assert lib.sqa_accumulate_weights(ctypes.byref(a), 256, s, None, 256, None) == 1
    assert lib.sqa_accumulate_weights(ctypes.byref(a), 256, s, 256, None, None) == 1  # no status word
    assert lib.sqa_accumulate_weights(ctypes.byref(a), 256, None, 256, 256, None) == 1  # e4m3 without scales
    assert lib.sqa_accumulate_weights(ctypes.byref(a), 256, s, 256, 258, None) == 1
    assert lib.sqa_accumulate_weights(None, 256, s, 256, 256, None) == 1


def _append_args(**kw):
    from small_q_attention_b200._native import KV_FP8_E4M3, SqaAppendArgs

    a = SqaAppendArgs()
    a.new_keys = a.new_values = a.key_cache = a.value_cache = a.block_tables = a.seq_lens = 256
    a.batch, a.q_len, a.num_kv_heads, a.head_dim, a.page_size = 2, 4, 8, 128, 16
    a.num_pages, a.max_pages, a.kv_dtype = 64, 32, KV_FP8_E4M3
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [(dict(head_dim=64), 2), (dict(q_len=0), 1), (dict(kv_dtype=0), 2),
                                     (dict(kv_layout=2), 2), (dict(page_stride=16), 1), (dict(new_keys=None), 1),
                                     (dict(key_cache=264), 1), (dict(status=258), 1), (dict(max_pages=1 << 27), 2)])
def test_append_scaled_refuses(lib, kw, code):
    assert lib.sqa_cache_append_scaled(ctypes.byref(_append_args(**kw)), ctypes.byref(_scales()), 0, None) == code


def test_append_scaled_refuses_scales_and_types(lib):
    a = ctypes.byref(_append_args())
    assert lib.sqa_cache_append_scaled(a, None, 0, None) == 1
    assert lib.sqa_cache_append_scaled(a, ctypes.byref(_scales(key=None)), 0, None) == 1
    assert lib.sqa_cache_append_scaled(a, ctypes.byref(_scales(stride=7)), 0, None) == 1
    assert lib.sqa_cache_append_scaled(a, ctypes.byref(_scales()), 2, None) == 2
    assert lib.sqa_cache_append_scaled(None, ctypes.byref(_scales()), 0, None) == 1


def _evict_args(**kw):
    from small_q_attention_b200._native import SqaEvictArgs

    a = SqaEvictArgs()
    a.key_cache = a.value_cache = a.scores = a.block_tables = a.seq_lens = 256
    a.new_lens = a.kept = 512
    a.batch, a.num_kv_heads, a.head_dim, a.page_size, a.num_pages, a.max_pages = 2, 8, 128, 16, 64, 32
    a.budget, a.recent, a.sinks = 100, 10, 4
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(head_dim=64), 2), (dict(page_size=8), 2), (dict(budget=0), 1), (dict(recent=97), 1), (dict(recent=-1), 1),
    (dict(sinks=-1), 1), (dict(kv_dtype=1), 1), (dict(kv_layout=3), 2), (dict(new_lens=256), 1), (dict(kept=None), 1),
    (dict(scores=258), 1), (dict(value_cache=264), 1), (dict(page_stride=12), 1), (dict(max_pages=1 << 27), 2),
])
def test_evict_refuses(lib, kw, code):
    assert lib.sqa_cache_evict(ctypes.byref(_evict_args(**kw)), None, None) == code


def test_evict_refuses_scales_of_a_16_bit_cache(lib):
    assert lib.sqa_cache_evict(ctypes.byref(_evict_args()), ctypes.byref(_scales()), None) == 1
    assert lib.sqa_cache_evict(ctypes.byref(_evict_args(kv_dtype=1)), ctypes.byref(_scales(key=None)), None) == 1
    assert lib.sqa_cache_evict(None, None, None) == 1


def test_empty_batches_need_no_gpu(lib):
    s = ctypes.byref(_scales())
    assert lib.sqa_cache_append_scaled(ctypes.byref(_append_args(batch=0)), s, 0, None) == 0
    assert lib.sqa_cache_evict(ctypes.byref(_evict_args(batch=0)), None, None) == 0
    assert lib.sqa_accumulate_weights(ctypes.byref(_args(batch=0)), 256, s, 256, 256, None) == 0


def test_struct_layouts_match_the_header(tmp_path):
    import shutil
    import subprocess
    from pathlib import Path

    from small_q_attention_b200._native import SqaEvictArgs, SqaScales

    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    both = ((SqaEvictArgs, "sqa_evict_args"), (SqaScales, "sqa_scales"))
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "small_q_attention.h"', "int main(void) {"]
    for cls, name in both:
        lines.append(f'  printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0; }"]) + "\n")
    subprocess.run([cc, "-I", str(Path(__file__).resolve().parents[1] / "include"), str(src), "-o", str(exe)], check=True)
    text = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    got = {(a, b): int(c) for a, b, c in (ln.split() for ln in text.splitlines())}
    for cls, name in both:
        assert got[(name, "size")] == ctypes.sizeof(cls)
        assert all(got[(name, f)] == getattr(cls, f).offset for f, _ in cls._fields_)


# ------------------------------------------------------------------ refusals of the Python layer
def test_cpu_tensors_are_refused_by_the_extension():
    from small_q_attention_b200 import _native, build

    build.build_torch_ext()
    ext = _native.torch_ext()
    f8 = torch.float8_e4m3fn
    q, kc = torch.zeros(1, 1, 4, 128, dtype=torch.float16), torch.zeros(2, 16, 1, 128).to(f8)
    s, bt, sl = torch.ones(2, 1), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    new = torch.zeros(1, 1, 1, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        ext.forward_scaled(q, kc, kc, s, s, bt, sl, 16, None, 0, None, None, False, None, 0, False, 0, 0.0, 1.0, 0)
    with pytest.raises(ValueError, match="CUDA"):
        ext.append_scaled(new, new, kc, kc, s, s, bt, sl, False, 0)
    with pytest.raises(ValueError, match="CUDA"):
        ext.accumulate_weights(q, kc, s, bt, sl, torch.zeros(1, 1, 4), torch.zeros(2, 1, 16), 16, None, 0, 0, False, 0, 0.0, 0)
    with pytest.raises(ValueError, match="CUDA"):
        ext.cache_evict(kc, kc, torch.zeros(2, 1, 16), bt, sl, 4, 0, 0, s, s, None, None, False, 0)


def test_no_cpu_fallback():
    if torch.cuda.is_available():
        pytest.skip("this host has a GPU")
    import small_q_attention_b200 as sqa

    for call in (lambda: sqa.small_q_attention_scaled(*[None] * 8), lambda: sqa.cache_append_scaled(*[None] * 8),
                 lambda: sqa.accumulate_attention_weights(*[None] * 7), lambda: sqa.cache_evict(*[None] * 6)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_the_scaled_operator_is_registered():
    from small_q_attention_b200 import _native, build

    build.build_torch_ext()
    _native.torch_ext()
    q = torch.empty(2, 4, 32, 128, dtype=torch.bfloat16, device="meta")
    k = torch.empty(64, 16, 8, 128, dtype=torch.float8_e4m3fn, device="meta")
    s, bt = torch.empty(64, 8, device="meta"), torch.empty(2, 32, dtype=torch.int32, device="meta")
    o, lse = torch.ops.sqa_b200.small_q_attention_scaled(q, k, k, s, s, bt, torch.empty(2, dtype=torch.int32, device="meta"), 16)
    assert o.shape == q.shape and o.dtype == torch.bfloat16 and lse.shape == (2, 4, 32) and lse.dtype == torch.float32
