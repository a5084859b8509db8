"""CPU oracle for the block-scaled e4m3 cache and for eviction (test infrastructure only).

Restates in 64 bits, token by token, what ``include/small_q_attention.h`` says of
``sqa_cache_append_scaled``, ``sqa_forward_scaled``, ``sqa_accumulate_weights`` and
``sqa_cache_evict``.  Caches are numpy float64 arrays of stored values ``[P, 16, Hkv, 128]``
(the e4m3 numbers of a scaled cache, without their scales) and scales ``[P, Hkv]``.
"""

from __future__ import annotations

import math

import numpy as np

__all__ = ["append_scaled_reference", "attention_scaled_reference", "evict_reference", "page_scale", "round_e4m3",
           "weights_reference"]

PAGE, GROUP = 16, 4


def page_scale(amax: float) -> float:
    """The smallest power of two with amax <= 448 * scale, 2^-100 at least."""
    e = -100
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def round_e4m3(x):
    """Nearest e4m3 value, ties to even, saturating; NaN stays NaN."""
    x = np.asarray(x, np.float64)
    big = np.abs(np.nan_to_num(x, nan=0.0, posinf=448.0, neginf=-448.0))
    exponent = np.maximum(np.frexp(big)[1] - 1, -6)
    step = np.exp2(exponent - 3.0)
    with np.errstate(invalid="ignore"):
        r = np.clip(np.rint(np.clip(x, -1e6, 1e6) / step) * step, -448, 448)
    return np.where(np.isnan(x), np.nan, r)


def _amax(x):
    x = np.abs(np.asarray(x, np.float64))
    return float(np.max(np.where(np.isfinite(x), x, 0.0), initial=0.0))


def append_scaled_reference(new_k, new_v, kc, vc, ks, vs, table, lens):
    """Copies of (kc, vc, ks, vs) with the new tokens in them; bad sequences and pages skipped."""
    out = [np.array(x, np.float64) for x in (kc, vc, ks, vs)]
    batch, q_len, hkv = new_k.shape[:3]
    for b in range(batch):
        n = int(lens[b])
        if n < q_len or (n + PAGE - 1) // PAGE > table.shape[1]:
            continue
        for first in range((n - q_len) // PAGE * PAGE, n, PAGE):
            page = int(table[b, first // PAGE])
            if not 0 <= page < kc.shape[0]:
                continue
            n0, n1 = max(n - q_len - first, 0), min(n - first, PAGE)
            rows = slice(first + n0 - (n - q_len), first + n1 - (n - q_len))
            for new, cache, scales in ((new_k, out[0], out[2]), (new_v, out[1], out[3])):
                for h in range(hkv):
                    x = np.asarray(new[b, rows, h], np.float64)
                    scale, was = page_scale(_amax(x)), scales[page, h]
                    if n0:
                        scale = max(scale, was)
                        if scale > was:
                            cache[page, :n0, h] = round_e4m3(cache[page, :n0, h] * was / scale)
                    cache[page, n0:n1, h] = round_e4m3(x / scale)
                    scales[page, h] = scale
    return out


def _row_tokens(cache, scales, table, b, h, n):
    t = np.arange(n)
    pages = np.asarray(table[b])[t // PAGE]
    x = np.asarray(cache, np.float64)[pages, t % PAGE, h]
    return x if scales is None else x * np.asarray(scales, np.float64)[pages, h][:, None]


def attention_scaled_reference(q, kc, vc, ks, vs, table, lens, *, mask_lens=None, sm_scale=None, out_scale=1.0):
    """(out, lse, spread): spread = {"abs": sum p |v|, "top": max p * max |v|, "dot": max over seen
    tokens of sm_scale * sum |q k|}, what the error bounds of a test are made of."""
    q = np.asarray(q, np.float64)
    batch, q_len, hq, dim = q.shape
    sm_scale = dim ** -0.5 if sm_scale is None else sm_scale
    out, lse = np.zeros(q.shape), np.full(q.shape[:3], -np.inf)
    spread = {"abs": np.zeros(q.shape), "top": np.zeros(q.shape[:3]), "dot": np.zeros(q.shape[:3])}
    for b in range(batch):
        n = min(int(lens[b]), PAGE * np.asarray(table).shape[1])
        whole = int(mask_lens[b]) if mask_lens is not None else int(lens[b])
        for h in range(hq // GROUP):
            k, v = _row_tokens(kc, ks, table, b, h, n), _row_tokens(vc, vs, table, b, h, n)
            for qi in range(q_len):
                seen = min(n, whole - q_len + qi + 1)
                if seen <= 0:
                    continue
                rows = q[b, qi, h * GROUP:(h + 1) * GROUP]
                x = rows @ k[:seen].T * sm_scale  # [4, seen]
                m = x.max(axis=1, keepdims=True)
                p = np.exp(x - m)
                total = p.sum(axis=1, keepdims=True)
                at = (b, qi, slice(h * GROUP, (h + 1) * GROUP))
                out[at] = p @ v[:seen] / total * out_scale
                lse[at] = (m + np.log(total))[:, 0]
                spread["abs"][at] = p @ np.abs(v[:seen]) / total * abs(out_scale)
                spread["top"][at] = np.max(p / total * np.abs(v[:seen]).max(axis=1), axis=1) * abs(out_scale)
                spread["dot"][at] = (np.abs(rows) @ np.abs(k[:seen]).T).max(axis=1) * sm_scale
    return out, lse, spread


def weights_reference(q, kc, ks, table, lens, lse, scores, *, mask_lens=None, sm_scale=None):
    """(scores after the step, largest sm_scale * sum |q k|)."""
    q, scores = np.asarray(q, np.float64), np.array(scores, np.float64)
    batch, q_len, hq, dim = q.shape
    sm_scale = dim ** -0.5 if sm_scale is None else sm_scale
    dot = 0.0
    for b in range(batch):
        n = min(int(lens[b]), PAGE * np.asarray(table).shape[1])
        whole = int(mask_lens[b]) if mask_lens is not None else int(lens[b])
        for h in range(hq // GROUP):
            k = _row_tokens(kc, ks, table, b, h, n)
            w = np.zeros(n)
            for qi in range(q_len):
                seen = min(n, whole - q_len + qi + 1)
                if seen <= 0:
                    continue
                for g in range(h * GROUP, (h + 1) * GROUP):
                    if lse[b, qi, g] == -np.inf:
                        continue
                    w[:seen] += np.exp(k[:seen] @ q[b, qi, g] * sm_scale - float(lse[b, qi, g]))
                    dot = max(dot, float((np.abs(k[:seen]) @ np.abs(q[b, qi, g])).max()) * sm_scale)
            for t in range(n):
                page = int(table[b, t // PAGE])
                old = scores[page, h, t % PAGE]
                scores[page, h, t % PAGE] = w[t] if t >= whole - q_len else old + w[t]
    return scores, dot


def _key(x):
    return -math.inf if math.isnan(x) else x


def evict_reference(kc, vc, scores, table, lens, budget, *, recent=0, sinks=0, ks=None, vs=None):
    """(kc, vc, scores, ks, vs, new_lens, kept) after the eviction; caches of any element type."""
    kc, vc, scores = kc.copy(), vc.copy(), scores.copy()
    ks, vs = (None, None) if ks is None else (ks.copy(), vs.copy())
    batch, hkv = len(lens), kc.shape[2]
    kept_all = np.full((batch, hkv, budget), -1, np.int32)
    new_lens = np.array(lens, np.int32)
    for b in range(batch):
        n = int(lens[b])
        pages = [int(x) for x in table[b, : (n + PAGE - 1) // PAGE]] if n > 0 else []
        if n < 0 or (n + PAGE - 1) // PAGE > table.shape[1]:
            continue
        if n <= budget:
            kept_all[b, :, :n] = np.arange(n)
            continue
        if any(not 0 <= x < kc.shape[0] for x in pages):
            continue
        new_lens[b] = budget
        for h in range(hkv):
            score = [float(scores[pages[t // PAGE], h, t % PAGE]) for t in range(n)]
            middle = sorted(range(sinks, n - recent), key=lambda t: (-_key(score[t]), t))
            kept = sorted(list(range(sinks)) + middle[: budget - sinks - recent] + list(range(n - recent, n)))
            kept_all[b, h] = kept
            for cache, scales in ((kc, ks), (vc, vs)):
                rows = [cache[pages[t // PAGE], t % PAGE, h].copy() for t in kept]
                if scales is not None:
                    rows = [r * scales[pages[t // PAGE], h] for r, t in zip(rows, kept)]
                    for first in range(0, budget, PAGE):
                        part = slice(first, min(first + PAGE, budget))
                        s = page_scale(_amax(np.stack(rows[part])))
                        rows[part] = list(round_e4m3(np.stack(rows[part]) / s))
                        scales[pages[first // PAGE], h] = s
                for i, r in enumerate(rows):
                    cache[pages[i // PAGE], i % PAGE, h] = r
            for i, t in enumerate(kept):
                scores[pages[i // PAGE], h, i % PAGE] = score[t]
    return kc, vc, scores, ks, vs, new_lens, kept_all
