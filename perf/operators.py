"""Measured cases of the block-scaled 8-bit cache and of eviction by attention weight.

Four operators over the paged KV cache (pages of 16 tokens, head_dim 128, 4 query heads per KV head):

* ``append``      quantise new K/V into an e4m3 cache with one scale per page and KV head
* ``attend``      causal paged MTP attention over that cache
* ``accumulate``  add each cached token's attention weight to its score
* ``evict``       keep the tokens of the highest scores within a budget, compacted in place

``run`` computes them in plain torch where ``own`` is false and through ``small_q_attention_b200``
where it is true; ``exact`` restates them in 64 bits.
"""

import math

import torch

own = False

PAGE, DIM, GROUP = 16, 128, 4
F8 = torch.float8_e4m3fn
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases
def _case(name, kind, batch, q_len, kv, dtype, hkv=8, layout="NHD", ragged=False, scaled=True, budget=0, recent=0,
          sinks=0):
    return {"name": name, "kind": kind, "batch": batch, "q_len": q_len, "kv": kv, "dtype": dtype, "hkv": hkv,
            "layout": layout, "ragged": ragged, "scaled": scaled, "budget": budget, "recent": recent, "sinks": sinks}


def listed():
    return [
        # one user, no drafts, a short context: the smallest call, where latency counts
        _case("attend 1x1x600", "attend", 1, 1, 600, "fp16"),
        # four users with four tokens in flight at 8K (the repository's cfg2)
        _case("attend 4x4x8192", "attend", 4, 4, 8192, "bf16"),
        # a busy server: many users of very different lengths, heads before tokens in a page
        _case("attend 48x3x8190 ragged", "attend", 48, 3, 8190, "fp16", layout="HND", ragged=True),
        # one user with a very long context and the widest draft (cfg5)
        _case("attend 1x16x262144", "attend", 1, 16, 262144, "fp16"),
        # the throughput configuration (cfg3): the largest call
        _case("attend 16x8x32768", "attend", 16, 8, 32768, "bf16"),
        # a decode step's append: a few tokens of each user into partly filled pages
        _case("append 16x4 at 4099", "append", 16, 4, 4099, "bf16"),
        # a prompt's append: thousands of tokens at once, the last page ragged
        _case("append 2x5003 prompt", "append", 2, 5003, 5003, "fp16", layout="HND"),
        # the weights of one token's step over a short 16-bit cache
        _case("accumulate 1x1x1000", "accumulate", 1, 1, 1000, "bf16", scaled=False),
        # cfg2's step over its 16-bit cache
        _case("accumulate 4x4x8192", "accumulate", 4, 4, 8192, "fp16", scaled=False),
        # cfg3's step over the 8-bit cache
        _case("accumulate 16x8x32768 e4m3", "accumulate", 16, 8, 32768, "bf16"),
        # prompts of 8K cut to a quarter before decoding starts
        _case("evict 4x8192 to 2048", "evict", 4, 1, 8192, "bf16", scaled=False, budget=2048, recent=256, sinks=4),
        # a busy server's 8-bit caches of very different lengths, some already short enough
        _case("evict 32x7001 to 1500 e4m3", "evict", 32, 1, 7001, "fp16", ragged=True, budget=1500, recent=500,
              sinks=1),
    ]


def draw(rng):
    kind = rng.choice(["attend", "attend", "append", "accumulate", "evict"])

    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    batch, hkv = spread(1, 64), rng.choice([1, 2, 4, 8])
    q_len = rng.randint(1, 16)
    room = 16 * 32768 * 8 // (batch * hkv)  # no more tokens x heads than the largest listed case
    if kind == "append" and rng.random() < 0.5:
        q_len = spread(1, min(8192, max(2, room // 64)))
        kv = q_len + rng.choice([0, rng.randint(0, 300)])
    else:
        kv = max(q_len, spread(1, min(65536, room // (2 if kind == "attend" and q_len > 8 else 1))))
    c = _case("", kind, batch, q_len, kv, rng.choice(["fp16", "bf16"]), hkv=hkv, layout=rng.choice(["NHD", "HND"]),
              ragged=rng.random() < 0.5, scaled=kind in ("attend", "append") or rng.random() < 0.5)
    if kind == "evict":
        c["budget"] = spread(1, max(2, kv))
        c["sinks"] = rng.randint(0, min(4, c["budget"]))
        c["recent"] = rng.randint(0, c["budget"] - c["sinks"])
        c["q_len"] = 1
    del c["name"]
    return c


def _lens(case):
    """Every sequence kv tokens long, or from kv down to an eighth of it (never under q_len)."""
    b, kv, q = case["batch"], case["kv"], case["q_len"]
    if not case["ragged"]:
        return [kv] * b
    return [max(q, kv - (kv - kv // 8) * i // max(1, b - 1)) for i in range(b)]


def _element(case):
    return 1 if case["scaled"] else 2


def work(case):
    lens, hkv, q = _lens(case), case["hkv"], case["q_len"]
    tokens, pages = sum(lens), sum((n + PAGE - 1) // PAGE for n in lens)
    rows, meta = case["batch"] * q * GROUP * hkv, 4 * pages + 4 * case["batch"]
    e = _element(case)
    if case["kind"] == "attend":
        return {"bytes": tokens * hkv * 2 * DIM + pages * hkv * 8 + 2 * rows * DIM * 2 + 4 * rows + meta,
                "flops": 4.0 * DIM * tokens * hkv * GROUP * q}
    if case["kind"] == "accumulate":
        return {"bytes": tokens * hkv * (DIM * e + 8) + pages * hkv * (4 if e == 1 else 0) + rows * (2 * DIM + 4) + meta,
                "flops": 2.0 * DIM * tokens * hkv * GROUP * q}
    if case["kind"] == "append":
        new, old, touched = case["batch"] * q, 0, 0
        for n in lens:
            old += (n - q) % PAGE
            touched += (n - 1) // PAGE - (n - q) // PAGE + 1
        return {"bytes": 2 * hkv * (new * DIM * 3 + old * DIM * 2 + touched * 8) + 4 * touched + 4 * case["batch"],
                "flops": 4.0 * DIM * hkv * (new + old)}
    moved = sum(case["budget"] for n in lens if n > case["budget"])
    read = sum(n for n in lens if n > case["budget"])
    return {"bytes": hkv * (4 * read + moved * (2 * (2 * DIM * e + 4) + 4)) + meta + 4 * case["batch"], "flops": float(hkv * read)}


# ------------------------------------------------------------------ inputs
def _pages(case, gen):
    """Distinct pages for every sequence, drawn from a pool a little larger than what they need."""
    b, width = case["batch"], (case["kv"] + PAGE - 1) // PAGE
    pool = b * width + 3
    return torch.randperm(pool, generator=gen, device="cuda")[: b * width].to(torch.int32).view(b, width), pool


def _amax(x):
    """Largest finite magnitude of each page and head of [P, 16, H, 128]."""
    return x.abs().amax(dim=(1, 3)).float()


def _values(case, pool, gen, spread):
    """[P, 16, H, 128] 16-bit values: pages of different magnitude, one token in a hundred four times as large."""
    x = torch.randn(pool, PAGE, case["hkv"], DIM, generator=gen, device="cuda", dtype=TYPES[case["dtype"]])
    x *= torch.exp(spread * torch.randn(pool, 1, case["hkv"], 1, generator=gen, device="cuda")).to(x.dtype)
    x[torch.rand(pool, PAGE, generator=gen, device="cuda") < 0.01] *= 4
    return x


def _paged(x, case):
    """The cache layout of [P, 16, H, 128]."""
    return x.permute(0, 2, 1, 3).contiguous() if case["layout"] == "HND" else x


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    tables, pool = _pages(case, gen)
    lens = _lens(case)
    s = {"case": case, "tables": tables, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
         "max_len": max(lens), "min_len": min(lens)}
    hkv, q, kind, b = case["hkv"], case["q_len"], case["kind"], case["batch"]
    for side in ("k", "v"):
        x = _values(case, pool, gen, 0.3)
        if case["scaled"]:
            amax = _amax(x)
            # attention takes any scale; the append and the eviction keep powers of two
            scale = amax / 448 if kind in ("attend", "accumulate") else torch.exp2(torch.ceil(torch.log2(amax / 448)))
            s[side + "s"] = scale
            x = (x.float() / scale[:, None, :, None]).clamp_(-448, 448).to(F8)
        s[side + "c"] = _paged(x, case)
    if kind in ("attend", "accumulate"):
        s["q"] = (1.5 * torch.randn(b, q, hkv * GROUP, DIM, generator=gen, device="cuda")).to(TYPES[case["dtype"]])
    if kind == "append":
        s["new"] = [torch.randn(b, q, hkv, DIM, generator=gen, device="cuda").to(TYPES[case["dtype"]])
                    * torch.exp(torch.randn(b, q, 1, 1, generator=gen, device="cuda")).to(TYPES[case["dtype"]])
                    for _ in range(2)]
    if kind in ("accumulate", "evict"):
        s["scores"] = torch.rand(pool, hkv, PAGE, generator=gen, device="cuda").pow_(8)
    if kind == "accumulate":  # what the step's attention returned
        s["lse"] = torch.stack([_row_logits(s, i).logsumexp(dim=-1) for i in range(b)])
        s["lse"] = s["lse"].float().permute(0, 2, 1, 3).reshape(b, q, hkv * GROUP).contiguous()
    return s


def _row_logits(s, i):
    """[H, q, 4, len] logits of sequence i, fp32, -inf where a row does not see a token."""
    case, q = s["case"], s["case"]["q_len"]
    n = int(_lens(case)[i])
    k = _gather(s, "k", s["tables"][i:i + 1])[0, :, :n]
    query = s["q"][i].float().view(q, case["hkv"], GROUP, DIM).permute(1, 0, 2, 3)
    x = torch.einsum("hqgd,htd->hqgt", query, k) * DIM ** -0.5
    unseen = torch.arange(n, device="cuda")[None, :] >= n - q + 1 + torch.arange(q, device="cuda")[:, None]
    return x.masked_fill(unseen[None, :, None, :], -math.inf)


# ------------------------------------------------------------------ plain forms
def _nhd(x, case):
    return x.transpose(1, 2) if case["layout"] == "HND" else x


def _gather(s, side, tables):
    """[B, H, width * 16, 128] fp32 values of the tables' pages."""
    case, at = s["case"], tables.long()
    x = _nhd(s[side + "c"], case)[at].float()  # [B, width, 16, H, 128]
    if case["scaled"]:
        x = x * s[side + "s"][at][:, :, None, :, None]
    return x.permute(0, 3, 1, 2, 4).reshape(at.shape[0], case["hkv"], -1, DIM)


def _logits(s):
    """[B, H, q, 4, T] logits and which of them a row sees."""
    case, q = s["case"], s["case"]["q_len"]
    k = _gather(s, "k", s["tables"])
    query = s["q"].float().view(-1, q, case["hkv"], GROUP, DIM).permute(0, 2, 1, 3, 4)
    x = torch.matmul(query.reshape(*query.shape[:2], q * GROUP, DIM), k.transpose(2, 3)) * DIM ** -0.5
    t = torch.arange(k.shape[2], device=k.device)
    limit = s["lens"].view(-1, 1) - q + 1 + torch.arange(q, device=k.device)  # [B, q]
    seen = t < limit[:, :, None]  # [B, q, T]
    x = x.view(*x.shape[:2], q, GROUP, -1)
    return x.masked_fill(~seen[:, None, :, None, :], -math.inf)


def _attend(s):
    case, q = s["case"], s["case"]["q_len"]
    x = _logits(s)
    m = x.amax(dim=-1, keepdim=True)
    p = torch.exp(x - m)
    total = p.sum(dim=-1, keepdim=True)
    v = _gather(s, "v", s["tables"])
    t = torch.arange(v.shape[2], device=v.device)
    v = v.masked_fill((t >= s["lens"].view(-1, 1))[:, None, :, None], 0.0)
    o = torch.matmul(p.flatten(2, 3), v).view(*p.shape[:4], DIM) / total
    o = o.permute(0, 2, 1, 3, 4).reshape(case["batch"], q, -1, DIM)
    lse = (m + torch.log(total)).squeeze(-1).permute(0, 2, 1, 3).reshape(case["batch"], q, -1)
    return {"out": o.to(s["q"].dtype), "lse": lse.contiguous()}


def _accumulate(s):
    case, q = s["case"], s["case"]["q_len"]
    lse = s["lse"].view(-1, q, case["hkv"], GROUP).permute(0, 2, 1, 3)[..., None]
    w = torch.exp(_logits(s) - lse).sum(dim=(2, 3))  # [B, H, T]
    width, at = s["tables"].shape[1], s["tables"].long()
    w = w.view(-1, case["hkv"], width, PAGE).transpose(1, 2)  # [B, width, H, 16]
    t = torch.arange(width * PAGE, device=w.device).view(1, width, 1, PAGE)
    n = s["lens"].view(-1, 1, 1, 1)
    old = s["scores"][at]
    s["scores"][at] = torch.where(t >= n, old, torch.where(t >= n - q, w, old + w))
    return {"scores": s["scores"]}


def _power_scale(amax):
    """The smallest power of two that brings amax within 448, 2^-100 at least."""
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, mantissa in [0.5, 1); 448 = 0.875 * 2^9
    exponent = (exponent - 9 + (mantissa > 0.875).int()).clamp(min=-100)
    return torch.ldexp(torch.ones_like(amax), exponent.masked_fill(amax == 0, -100))


def _to_e4m3(x):
    return x.clamp(-448.0, 448.0).to(F8)


def _append(s):
    case, q, b = s["case"], s["case"]["q_len"], s["case"]["batch"]
    n = s["lens"].long()
    first, count = (n - q) // PAGE, (q + PAGE - 2) // PAGE + 1  # first touched page, touched pages at most
    page = first[:, None] + torch.arange(count, device=n.device)  # [B, count]
    used = page * PAGE < n[:, None]
    at = s["tables"].long().gather(1, page.clamp(max=s["tables"].shape[1] - 1))
    t = page[:, :, None] * PAGE + torch.arange(PAGE, device=n.device)  # [B, count, 16]
    new = (t >= n[:, None, None] - q) & (t < n[:, None, None])
    old = t < n[:, None, None] - q
    qi = (t - (n - q)[:, None, None]).clamp(0, q - 1)
    for side, x in zip("kv", s["new"]):
        cache = _nhd(s[side + "c"], case)
        scales = s[side + "s"]
        x = x.float()[torch.arange(b, device=n.device)[:, None, None], qi]  # [B, count, 16, H, 128]
        need = _power_scale(x.abs().masked_fill(~new[..., None, None], 0.0).amax(dim=(2, 4)))  # [B, count, H]
        was = scales[at]
        scale = torch.where(old.any(dim=2)[:, :, None], torch.maximum(was, need), need)
        had = cache[at]
        kept = torch.where((scale > was)[:, :, None, :, None],
                           _to_e4m3(had.float() * was[:, :, None, :, None] / scale[:, :, None, :, None]).float(), had.float())
        held = torch.where(new[..., None, None], _to_e4m3(x / scale[:, :, None, :, None]).float(),
                           torch.where(old[..., None, None], kept, had.float()))
        cache.view(torch.uint8)[at[used]] = held[used].to(F8).view(torch.uint8)
        scales[at[used]] = scale[used]
    return {"k": s["kc"], "v": s["vc"], "ks": s["ks"], "vs": s["vs"]}


def _evict(s):
    case, hkv, b = s["case"], s["case"]["hkv"], s["case"]["batch"]
    budget, recent, sinks = case["budget"], case["recent"], case["sinks"]
    at, n = s["tables"].long(), s["lens"].view(-1, 1, 1)
    width = at.shape[1]
    t = torch.arange(width * PAGE, device=n.device)
    score = s["scores"][at].permute(0, 2, 1, 3).reshape(b, hkv, -1)
    score = torch.where((t < sinks) | (t >= n - recent), math.inf, score).masked_fill(t >= n, -math.inf)
    cut = min(budget, width * PAGE)
    kept = score.sort(dim=-1, descending=True, stable=True).indices[..., :cut].sort(dim=-1).values  # [B, H, cut]
    kept = torch.where(n > budget, kept, t[:cut])
    goes = (n > budget).expand(b, hkv, cut)
    lanes = (torch.arange(b, device=n.device)[:, None, None], torch.arange(hkv, device=n.device)[None, :, None])
    page, slot, head = at[lanes[0], kept // PAGE], kept % PAGE, lanes[1].expand(b, hkv, cut)
    to_page = at[lanes[0], t[:cut] // PAGE].expand(b, hkv, cut)
    to_slot = (t[:cut] % PAGE).expand(b, hkv, cut)
    target = (to_page[goes], to_slot[goes], head[goes])
    for side in "kv":
        cache = _nhd(s[side + "c"], case)
        x = cache.view(torch.uint8 if case["scaled"] else torch.int16)[page, slot, head]  # [B, H, cut, 128]
        if case["scaled"]:
            scales = s[side + "s"]
            x = x.view(F8).float() * scales[page, head][..., None]
            groups = torch.nn.functional.pad(x, (0, 0, 0, -cut % PAGE)).view(b, hkv, -1, PAGE, DIM)
            scale = _power_scale(groups.abs().amax(dim=(3, 4)))  # [B, H, pages]
            x = _to_e4m3(x / scale.repeat_interleave(PAGE, dim=2)[:, :, :cut, None]).view(torch.uint8)
            first = goes[..., ::PAGE]
            scales[to_page[..., ::PAGE][first], head[..., ::PAGE][first]] = scale[first]
        cache.view(x.dtype)[target] = x[goes]
    moved = s["scores"][page, head, slot]
    s["scores"][to_page[goes], head[goes], to_slot[goes]] = moved[goes]
    kept = torch.where(t[:cut] < n, kept, -1).int()
    kept = torch.nn.functional.pad(kept, (0, budget - cut), value=-1)
    out = {"lens": s["lens"].clamp(max=budget), "kept": kept, "scores": s["scores"]}
    return out | _held(s)


def _held(s):
    """The caches and, where there are some, their scales."""
    return {"k": s["kc"], "v": s["vc"], **({"ks": s["ks"], "vs": s["vs"]} if s["case"]["scaled"] else {})}


def _own(s):
    import small_q_attention_b200 as sqa

    case = s["case"]
    if case["kind"] == "attend":
        out, lse = sqa.small_q_attention_scaled(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["tables"], s["lens"], PAGE,
                                                s["max_len"], min_seq_len=s["min_len"], kv_layout=case["layout"],
                                                return_lse=True)
        return {"out": out, "lse": lse}
    if case["kind"] == "accumulate":
        sqa.accumulate_attention_weights(s["q"], s["kc"], s["tables"], s["lens"], s["lse"], s["scores"], PAGE,
                                         s["max_len"], key_scales=s.get("ks"), kv_layout=case["layout"])
        return {"scores": s["scores"]}
    if case["kind"] == "append":
        sqa.cache_append_scaled(*s["new"], s["kc"], s["vc"], s["ks"], s["vs"], s["tables"], s["lens"],
                                kv_layout=case["layout"])
        return {"k": s["kc"], "v": s["vc"], "ks": s["ks"], "vs": s["vs"]}
    lens, kept = sqa.cache_evict(s["kc"], s["vc"], s["scores"], s["tables"], s["lens"], case["budget"],
                                 recent=case["recent"], sinks=case["sinks"], key_scales=s.get("ks"),
                                 value_scales=s.get("vs"), kv_layout=case["layout"])
    return {"lens": lens, "kept": kept, "scores": s["scores"], **_held(s)}


def run(state):
    if own:
        return _own(state)
    return {"attend": _attend, "accumulate": _accumulate, "append": _append, "evict": _evict}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ the definition, in 64 bits
def _round_e4m3(x):
    """e4m3 with round to nearest even: 3 bits behind the leading one, no exponent under -6, 448 at most."""
    exponent = torch.frexp(x)[1] - 1
    step = torch.exp2(exponent.clamp(min=-6).double() - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_scale(amax):
    e = torch.ceil(torch.log2(amax / 448))
    e = torch.where(amax > 448 * torch.exp2(e), e + 1, e)  # log2 may be off beside a power of two
    e = torch.where(amax <= 448 * torch.exp2(e - 1), e - 1, e)
    return torch.exp2(e.clamp(min=-100))


def _sequence(s, side, i, n):
    """[n, H, 128] values of sequence i in 64 bits, its places (page, slot) and its stored values."""
    t = torch.arange(n, device="cuda")
    page, slot = s["tables"][i].long()[t // PAGE], t % PAGE
    cache = s[side + "c"]
    held = (cache[page, :, slot] if s["case"]["layout"] == "HND" else cache[page, slot]).double()
    scale = s[side + "s"][page].double()[..., None] if s["case"]["scaled"] else 1.0
    return held * scale, page, slot, held


def exact(case, seed):
    s = prepare(case, seed)
    lens, q, hkv, kind = _lens(case), case["q_len"], case["hkv"], case["kind"]
    if kind in ("attend", "accumulate"):
        out, lses, scores = [], [], s["scores"].double() if "scores" in s else None
        for i, n in enumerate(lens):
            k, page, slot, _ = _sequence(s, "k", i, n)
            v = _sequence(s, "v", i, n)[0] if kind == "attend" else None
            rows, row_lse = [], []
            weight = torch.zeros(n, hkv, dtype=torch.float64, device="cuda")
            for j in range(q):
                m = n - q + j + 1  # tokens that draft j sees
                for g in range(GROUP):
                    x = torch.einsum("hd,thd->th", s["q"][i, j, g::GROUP].double(), k[:m]) / math.sqrt(DIM)
                    if kind == "attend":
                        rows.append(torch.einsum("th,thd->hd", torch.softmax(x, dim=0), v[:m]))
                        row_lse.append(torch.logsumexp(x, dim=0))
                    else:
                        weight[:m] += torch.exp(x - s["lse"][i, j, g::GROUP].double())
            if kind == "attend":
                # [q, 4, H, ...] -> [q, H * 4, ...]
                out.append(torch.stack(rows).view(q, GROUP, hkv, DIM).transpose(1, 2).reshape(q, -1, DIM))
                lses.append(torch.stack(row_lse).view(q, GROUP, hkv).transpose(1, 2).reshape(q, -1))
            else:
                before = scores[page, :, slot]
                before[n - q:] = 0
                scores[page, :, slot] = before + weight
        return {"out": torch.stack(out), "lse": torch.stack(lses)} if kind == "attend" else {"scores": scores}
    if kind == "append":
        return _exact_append(s, lens, q)
    return _exact_evict(s, lens)


def _store(cache, layout, page, slot, x):
    if layout == "HND":
        cache[page, :, slot] = x
    else:
        cache[page, slot] = x


def _exact_append(s, lens, q):
    got = {"k": s["kc"].double(), "v": s["vc"].double(), "ks": s["ks"].double(), "vs": s["vs"].double()}
    for side, new in zip("kv", s["new"]):
        cache, scales = got[side], got[side + "s"]
        for i, n in enumerate(lens):
            begin = (n - q) // PAGE * PAGE  # the first touched page's first token
            _, page, slot, held = _sequence(s, side, i, n)
            page, slot, held = page[begin:], slot[begin:], held[begin:]
            old = n - q - begin  # tokens of the first page that were there
            pages = page[::PAGE]
            x = torch.zeros(len(pages) * PAGE, s["case"]["hkv"], DIM, dtype=torch.float64, device="cuda")
            x[old:n - begin] = new[i].double()
            scale = _exact_scale(x.view(len(pages), PAGE, -1, DIM).abs().amax(dim=(1, 3)))
            was = scales[pages[0]].clone()
            if old:
                scale[0] = torch.maximum(scale[0], was)
            x = x[: n - begin] / scale.repeat_interleave(PAGE, dim=0)[: n - begin, :, None]
            x[:old] = held[:old] * (was / scale[0])[None, :, None]
            _store(cache, s["case"]["layout"], page, slot, _round_e4m3(x))
            scales[pages] = scale
    return got


def _exact_evict(s, lens):
    case = s["case"]
    budget, recent, sinks, hkv = case["budget"], case["recent"], case["sinks"], case["hkv"]
    got = {side: s[side + "c"].double() for side in "kv"}
    if case["scaled"]:
        got |= {side + "s": s[side + "s"].double() for side in "kv"}
    got["scores"] = s["scores"].double()
    kept_all = torch.full((len(lens), hkv, budget), -1, dtype=torch.int32, device="cuda")
    for i, n in enumerate(lens):
        if n <= budget:
            kept_all[i, :, :n] = torch.arange(n, dtype=torch.int32, device="cuda")
            continue
        values = {side: _sequence(s, side, i, n) for side in "kv"}
        page, slot = values["k"][1:3]
        score = s["scores"][page, :, slot].double()  # [n, H]
        middle = torch.arange(sinks, n - recent, device="cuda")
        best = torch.argsort(-score[middle], dim=0, stable=True)[: budget - sinks - recent]
        ends = torch.cat([torch.arange(sinks, device="cuda"), torch.arange(n - recent, n, device="cuda")])
        kept = torch.cat([middle[best], ends[:, None].expand(-1, hkv)]).sort(dim=0).values  # [budget, H]
        kept_all[i] = kept.T.int()
        got["scores"][page[:budget], :, slot[:budget]] = score.gather(0, kept)
        for side in "kv":
            x = values[side][0].gather(0, kept[..., None].expand(-1, -1, DIM))
            if case["scaled"]:
                pages = page[:budget:PAGE]
                scale = torch.stack([_exact_scale(part.abs().amax(dim=(0, 2))) for part in x.split(PAGE)])
                x = _round_e4m3(x / scale.repeat_interleave(PAGE, dim=0)[:budget, :, None])
                got[side + "s"][pages] = scale
            _store(got[side], case["layout"], page[:budget], slot[:budget], x)
    return {"lens": None, "kept": None} | got
