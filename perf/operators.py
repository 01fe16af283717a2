"""Serving several requests at once: the operators of the paged 8-bit key/value cache, as measurable cases.

A request's prompt (image patches and instruction tokens) is attended once, packed with the prompts of the other
requests; its keys and values then live in pages of 16 to 128 tokens in 8 bits, and every later call (single
tokens, or an action suffix of a few dozen) attends to them through the request's row of the block table.

=========  ==================================  ==============================================================
kind       entry point                         ranges
=========  ==================================  ==============================================================
plan       ``kv_cache.kv_plan``                1..512 requests, 1..1200 new tokens each, pages of 16..128
write      ``kv_cache.kv_write``               1..64 requests, 1..1168 tokens each, head dims 64, 128, 256,
                                               keys and values in 16 or 32 bits, token-major or head-major
prompt     ``kv_cache.prompt_attention``       1..16 prompts, 1..8192 tokens, 1..32 heads in groups of 1..8,
                                               causal, causal behind a bidirectional prefix, or full
attention  ``kv_cache.kv_attention``           1..64 requests, 1..63 queries each over 1..131072 cached tokens
=========  ==================================  ==============================================================

The lengths of a case follow from its own values, so that ``work`` knows them; contents, page orders and scales
follow from the seed.

The cache (e4m3, a float32 scale for each page and key/value head):
    keys    [pages, kv heads, page, head dim]      values  [pages, kv heads, head dim, page]
    scale = 2^e, the smallest e >= -64 with max|x| <= 448 * 2^e over the page's tokens; appending to a page keeps
    the tokens before the first new one and never lowers its scale.
"""

import math
import os
import random
import sys

import torch

own = False

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlc-vla_amd"))

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
F8 = torch.float8_e4m3fn


def listed():
    return [
        # bookkeeping of one decode step of 16 requests: the smallest call, launch latency
        {"name": "plan_decode", "kind": "plan", "requests": 16, "past": 1168, "new": 1, "ragged": True, "page": 64},
        # admitting a burst of 256 prompts at once, 16-token pages
        {"name": "plan_prompts", "kind": "plan", "requests": 256, "past": 0, "new": 1168, "ragged": True, "page": 16},
        # one layer's float32 keys and fp16 values as prefill leaves them: three images and 200 prompt tokens
        {"name": "write_prefix", "kind": "write", "requests": 1, "past": 0, "new": 968, "ragged": False, "kv": 1,
         "hd": 256, "page": 64, "ktype": "f32", "vtype": "f16", "head_major": True},
        # one generated token for each of 64 requests: every page is half full
        {"name": "write_decode", "kind": "write", "requests": 64, "past": 4000, "new": 1, "ragged": True, "kv": 8,
         "hd": 128, "page": 16, "ktype": "bf16", "vtype": "bf16", "head_major": False},
        # 32 ragged prompts of a model with eight kv heads
        {"name": "write_prompts", "kind": "write", "requests": 32, "past": 0, "new": 1168, "ragged": True, "kv": 8,
         "hd": 128, "page": 32, "ktype": "f16", "vtype": "f16", "head_major": False},
        # a few short prompts of the 2-layer model: launch latency
        {"name": "prompt_small", "kind": "prompt", "requests": 5, "tokens": 63, "ragged": True, "heads": 2, "kv": 1,
         "hd": 64, "type": "f16", "mask": "causal"},
        # six requests of the pi0.5 prefix expert: image and prompt tokens see each other, generated text is causal
        {"name": "prompt_prefix", "kind": "prompt", "requests": 6, "tokens": 968, "ragged": True, "heads": 8, "kv": 1,
         "hd": 256, "type": "f16", "mask": "prefix"},
        # long documents, causal, four query heads on a kv head
        {"name": "prompt_long", "kind": "prompt", "requests": 2, "tokens": 8192, "ragged": True, "heads": 16, "kv": 4,
         "hd": 128, "type": "bf16", "mask": "causal"},
        # the next token of one request behind its prefix: latency
        {"name": "decode_one", "kind": "attention", "requests": 1, "cached": 969, "new": 1, "ragged": False,
         "heads": 8, "kv": 1, "hd": 256, "page": 64, "type": "f16", "causal": True},
        # the action suffixes of eight requests: 50 tokens each that see their whole prefix and one another
        {"name": "suffix_batch", "kind": "attention", "requests": 8, "cached": 1018, "new": 50, "ragged": True,
         "heads": 8, "kv": 1, "hd": 256, "page": 64, "type": "f16", "causal": False},
        # a decode step of 48 requests of a grouped-head model
        {"name": "decode_batch", "kind": "attention", "requests": 48, "cached": 4096, "new": 1, "ragged": True,
         "heads": 32, "kv": 8, "hd": 128, "page": 16, "type": "bf16", "causal": True},
        # one token each of two very long requests: the cache's length has to be split
        {"name": "decode_long", "kind": "attention", "requests": 2, "cached": 131072, "new": 1, "ragged": True,
         "heads": 8, "kv": 1, "hd": 256, "page": 64, "type": "bf16", "causal": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "write", "write", "prompt", "prompt", "attention", "attention", "attention"])
    page = rng.choice([16, 32, 64, 128])
    ragged = rng.random() < 0.8
    if kind == "plan":
        return {"kind": kind, "requests": _log_int(rng, 1, 256), "past": rng.choice([0, _log_int(rng, 1, 4000)]),
                "new": rng.choice([1, _log_int(rng, 1, 1168)]), "ragged": ragged, "page": page}
    if kind == "write":
        kt, vt = rng.choice([("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f32")])
        return {"kind": kind, "requests": _log_int(rng, 1, 32), "past": rng.choice([0, _log_int(rng, 1, 4000)]),
                "new": _log_int(rng, 1, 1168), "ragged": ragged, "kv": rng.choice([1, 1, 2, 3, 4]),
                "hd": rng.choice([64, 128, 256]), "page": page, "ktype": kt, "vtype": vt,
                "head_major": rng.random() < 0.3}
    kv, hd = rng.choice([1, 1, 2, 4]), rng.choice([64, 128, 256])
    heads = kv * rng.choice([1, 2, 4, 7, 8])
    if kind == "prompt":
        requests = _log_int(rng, 1, 16)
        most = int(math.sqrt(84e9 / (requests * heads * hd)))  # query-key pairs of the largest listed case
        return {"kind": kind, "requests": requests, "tokens": _log_int(rng, 1, min(8192, most)), "ragged": ragged,
                "heads": heads, "kv": kv, "hd": hd, "type": rng.choice(["f16", "bf16"]),
                "mask": rng.choice(["causal", "causal", "prefix", "full"])}
    requests = _log_int(rng, 1, 64)
    most = 48 * 4096 * 8 * 128 // (requests * kv * hd)
    new = rng.choice([1, 1, 1, _log_int(rng, 1, 63)])
    cached = _log_int(rng, new, max(new, min(131072, most, (1 << 28) // (requests * heads * new))))
    return {"kind": kind, "requests": requests, "cached": cached, "new": new, "ragged": ragged, "heads": heads,
            "kv": kv, "hd": hd, "page": page, "type": rng.choice(["f16", "bf16"]), "causal": rng.random() < 0.8}


# ---- lengths -------------------------------------------------------------------------------------------------


def _lens(case):
    """(past, new) tokens of each request, from the case's own values."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    n, kind = case["requests"], case["kind"]

    def spread(most, least):
        if not case["ragged"] or most <= least:
            return [most] * n
        v = [r.randint(max(least, most // 8), most) for _ in range(n)]
        v[r.randrange(n)] = most
        return v

    if kind == "prompt":
        return [0] * n, spread(case["tokens"], 1)
    if kind == "attention":
        new = [case["new"]] * n
        return [t - case["new"] for t in spread(case["cached"], case["new"])], new
    return (spread(case["past"], 0) if case["past"] else [0] * n), spread(case["new"], 1)


def _cdiv(a, b):
    return -(-a // b)


def _prefixes(case, new):
    """The bidirectional tokens of each prompt: five in six of them, at least one."""
    return [max(1, t * 5 // 6) for t in new]


# ---- inputs --------------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cu(new):
    cu = [0]
    for t in new:
        cu.append(cu[-1] + t)
    return cu


def _pages(case, seed, lens, spare):
    """A block table over `lens` tokens of each request, its pages in an order of their own, and the free pages."""
    page = case["page"]
    need = [_cdiv(t, page) for t in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    wide = _cdiv(max(p + q for p, q in zip(*_lens(case))), page) if case["kind"] != "prompt" else 1
    table = torch.full((len(lens), wide), -1, dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    return table.cuda(), order[at:].contiguous().cuda(), total


def _random(shape, dtype, g):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _cache(pages, kv, hd, page, g):
    """Pages as an earlier write left them: values over most of the format's range under each page's scale."""
    shape = ((pages, kv, page, hd), (pages, kv, hd, page))
    data = [(torch.randn(s, generator=g, device="cuda") * 96.0).clamp_(-448.0, 448.0).to(F8) for s in shape]
    scale = [torch.exp2(torch.randint(-8, -5, (pages, kv), generator=g, device="cuda").float()) for _ in range(2)]
    return data[0], scale[0], data[1], scale[1]


def prepare(case, seed):
    past, new = _lens(case)
    cu = _cu(new)
    tokens, g = cu[-1], _gen(seed)
    s = {"case": case, "cu": _ints(cu), "tokens": tokens}
    if case["kind"] == "prompt":
        dt, (h, kv, hd) = DTYPES[case["type"]], (case["heads"], case["kv"], case["hd"])
        s["q"], s["k"], s["v"] = (_random((tokens, n, hd), dt, g) for n in (h, kv, kv))
        s["bidir"] = _ints(_prefixes(case, new)) if case["mask"] == "prefix" else None
        s["longest"] = max(new)
        return s
    total = [p + q for p, q in zip(past, new)]
    s["past"], s["new"], s["kv_lens"] = _ints(past), _ints(new), _ints(total)
    if case["kind"] == "plan":
        extra = sum(_cdiv(t, case["page"]) for t in total) - sum(_cdiv(p, case["page"]) for p in past)
        s["table"], s["free"], s["pages"] = _pages(case, seed, past, extra + 7)
        return s
    kv, hd, page = case["kv"], case["hd"], case["page"]
    s["table"], _, s["pages"] = _pages(case, seed, total, 3)
    s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"] = _cache(s["pages"], kv, hd, page, g)
    if case["kind"] == "write":
        shape = (kv, tokens, hd) if case["head_major"] else (tokens, kv, hd)
        # keys and values of different heads and tokens differ in size, some far outside the others
        size = torch.exp2(torch.randn((tokens, kv, 1), generator=g, device="cuda"))
        size = size.transpose(0, 1) if case["head_major"] else size
        s["k"], s["v"] = ((torch.randn(shape, generator=g, device="cuda") * size).to(DTYPES[case[t]])
                          for t in ("ktype", "vtype"))
        if case["head_major"]:
            s["k"], s["v"] = s["k"].transpose(0, 1), s["v"].transpose(0, 1)
        slots = []
        table = s["table"].tolist()
        for b in range(len(new)):
            slots += [table[b][p // page] * page + p % page for p in range(past[b], past[b] + new[b])]
        s["slots"] = _ints(slots)
        return s
    s["q"] = _random((tokens, case["heads"], hd), DTYPES[case["type"]], g)
    s["longest"] = max(total)
    return s


# ---- one pass ------------------------------------------------------------------------------------------------


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        from mlc_vla import kv_cache as C

        if kind == "plan":
            p = C.kv_plan(s["past"], s["new"], s["table"], s["free"], num_pages=s["pages"], page_size=case["page"],
                          tokens=s["tokens"])
            return {"table": s["table"], "cu": p.cu_seqlens.torch, "kv_lens": p.kv_lens.torch,
                    "slots": p.slot_map.torch, "status": p.status.torch}
        if kind == "write":
            C.kv_write(s["k"], s["v"], s["cu"], s["slots"], s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"])
            return {n: s[n] for n in ("k_cache", "k_scale", "v_cache", "v_scale")}
        if kind == "prompt":
            return C.prompt_attention(s["q"], s["k"], s["v"], s["cu"], causal=case["mask"] != "full",
                                      bidir=s["bidir"]).torch
        return C.kv_attention(s["q"], s["cu"], s["kv_lens"], s["table"], s["k_cache"], s["k_scale"], s["v_cache"],
                              s["v_scale"], causal=case["causal"], max_kv=s["longest"]).torch
    return {"plan": _plan, "write": _write, "prompt": _prompt, "attention": _attention}[kind](s)


def _plan(s):
    page, table, free = s["case"]["page"], s["table"], s["free"].long()
    past, new = s["past"].long(), s["new"].long()
    wide = table.shape[1]
    cu = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0)])
    had, has = (past + page - 1) // page, (past + new + page - 1) // page
    fits = (has <= wide) & (cu[1:] <= s["tokens"])
    need = torch.where(fits, has - had, 0)
    end = need.cumsum(0)
    base = end - need
    granted = fits & ((need == 0) | (end <= free.numel()))
    col = torch.arange(wide, device="cuda")[None, :]
    fresh = granted[:, None] & (col >= had[:, None]) & (col < has[:, None])
    at = (base[:, None] + col - had[:, None]).clamp(0, max(0, free.numel() - 1))
    table.copy_(torch.where(fresh, free[at], table.long()).to(torch.int32))
    t = torch.arange(s["tokens"], device="cuda")
    b = (torch.searchsorted(cu, t, right=True) - 1).clamp(max=new.numel() - 1)
    pos = past[b] + t - cu[b]
    ids = table.long()[b, (pos // page).clamp(max=wide - 1)]
    slots = torch.where(granted[b] & (t < cu[-1]) & (ids >= 0), ids * page + pos % page, -1)
    status = torch.stack([torch.where(granted, need, 0).sum(), (~granted).sum()])
    return {"table": table, "cu": cu.to(torch.int32),
            "kv_lens": torch.where(granted, past + new, 0).to(torch.int32), "slots": slots.to(torch.int32),
            "status": status.to(torch.int32)}


def _scale_for(amax):
    """2^e with the smallest e >= -64 such that amax <= 448 * 2^e."""
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(amax > 0, e, -64).clamp(min=-64)
    return torch.exp2(e.float())


def _write_one(x, cu, slots, cache, scale, page):
    """x [tokens, kv, hd] into cache [pages, kv, page, hd] (a view of either cache) under scale [pages, kv]."""
    x = x.float()
    pages, kv = scale.shape
    ids, off = slots.long() // page, slots.long() % page
    amax = torch.zeros((pages, kv), device="cuda").index_reduce_(0, ids, x.abs().amax(-1), "amax")
    first = slots.long()[cu[:-1].long()]  # only the first page of a request can hold tokens that are kept
    kept = torch.zeros(pages, dtype=torch.long, device="cuda").index_put_((first // page,), first % page)
    need = _scale_for(amax)
    touched = torch.zeros(pages, dtype=torch.bool, device="cuda").index_fill_(0, ids, True)[:, None]
    now = torch.where(touched, torch.where(kept[:, None] > 0, torch.maximum(scale, need), need), scale)
    head = first // page
    old = cache.view(torch.uint8)[head].view(F8).float() * scale[head][..., None, None]
    again = (old / now[head][..., None, None]).to(F8).view(torch.uint8)
    stay = (torch.arange(page, device="cuda")[None, :] < kept[head][:, None])[:, None, :, None]
    raw = cache.view(torch.uint8)
    raw[head] = torch.where(stay, again, raw[head])
    raw[ids, :, off] = (x / now[ids][..., None]).clamp(-448.0, 448.0).to(F8).view(torch.uint8)
    scale.copy_(now)


def _write(s):
    page, cu, slots = s["case"]["page"], s["cu"], s["slots"]
    _write_one(s["k"], cu, slots, s["k_cache"], s["k_scale"], page)
    _write_one(s["v"], cu, slots, s["v_cache"].transpose(2, 3), s["v_scale"], page)
    return {n: s[n] for n in ("k_cache", "k_scale", "v_cache", "v_scale")}


def _softmax_products(q, k, v, see):
    """q [B, n, H, d], k and v [B, KV, L, d] in float32, see [B, n, L]: softmax(q k / sqrt(d)) v over what each
    row sees; a row that sees nothing is zero."""
    b, n, h, d = q.shape
    kv = k.shape[1]
    q = q.reshape(b, n, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(b, kv, h // kv * n, d) / math.sqrt(d)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()).view(b, kv, h // kv, n, -1)
    x = x.masked_fill_(~see[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
    total = x.sum(-1, keepdim=True)
    out = torch.matmul(x.view(b, kv, h // kv * n, -1), v).view(b, kv, h // kv, n, d) / total.clamp(min=1e-30)
    return out.permute(0, 3, 1, 2, 4).reshape(b, n, h, d)


def _rows(cu, longest, tokens):
    """[B, longest] token of each padded row, and which of them there are."""
    cu = cu.long()
    i = torch.arange(longest, device="cuda")[None, :]
    return (cu[:-1, None] + i).clamp(max=tokens - 1), i < (cu[1:] - cu[:-1])[:, None]


def _unpad(x, cu, tokens, dtype):
    t = torch.arange(tokens, device="cuda")
    b = torch.searchsorted(cu.long(), t, right=True) - 1
    return x[b, t - cu.long()[b]].to(dtype)


def _prompt(s):
    at, there = _rows(s["cu"], s["longest"], s["tokens"])
    q, k, v = s["q"][at].float(), s["k"][at].float().transpose(1, 2), s["v"][at].float().transpose(1, 2).contiguous()
    i = torch.arange(s["longest"], device="cuda")
    if s["case"]["mask"] == "full":
        see = there[:, None, :].expand(-1, s["longest"], -1)
    else:
        last = i[None, :].expand(at.shape[0], -1) + 1
        if s["bidir"] is not None:
            last = torch.maximum(last, s["bidir"].long()[:, None])
        see = (i[None, None, :] < last[:, :, None]) & there[:, None, :]
    return _unpad(_softmax_products(q, k, v, see), s["cu"], s["tokens"], s["q"].dtype)


def _attention(s):
    case, table = s["case"], s["table"].long().clamp(min=0)
    b, wide = table.shape
    kv, hd, page, n = case["kv"], case["hd"], case["page"], case["new"]
    k = s["k_cache"].view(torch.uint8)[table].view(F8).float() * s["k_scale"][table][..., None, None]
    v = s["v_cache"].view(torch.uint8)[table].view(F8).float() * s["v_scale"][table][..., None, None]
    k = k.transpose(1, 2).reshape(b, kv, wide * page, hd)
    v = v.permute(0, 2, 1, 4, 3).reshape(b, kv, wide * page, hd)
    at, _ = _rows(s["cu"], n, s["tokens"])
    total = s["kv_lens"].long()[:, None]
    last = total - n + 1 + torch.arange(n, device="cuda")[None, :] if case["causal"] else total.expand(-1, n)
    j = torch.arange(wide * page, device="cuda")
    see = j[None, None, :] < last[:, :, None]
    # what lies behind a request's last token is not its own
    v = torch.where((j[None, :] < total)[:, None, :, None], v, 0.0)
    return _unpad(_softmax_products(s["q"][at].float(), k, v, see), s["cu"], s["tokens"], s["q"].dtype)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------


def _attend64(q, k, v, limit):
    """One request: q [n, H, d], k and v [L, KV, d], limit [n] keys that each row sees."""
    n, h, d = q.shape
    out = torch.zeros((n, h, d), dtype=torch.float64, device="cuda")
    hidden = torch.arange(k.shape[0], device="cuda")[None, :] >= limit[:, None]
    for i in range(h):
        j = i // (h // k.shape[1])
        x = (q[:, i].double() @ k[:, j].double().t()) * d ** -0.5
        x[hidden] = -math.inf
        out[:, i] = torch.softmax(x, -1) @ v[:, j].double()
    return out


def _e4m3(x):
    """The nearest value of the 8-bit format (4 exponent bits, 3 mantissa bits), ties to the even one."""
    x = x.clamp(-448.0, 448.0)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3.0)
    return torch.round(x / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    past, new = _lens(case)
    if case["kind"] == "plan":
        return None
    cu = _cu(new)
    if case["kind"] == "prompt":
        full = [max(t, 0) if case["mask"] == "full" else (p if case["mask"] == "prefix" else 0)
                for t, p in zip(new, _prefixes(case, new))]
        out = []
        for a, z, f in zip(cu, cu[1:], full):
            out.append(_attend64(s["q"][a:z], s["k"][a:z], s["v"][a:z],
                                 (torch.arange(z - a, device="cuda") + 1).clamp(min=f)))
        return torch.cat(out)
    page, table = case["page"], s["table"].tolist()
    if case["kind"] == "attention":
        out = []
        for b, (a, z) in enumerate(zip(cu, cu[1:])):
            total = past[b] + new[b]
            ids = torch.tensor(table[b][:_cdiv(total, page)], device="cuda")
            k = (s["k_cache"].double()[ids] * s["k_scale"].double()[ids][..., None, None]).permute(0, 2, 1, 3)
            v = (s["v_cache"].double()[ids] * s["v_scale"].double()[ids][..., None, None]).permute(0, 3, 1, 2)
            k, v = (x.reshape(-1, case["kv"], case["hd"])[:total] for x in (k, v))
            limit = torch.arange(past[b], total, device="cuda") + 1
            out.append(_attend64(s["q"][a:z], k, v, limit if case["causal"] else torch.full_like(limit, total)))
        return torch.cat(out)
    got = {}
    for name in ("k", "v"):
        x = s[name].double()
        data = s[name + "_cache"].double()
        data = data if name == "k" else data.transpose(2, 3)
        scale = s[name + "_scale"].double()
        for b in range(len(new)):
            at = past[b]
            while at < past[b] + new[b]:
                to = min(past[b] + new[b], (at // page + 1) * page)
                i, o, keep = table[b][at // page], at % page, at % page
                part = x[cu[b] + at - past[b]:cu[b] + to - past[b]].transpose(0, 1)  # [kv, tokens, hd]
                amax = part.abs().amax((1, 2))
                want = torch.exp2(torch.ceil(torch.log2(amax.clamp(min=2.0 ** -80) / 448.0)).clamp(min=-64.0))
                now = torch.maximum(want, scale[i]) if keep else want
                if keep:
                    data[i, :, :keep] = _e4m3(data[i, :, :keep] * (scale[i] / now)[:, None, None])
                data[i, :, o:o + to - at] = _e4m3(part / now[:, None, None])
                scale[i] = now
                at = to
        got[name + "_cache"] = data if name == "k" else data.transpose(2, 3).contiguous()
        got[name + "_scale"] = scale
    return got


# ---- work ----------------------------------------------------------------------------------------------------


def work(case):
    """Bytes and operations of one pass: each input read once, each output written once."""
    past, new = _lens(case)
    tokens = sum(new)
    if case["kind"] == "plan":
        pages = sum(_cdiv(p + t, case["page"]) for p, t in zip(past, new))
        return {"bytes": 4 * (5 * len(new) + 2 * pages + tokens), "flops": 0}
    size = {"f16": 2, "bf16": 2, "f32": 4}
    kv, hd = case["kv"], case["hd"]
    if case["kind"] == "write":
        page = case["page"]
        touched = sum(_cdiv(p + t, page) - p // page for p, t in zip(past, new))
        return {"bytes": tokens * kv * hd * (size[case["ktype"]] + size[case["vtype"]] + 2) + touched * kv * 16
                + tokens * 4, "flops": 0}
    heads = case["heads"]
    if case["kind"] == "prompt":
        if case["mask"] == "full":
            pairs = sum(t * t for t in new)
        elif case["mask"] == "causal":
            pairs = sum(t * (t + 1) // 2 for t in new)
        else:
            pairs = sum(p * p + (t * (t + 1) - p * (p + 1)) // 2 for t, p in zip(new, _prefixes(case, new)))
        return {"bytes": 2 * tokens * hd * 2 * (heads + kv), "flops": 4 * pairs * heads * hd}
    pairs = sum((p * t + t * (t + 1) // 2) if case["causal"] else (p + t) * t for p, t in zip(past, new))
    pages = sum(_cdiv(p + t, case["page"]) for p, t in zip(past, new))
    return {"bytes": sum(p + t for p, t in zip(past, new)) * 2 * kv * hd + pages * (kv * 8 + 4)
            + 4 * tokens * heads * hd, "flops": 4 * pairs * heads * hd}
