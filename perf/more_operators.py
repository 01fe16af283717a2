"""Generating text for several requests: what a decode step needs around the attention over the paged 8-bit cache,
as measurable cases.

Before the attention, the new tokens' queries and keys are normalised and turned to their positions.  After the last
layer, the logits become log probabilities: of given tokens (scores), of the best alternatives (beams), with the
entropy.  Between steps the cache's pages change hands: beams and samples fork from a request, finished requests' pages
become free, a pool is made dense before it shrinks, or is copied into a larger one.

=========  =================================  ===============================================================
kind       entry point                        ranges
=========  =================================  ===============================================================
rope       ``kv_cache.qk_rope``               1..256 requests, 1..8192 tokens each, positions up to 140000, 1..32
                                              heads, head dims 64, 128, 256, partly rotated ones, 16 and 32 bits
logprobs   ``logits.token_logprobs``          1..1024 rows of 32..257152 logits, up to 64 alternatives, masked ones
copy       ``kv_cache.kv_copy``               1..4096 pages of up to 18 layers, into the same pool or another
fork       ``kv_cache.kv_fork``               1..64 requests into 1..512, pages of 16..128 tokens
compact    ``kv_cache.kv_compact``            1..256 requests on pages anywhere in the pool
free       ``kv_cache.kv_free``               1..512 requests, some sharing pages, pools of up to 262144 pages
=========  =================================  ===============================================================

The lengths of a case follow from its own values, so that ``work`` knows them; contents and page orders follow from the
seed.

The cache (e4m3, a float32 scale for each page and key/value head), of all layers:
    keys    [layers, pages, kv heads, page, head dim]      values  [layers, pages, kv heads, head dim, page]
"""

import math
import os
import random
import sys

import torch

own = False

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlc-vla_amd"))

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZES = {"f16": 2, "bf16": 2, "f32": 4}
F8 = torch.float8_e4m3fn
VOCAB = 257152  # of the language model whose embedding table the framework holds


def listed():
    return [
        # the next token of 16 requests, rotation only, as the prefix expert has it: latency
        {"name": "rope_decode", "kind": "rope", "requests": 16, "past": 1168, "new": 1, "ragged": True, "heads": 8,
         "kv": 1, "hd": 256, "rotary": 256, "type": "f16", "norm": False, "theta": 10000.0, "fused": True},
        # chunks of eight long documents, normalised heads in groups of four, out of one projection of q, k and v
        {"name": "rope_long", "kind": "rope", "requests": 8, "past": 131072, "new": 4096, "ragged": True, "heads": 32,
         "kv": 8, "hd": 128, "rotary": 128, "type": "bf16", "norm": True, "theta": 1000000.0, "fused": True},
        # a decode step of 16 requests over the whole vocabulary, with 20 alternatives
        {"name": "logprobs_decode", "kind": "logprobs", "rows": 16, "vocab": VOCAB, "pad": 0, "given": 1, "top": 20,
         "type": "bf16", "scale": 1.0, "masked": 0.0},
        # scores of a prompt's 1001 tokens, with the five best of each
        {"name": "logprobs_prompt", "kind": "logprobs", "rows": 1001, "vocab": VOCAB, "pad": 0, "given": 1, "top": 5,
         "type": "bf16", "scale": 1.0, "masked": 0.0},
        # a few pages of a shared prefix put aside, 18 layers
        {"name": "copy_few", "kind": "copy", "count": 5, "pages": 64, "into": 0, "page": 64, "kv": 1, "hd": 256,
         "layers": 18},
        # a pool moved into a larger one
        {"name": "copy_pool", "kind": "copy", "count": 4001, "pages": 4096, "into": 6144, "page": 16, "kv": 8,
         "hd": 128, "layers": 2},
        # four beams of each of four requests
        {"name": "fork_beams", "kind": "fork", "requests": 4, "children": 16, "len": 1168, "ragged": True, "page": 64,
         "kv": 1, "hd": 256, "layers": 18},
        # eight samples of each of 64 prompts
        {"name": "fork_samples", "kind": "fork", "requests": 64, "children": 512, "len": 1168, "ragged": True,
         "page": 64, "kv": 1, "hd": 256, "layers": 6},
        # a small pool after half of its requests have ended
        {"name": "compact_small", "kind": "compact", "requests": 16, "len": 300, "ragged": True, "page": 16,
         "pages": 512, "kv": 1, "hd": 256, "layers": 2},
        # a large one, grouped heads
        {"name": "compact_large", "kind": "compact", "requests": 48, "len": 4096, "ragged": True, "page": 16,
         "pages": 12000, "kv": 8, "hd": 128, "layers": 1},
        # the free list of one decode step's pool
        {"name": "free_small", "kind": "free", "requests": 16, "len": 1168, "ragged": True, "page": 64,
         "pages": 1024},
        # 512 requests on small pages of the largest pool
        {"name": "free_large", "kind": "free", "requests": 512, "len": 4096, "ragged": True, "page": 16,
         "pages": 262144},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "rope", "logprobs", "logprobs", "logprobs", "copy", "fork", "compact", "free"])
    ragged = rng.random() < 0.8
    if kind == "rope":
        kv, hd = rng.choice([1, 1, 2, 4, 8]), rng.choice([64, 128, 256])
        heads = kv * rng.choice([1, 2, 4, 7, 8]) if kv < 8 else 32
        requests = _log_int(rng, 1, 256)
        most = 8 * 4096 * 40 * 128 // (requests * (heads + kv) * hd)
        typ = rng.choice(["f16", "bf16", "bf16", "f32"])
        new = rng.choice([1, _log_int(rng, 1, max(1, min(8192, most // (2 if typ == "f32" else 1))))])
        return {"kind": kind, "requests": requests, "past": rng.choice([0, _log_int(rng, 1, 131072)]), "new": new,
                "ragged": ragged, "heads": heads, "kv": kv, "hd": hd,
                "rotary": rng.choice([hd, hd, hd // 2, hd - 16]), "type": typ, "norm": rng.random() < 0.5,
                "theta": rng.choice([10000.0, 500000.0, 1000000.0]), "fused": rng.random() < 0.7}
    if kind == "logprobs":
        vocab = rng.choice([VOCAB, _log_int(rng, 32, VOCAB)])
        typ = rng.choice(["f16", "bf16", "f32"])
        rows = _log_int(rng, 1, max(1, min(1001, 1001 * VOCAB // vocab) // (2 if typ == "f32" else 1)))
        return {"kind": kind, "rows": rows, "vocab": vocab, "pad": rng.choice([0, 0, rng.randint(1, 63)]),
                "given": rng.choice([1, 1, 0, rng.randint(2, 5)]),
                "top": min(vocab, rng.choice([0, 1, 5, 20, rng.randint(2, 64)])), "type": typ,
                "scale": rng.choice([1.0, 1.0, 0.5, 1.25]), "masked": rng.choice([0.0, 0.0, 0.5, 0.999])}
    page, kv, hd = rng.choice([16, 32, 64, 128]), rng.choice([1, 1, 2, 4, 8]), rng.choice([64, 128, 256])
    layers = rng.choice([1, 2, 6, 18])
    each = 2 * layers * page * kv * hd
    if kind == "copy":
        count = _log_int(rng, 1, max(1, min(4096, 2 ** 28 // each)))
        return {"kind": kind, "count": count, "pages": 2 * count + 3,
                "into": rng.choice([0, count + rng.randint(0, 64)]), "page": page, "kv": kv, "hd": hd,
                "layers": layers}
    if kind == "free":
        requests, length = _log_int(rng, 1, 512), _log_int(rng, 1, 4096)
        most = requests * _cdiv(length, page) + 5
        return {"kind": kind, "requests": requests, "len": length, "ragged": ragged, "page": page,
                "pages": max(most, _log_int(rng, 64, 262144))}
    length = _log_int(rng, 1, 4096)
    room = 3 * 2 ** 27 // each  # pages of a pool
    if kind == "fork":
        requests = _log_int(rng, 1, max(1, min(64, room // (_cdiv(length, page) + 8))))
        children = _log_int(rng, 1, max(1, min(512, 2 ** 28 // each, room)))
        return {"kind": kind, "requests": requests, "children": children, "len": length, "ragged": ragged,
                "page": page, "kv": kv, "hd": hd, "layers": layers}
    requests = _log_int(rng, 1, max(1, min(256, room // (2 * _cdiv(length, page)))))
    pages = int(requests * _cdiv(length, page) * rng.uniform(1.05, 2.0)) + 2
    return {"kind": kind, "requests": requests, "len": length, "ragged": ragged, "page": page, "pages": pages,
            "kv": kv, "hd": hd, "layers": layers}


# ---- lengths -------------------------------------------------------------------------------------------------


def _cdiv(a, b):
    return -(-a // b)


def _spread(case, most, least, n):
    if not case["ragged"] or most <= least:
        return [most] * n
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")) + str(most))
    v = [r.randint(max(least, most // 8), most) for _ in range(n)]
    v[r.randrange(n)] = most
    return v


def _rope_lens(case):
    n = case["requests"]
    return (_spread(case, case["past"], 0, n) if case["past"] else [0] * n), _spread(case, case["new"], 1, n)


def _holdings(case):
    """(length, pages, pages shared with the request before) of each request."""
    lens = _spread(case, case["len"], 1, case["requests"])
    need = [_cdiv(t, case["page"]) for t in lens]
    shared = [0] * len(lens)
    if case["kind"] in ("free", "compact"):  # every fourth and the one before it are forks of one prompt
        for b in range(3, len(lens), 4):
            shared[b] = min(need[b], need[b - 1]) // 2
    return lens, need, shared


def _parents(case):
    """Which request each row of the new table continues: every one at least once where there are enough rows."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    n, c = case["requests"], case["children"]
    v = [i % n for i in range(c)] if not case["ragged"] else [r.randrange(n) for _ in range(c)]
    r.shuffle(v)
    return v


def _forked(case):
    """How many rows of the new table need a page of their own, from the lengths."""
    lens, seen, got = _holdings(case)[0], set(), 0
    for p in _parents(case):
        got += p in seen and lens[p] % case["page"] != 0
        seen.add(p)
    return got


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


def _cache(case, pages, g):
    """Pages as earlier writes left them: finite codes under scales of each page and head."""
    layers, kv, hd, page = case["layers"], case["kv"], case["hd"], case["page"]
    data = []
    for _ in range(2):
        x = torch.randint(0, 256, (layers, pages, kv, page * hd), dtype=torch.uint8, generator=g, device="cuda")
        data.append(torch.where((x & 127) == 127, x - 1, x))
    scale = [torch.exp2(torch.randint(-8, -5, (layers, pages, kv), generator=g, device="cuda").float())
             for _ in range(2)]
    return {"k": data[0].view(layers, pages, kv, page, hd).view(F8), "k_scale": scale[0],
            "v": data[1].view(layers, pages, kv, hd, page).view(F8), "v_scale": scale[1]}


def _table(case, order):
    """A block table whose requests take their pages from `order` in turn."""
    lens, need, shared = _holdings(case)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, (n, s) in enumerate(zip(need, shared)):
        if s:
            table[b, :s] = table[b - 1, :s]
        table[b, s:n] = order[at:at + n - s]
        at += n - s
    return table.cuda(), _ints(lens)


def prepare(case, seed):
    g, cpu = _gen(seed), torch.Generator().manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "rope":
        past, new = _rope_lens(case)
        cu = _cu(new)
        s["cu"], s["kv_lens"] = _ints(cu), _ints([p + t for p, t in zip(past, new)])
        t, h, kv, hd, dt = cu[-1], case["heads"], case["kv"], case["hd"], DTYPES[case["type"]]
        if case["fused"]:
            x = torch.randn((t, h + 2 * kv, hd), generator=g, device="cuda").to(dt)
            s["q"], s["k"] = x[:, :h], x[:, h:h + kv]
        else:
            s["q"], s["k"] = (torch.randn((t, n, hd), generator=g, device="cuda").to(dt) for n in (h, kv))
        s["q_weight"], s["k_weight"] = ((0.2 * torch.randn(hd, generator=g, device="cuda")).to(dt) if case["norm"]
                                        else None for _ in range(2))
        return s
    if case["kind"] == "logprobs":
        rows, vocab, dt = case["rows"], case["vocab"], DTYPES[case["type"]]
        whole = torch.empty((rows, vocab + case["pad"]), dtype=dt, device="cuda")
        for a in range(0, rows, 64):  # a piece at a time, as float32 of all rows would be large
            z = min(rows, a + 64)
            x = 2.5 * torch.randn((z - a, vocab + case["pad"]), generator=g, device="cuda")
            # a few likely continuations of each row
            best = torch.randint(0, vocab, (z - a, 8), generator=g, device="cuda")
            x.scatter_add_(1, best, 9.0 + 3.0 * torch.randn(best.shape, generator=g, device="cuda"))
            whole[a:z] = x
        s["logits"] = whole[:, :vocab]
        if case["masked"]:  # a grammar that allows some tokens
            hidden = torch.rand(vocab, generator=g, device="cuda") < case["masked"]
            s["logits"].masked_fill_(hidden[None, :], -math.inf)
        s["tokens"] = None
        if case["given"]:
            shape = (rows, case["given"]) if case["given"] > 1 else (rows,)
            ids = torch.randint(0, vocab, shape, generator=g, device="cuda", dtype=torch.int32)
            s["tokens"] = torch.where(torch.rand(shape, generator=g, device="cuda") < 0.05, -1, ids)  # padding
        return s
    if case["kind"] == "copy":
        n, pages = case["count"], case["pages"]
        s["cache"] = _cache(case, pages, g)
        s["into"] = _cache(case, case["into"], g) if case["into"] else s["cache"]
        order = torch.randperm(pages, generator=cpu).to(torch.int32)
        s["src"] = order[:n].cuda()
        s["dst"] = (torch.randperm(case["into"], generator=cpu).to(torch.int32)[:n] if case["into"]
                    else order[n:2 * n]).cuda()
        return s
    lens, need, shared = _holdings(case)
    live = sum(need) - sum(shared)
    if case["kind"] == "fork":
        spare = case["children"] + 7
        order = torch.randperm(live + spare, generator=cpu).to(torch.int32)
        s["table"], s["lens"] = _table(case, order)
        s["parents"] = _ints(_parents(case))
        s["free"] = torch.cat([order[live:].sort().values, torch.full((live,), -1, dtype=torch.int32)]).cuda()
        s["count"] = _ints([spare])
        s["cache"] = _cache(case, live + spare, g)
        return s
    pages = case["pages"]
    if case["kind"] == "free":
        order = torch.randperm(pages, generator=cpu).to(torch.int32)
        s["table"], s["lens"] = _table(case, order)
        return s
    # of the pages in use, as many lie behind the first `live` of the pool as a random order would put there
    far = _moved(case)
    low = torch.randperm(live, generator=cpu)[:live - far]
    high = live + torch.randperm(pages - live, generator=cpu)[:far]
    order = torch.cat([low, high])[torch.randperm(live, generator=cpu)].to(torch.int32)
    s["table"], s["lens"] = _table(case, order)
    s["cache"] = _cache(case, pages, g)
    return s


def _moved(case):
    _, need, shared = _holdings(case)
    live = sum(need) - sum(shared)
    return live * (case["pages"] - live) // case["pages"]


# ---- one pass ------------------------------------------------------------------------------------------------


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        from mlc_vla import kv_cache as C
        from mlc_vla import logits as L

        if kind == "rope":
            q, k = C.qk_rope(s["q"], s["k"], s["cu"], s["kv_lens"], theta=case["theta"], rotary_dim=case["rotary"],
                             norm=case["norm"], q_weight=s["q_weight"], k_weight=s["k_weight"])
            return {"q": q.torch, "k": k.torch}
        if kind == "logprobs":
            r = L.token_logprobs(s["logits"], s["tokens"], top=case["top"], scale=case["scale"])
            return {n: t.torch for n, t in zip(r._fields, r) if t is not None}
        cache = [s["cache"][n] for n in ("k", "k_scale", "v", "v_scale")] if "cache" in s else None
        if kind == "copy":
            C.kv_copy(s["src"], s["dst"], *cache, into=[s["into"][n] for n in ("k", "k_scale", "v", "v_scale")])
            return dict(s["into"])
        if kind == "fork":
            r = C.kv_fork(s["parents"], s["table"], s["lens"], s["free"], *cache, free_count=s["count"])
            return {"table": r.block_table.torch, "lens": r.kv_lens.torch, "status": r.status.torch, **s["cache"]}
        if kind == "compact":
            r = C.kv_compact(s["table"], s["lens"], *cache)
            return {"table": r.block_table.torch, "status": r.status.torch, **s["cache"]}
        r = C.kv_free(s["table"], s["lens"], num_pages=case["pages"], page_size=case["page"])
        return {"free": r.free_pages.torch, "count": r.free_count.torch}
    return {"rope": _rope, "logprobs": _logprobs, "copy": _copy, "fork": _fork, "compact": _compact,
            "free": _free}[kind](s)


def _turns(s, tokens, dtype):
    """cos and sin [tokens, rotary / 2] of the packed tokens' angles, which need 64 bits at far positions."""
    case, cu = s["case"], s["cu"].long()
    t = torch.arange(tokens, device="cuda")
    b = torch.searchsorted(cu, t, right=True) - 1
    pos = s["kv_lens"].long()[b] - cu[b + 1] + t
    half = torch.arange(case["rotary"] // 2, device="cuda", dtype=torch.float64)
    angle = pos.double()[:, None] * case["theta"] ** (-2.0 * half / case["rotary"])
    return torch.cos(angle).to(dtype)[:, None, :], torch.sin(angle).to(dtype)[:, None, :]


def _rope(s):
    case = s["case"]
    cos, sin = _turns(s, s["q"].shape[0], torch.float32)
    rd, got = case["rotary"], {}
    for n in ("q", "k"):
        x = s[n].float()
        if case["norm"]:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (1.0 + s[n + "_weight"].float())
        a, b = x[..., :rd // 2], x[..., rd // 2:rd]
        got[n] = torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rd:]], -1).to(s[n].dtype)
    return got


def _logprobs(s):
    case = s["case"]
    x = s["logits"].float() * case["scale"]
    top = x.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, torch.zeros_like(top))
    y = x - top
    e = torch.exp(y)
    total = e.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    none = total == 0  # nothing is allowed
    got = {}
    if s["tokens"] is not None:
        ids = s["tokens"].long().view(case["rows"], -1)
        there = (ids >= 0) & (ids < case["vocab"])
        lp = torch.where(none, -math.inf, x.gather(1, ids.clamp(0, case["vocab"] - 1)) - lse)
        got["logprobs"] = torch.where(there, lp, 0.0).view(s["tokens"].shape)
    less = torch.where(e > 0, y * e, 0.0).sum(-1, keepdim=True)
    got["entropy"] = torch.where(none, 0.0, torch.log(total) - less / total)[:, 0]
    if case["top"]:
        # equal logits rank by their index: order the values as integers, the index below them
        bits = (s["logits"].float() + 0.0).view(torch.int32).long()
        key = torch.where(bits >= 0, bits, -(bits & 0x7fffffff) - 1)
        key = (key << 32) + (case["vocab"] - 1 - torch.arange(case["vocab"], device="cuda"))
        best = case["vocab"] - 1 - (torch.topk(key, case["top"], -1).values & 0xffffffff)
        got["top_ids"] = best.to(torch.int32)
        got["top_logprobs"] = torch.where(none, -math.inf, x.gather(1, best) - lse)
    return got


def _copy_pages(src, dst, cache, into):
    for n, x in cache.items():
        raw, to = (t.view(torch.uint8) if t.dtype == F8 else t for t in (x, into[n]))
        to[:, dst] = raw[:, src]


def _copy(s):
    _copy_pages(s["src"].long(), s["dst"].long(), s["cache"], s["into"])
    return dict(s["into"])


def _fork(s):
    page, table, lens, p = s["case"]["page"], s["table"], s["lens"].long(), s["parents"].long()
    n, wide = p.numel(), table.shape[1]
    i = torch.arange(n, device="cuda")
    there = (p >= 0) & (p < lens.numel())
    p = p.clamp(0, lens.numel() - 1)
    mine = torch.where(there, lens[p], 0)
    first = torch.full((lens.numel(),), n, device="cuda").scatter_reduce_(0, p, torch.where(there, i, n), "amin")
    need = (mine % page != 0) & (i != first[p])
    end = need.long().cumsum(0)
    ok = ~need | (end <= s["count"].long())
    fresh = s["free"].long()[(end - 1).clamp(0, s["free"].numel() - 1)]
    pages = torch.where(ok, _cdiv(mine, page), 0)[:, None]
    col = torch.arange(wide, device="cuda")[None, :]
    new = torch.where(col < pages, table[p].long(), -1)
    new = torch.where((need & ok)[:, None] & (col == pages - 1), fresh[:, None], new)
    at = (need & ok).nonzero()[:, 0]
    _copy_pages(table.long()[p[at], _cdiv(mine, page)[at] - 1], fresh[at], s["cache"], s["cache"])
    return {"table": new.to(torch.int32), "lens": torch.where(ok, mine, 0).to(torch.int32),
            "status": torch.stack([(need & ok).sum(), (~ok).sum()]).to(torch.int32), **s["cache"]}


def _used(s, pages):
    """Which pages are in use, and which entries of the table hold one."""
    table, page = s["table"].long(), s["case"]["page"]
    held = torch.arange(table.shape[1], device="cuda")[None, :] < ((s["lens"].long() + page - 1) // page)[:, None]
    used = torch.zeros(pages + 1, dtype=torch.bool, device="cuda")
    used[torch.where(held, table, pages).flatten()] = True
    return used[:pages], held


def _compact(s):
    pages, table = s["case"]["pages"], s["table"].long()
    used, held = _used(s, pages)
    live = used.sum()
    at = torch.arange(pages, device="cuda")
    src, dst = (used & (at >= live)).nonzero()[:, 0], (~used & (at < live)).nonzero()[:, 0]
    to = at.clone()
    to[src] = dst
    _copy_pages(src, dst, s["cache"], s["cache"])
    return {"table": torch.where(held, to[table.clamp(min=0)], table).to(torch.int32),
            "status": torch.stack([live, (used & (at >= live)).sum()]).to(torch.int32), **s["cache"]}


def _free(s):
    pages = s["case"]["pages"]
    free = ~_used(s, pages)[0]
    at = torch.where(free, free.long().cumsum(0) - 1, pages)
    got = torch.full((pages + 1,), -1, dtype=torch.int32, device="cuda")
    got[at] = torch.arange(pages, dtype=torch.int32, device="cuda")
    got = torch.where(torch.arange(pages, device="cuda") < free.sum(), got[:pages], -1)
    return {"free": got, "count": free.sum().to(torch.int32).view(1)}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------


def exact(case, seed):
    if case["kind"] not in ("rope", "logprobs"):
        return None  # page numbers, and bytes copied as they are
    s = prepare(case, seed)
    if case["kind"] == "rope":
        past, new = _rope_lens(case)
        pos = torch.cat([torch.arange(p, p + t, device="cuda", dtype=torch.float64) for p, t in zip(past, new)])
        rd, got = case["rotary"], {}
        freq = torch.tensor([case["theta"] ** (-2 * i / rd) for i in range(rd // 2)], dtype=torch.float64,
                            device="cuda")
        turn = torch.polar(torch.ones((pos.numel(), rd // 2), dtype=torch.float64, device="cuda"),
                           torch.outer(pos, freq))
        for n in ("q", "k"):
            x = s[n].double()
            if case["norm"]:
                x /= ((x ** 2).sum(-1, keepdim=True) / case["hd"] + 1e-6).sqrt()
                x *= 1 + s[n + "_weight"].double()
            z = torch.complex(x[..., :rd // 2], x[..., rd // 2:rd]) * turn[:, None, :]
            x[..., :rd // 2], x[..., rd // 2:rd] = z.real, z.imag
            got[n] = x
        return got
    parts = []
    for a in range(0, case["rows"], 64):
        x = s["logits"][a:a + 64].double() * case["scale"]
        lp = x - torch.logsumexp(x, -1, keepdim=True)
        lp = torch.where(torch.isnan(lp), -math.inf, lp)
        part = {}
        if s["tokens"] is not None:
            ids = s["tokens"][a:a + 64].long()
            part["logprobs"] = torch.where(ids < 0, 0.0, lp.gather(1, ids.clamp(min=0).view(len(x), -1)).view(ids.shape))
        part["entropy"] = torch.special.entr(lp.exp()).sum(-1)
        if case["top"]:
            part["top_logprobs"] = lp.topk(case["top"], -1).values
        parts.append(part)
    got = {n: torch.cat([p[n] for p in parts]) for n in parts[0]}
    if case["top"]:
        got["top_ids"] = None
    return got


# ---- work ----------------------------------------------------------------------------------------------------


def work(case):
    """Bytes and operations of one pass: each input read once, each output written once."""
    kind = case["kind"]
    if kind == "rope":
        tokens, rows = sum(_rope_lens(case)[1]), case["heads"] + case["kv"]
        size = SIZES[case["type"]]
        return {"bytes": 2 * tokens * rows * case["hd"] * size + 8 * case["requests"]
                + (2 * case["hd"] * size if case["norm"] else 0),
                "flops": tokens * rows * case["hd"] * (8 if case["norm"] else 3)}
    if kind == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * SIZES[case["type"]] + case["rows"] * (4 + 8 * case["given"] + 8 * case["top"]),
                "flops": 5 * n}
    if kind == "free":
        _, need, _ = _holdings(case)
        return {"bytes": 4 * (sum(need) + case["requests"] + case["pages"] + 1), "flops": 0}
    each = case["layers"] * case["kv"] * (2 * case["page"] * case["hd"] + 8)  # a page of all layers with its scales
    if kind == "copy":
        return {"bytes": case["count"] * (2 * each + 8), "flops": 0}
    _, need, _ = _holdings(case)
    if kind == "fork":
        return {"bytes": _forked(case) * (2 * each + 4) + 4 * (sum(need) + case["requests"])
                + 4 * case["children"] * (2 + max(need)) + 8, "flops": 0}
    return {"bytes": _moved(case) * 2 * each + 4 * (sum(need) + case["requests"] + case["requests"] * max(need)) + 8,
            "flops": 0}
