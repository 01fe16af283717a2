"""The request entry points on the GPU (mlc_vla.kv_cache): plan, cache writer, attention over the cache and over
packed prompts, against plain implementations in 64 bits (kvref.py, which derives the tolerances), and a serving
run of all of them together, captured and on other streams too."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import kvref as R
from conftest import TINY_KWARGS
from mlc_vla import _native as N
from mlc_vla import kv_cache as C
from mlc_vla import runtime

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _ints(v):
    return torch.tensor(list(v), dtype=torch.int32, device="cuda")


def _host(t):
    return t.detach().cpu().to(torch.float64).numpy()


def _say(request):
    print(request.node.name, flush=True)


@pytest.fixture(autouse=True)
def _named(request):
    _say(request)


# ---- plan ------------------------------------------------------------------------------------------


def _plan_case(rng, b, page, most_past, most_new, wide=None, spare=5):
    past, new = rng.integers(0, most_past + 1, b), rng.integers(0, most_new + 1, b)
    had = -(-past // page)
    has = -(-(past + new) // page)
    wide = int(has.max(initial=0)) + 2 if wide is None else wide
    total = int(has.sum()) + spare
    order = rng.permutation(total).astype(np.int32)
    table = np.full((b, wide), -7, np.int32)
    at = 0
    for i in range(b):
        n = min(int(had[i]), wide)
        table[i, :n] = order[at:at + n]
        at += int(had[i])
    return past, new, table, order[at:], total


def _check_plan(past, new, table, free, pages, page, tokens):
    want_table = table.copy()
    want = R.plan(past, new, want_table, free, pages, page, tokens)
    t = torch.from_numpy(table.copy()).cuda()
    got = C.kv_plan(_ints(past), _ints(new), t, _ints(free), num_pages=pages, page_size=page, tokens=tokens)
    for name, x, w in zip(got._fields, got, want):
        np.testing.assert_array_equal(x.numpy(), w, err_msg=name)
    np.testing.assert_array_equal(t.cpu().numpy(), want_table)
    return got


@pytest.mark.parametrize("b,page,past,new", [(1, 64, 0, 1), (5, 16, 40, 70), (16, 128, 1168, 1), (256, 32, 100, 33),
                                             (257, 16, 0, 5), (700, 64, 500, 3), (4096, 16, 20, 2)])
def test_plan(b, page, past, new):
    rng = np.random.default_rng(b + page)
    p, q, table, free, pages = _plan_case(rng, b, page, past, new)
    _check_plan(p, q, table, free, pages, page, int(q.sum()))
    _check_plan(p, q, table, free, pages, page, int(q.sum()) + 1500)  # a padded batch: -1 behind the last request


def test_plan_refusals_on_the_device():
    page, wide = 16, 8
    past = np.array([20, -1, 16, 100, 5, 0, 33, 128, 0])
    new = np.array([20, 5, -3, 40, 0, 64, 20, 0, 1])
    table = np.arange(9 * wide, dtype=np.int32).reshape(9, wide)
    for free in (list(range(72, 90)), [72, 73, 74], [], [500, -4, 80, 81, 82, 83, 84, 85, 86]):
        for tokens in (150, 140, 25, 0):
            _check_plan(past, new, table, np.array(free, np.int32), 90, page, tokens)
    # pages of the row that are not there give no slot
    table[0, 1] = 4000
    table[8, 0] = -1
    _check_plan(past, new, table, np.arange(72, 90, dtype=np.int32), 90, page, 150)
    # lengths near the largest int
    big = 2 ** 31 - 1
    _check_plan(np.array([big, 0, 3]), np.array([big, big, 4]), table[:3], np.arange(9, dtype=np.int32), 90, page, 50)


def test_plan_without_requests_or_tokens():
    _check_plan(np.zeros(0, int), np.zeros(0, int), np.zeros((0, 3), np.int32), np.arange(3, dtype=np.int32), 5, 16, 7)
    _check_plan(np.array([17]), np.array([0]), np.array([[3, 4]], np.int32), np.zeros(0, np.int32), 5, 16, 0)
    _check_plan(np.array([0]), np.array([4]), np.zeros((1, 0), np.int32), np.arange(3, dtype=np.int32), 5, 16, 4)


def test_plan_writes_into_a_given_plan():
    rng = np.random.default_rng(3)
    p, q, table, free, pages = _plan_case(rng, 9, 32, 60, 50)
    t = torch.from_numpy(table).cuda()
    args = (_ints(p), _ints(q), t, _ints(free))
    kw = dict(num_pages=pages, page_size=32, tokens=int(q.sum()))
    a = C.kv_plan(*args, **kw)
    b = C.KVPlan(*(torch.full_like(x.torch, 77) for x in a))
    assert C.kv_plan(*args, **kw, out=b) is b
    for x, y in zip(a, b):
        assert torch.equal(x.torch, y)
    with pytest.raises(ValueError, match="out"):
        C.kv_plan(*args, **{**kw, "tokens": kw["tokens"] + 1}, out=b)


# ---- write -----------------------------------------------------------------------------------------


def _cache(rng, pages, kv, hd, page, fill=True):
    """Caches with codes everywhere (so that what must stay is seen) and scales, and their values as arrays."""
    kc, vc = (torch.from_numpy(rng.integers(0, 255, s, dtype=np.uint8)).cuda().view(F8)
              for s in ((pages, kv, page, hd), (pages, kv, hd, page)))
    for c in (kc, vc):
        raw = c.view(torch.uint8)
        raw[(raw & 0x7f) == 0x7f] = 0x31  # no NaN
        if not fill:
            raw.zero_()
    ks, vs = (torch.from_numpy(np.exp2(rng.integers(-12, 3, (pages, kv))).astype(np.float32)).cuda() for _ in range(2))
    return kc, ks, vc, vs


def _slots(past, new, page, rng, spare=2):
    need = [-(-(p + n) // page) for p, n in zip(past, new)]
    order = rng.permutation(sum(need) + spare)
    out, at = [], 0
    for p, n, k in zip(past, new, need):
        ids = order[at:at + k]
        out += [int(ids[t // page]) * page + t % page for t in range(p, p + n)]
        at += k
    return out, len(order)


def _check_write(k, v, cu, slots, cache):
    kc, ks, vc, vs = cache
    page = kc.shape[2]
    want_k = R.write(_host(k), cu, slots, _host(kc), _host(ks), page)
    want_v = R.write(_host(v), cu, slots, _host(vc).transpose(0, 1, 3, 2).copy(), _host(vs), page)
    C.kv_write(k, v, _ints(cu), _ints(slots), kc, ks, vc, vs)
    for got, want in ((kc, want_k[0]), (ks, want_k[1]), (vc, want_v[0].transpose(0, 1, 3, 2)), (vs, want_v[1])):
        np.testing.assert_array_equal(_host(got), want)


def _rows(rng, shape, dtype, spread=3.0):
    x = rng.standard_normal(shape) * np.exp2(rng.uniform(-spread, spread, shape[:-1] + (1,)))
    return torch.from_numpy(x).to(dtype).cuda()


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("hd,kv,kt,vt", [(64, 1, "f16", "f16"), (128, 3, "bf16", "bf16"), (256, 1, "f32", "f16"),
                                         (256, 2, "f32", "f32")])
def test_write(page, hd, kv, kt, vt):
    rng = np.random.default_rng(page + hd)
    past, new = [0, page - 1, 3, page, 37, 0], [1, 2, page + 5, 3 * page, 1, 200]
    slots, pages = _slots(past, new, page, rng)
    cu = np.concatenate([[0], np.cumsum(new)])
    k, v = _rows(rng, (cu[-1], kv, hd), TYPES[kt]), _rows(rng, (cu[-1], kv, hd), TYPES[vt])
    cache = _cache(rng, pages, kv, hd, page)
    _check_write(k, v, cu, slots, cache)
    _check_write(k, v, cu, slots, cache)  # again over itself


@pytest.mark.parametrize("hd,kv", [(64, 2), (128, 1), (256, 2)])
@pytest.mark.parametrize("kt", ["f16", "f32"])
def test_write_strides_and_alignment(hd, kv, kt):
    rng = np.random.default_rng(hd)
    new = [70, 1, 31]
    slots, pages = _slots([5, 0, 16], new, 32, rng)
    cu = np.concatenate([[0], np.cumsum(new)])
    n = int(cu[-1])
    head_major = _rows(rng, (kv, n, hd), TYPES[kt]).transpose(0, 1)          # prefill's [KV][P][hd]
    wide = _rows(rng, (n, kv, hd + 24), TYPES["f16"])[:, :, 8:8 + hd]         # a slice of a wider row
    odd = _rows(rng, (n, kv, hd + 3), TYPES[kt])[:, :, 1:1 + hd]              # rows at odd addresses
    back = _rows(rng, (n, kv, hd), TYPES["bf16"]).flip(0)[::1]
    for k, v in ((head_major, wide), (odd, odd), (back, head_major), (wide[:1].expand(n, kv, hd), odd)):
        _check_write(k, v, cu, slots, _cache(rng, pages, kv, hd, 32))


@pytest.mark.parametrize("hd,kv,page", [(64, 5, 16), (128, 8, 32), (256, 3, 128)])
def test_write_of_many_pages(hd, kv, page):
    """Enough pages that a workgroup takes several heads in turn: what a call for each request writes."""
    rng = np.random.default_rng(page)
    new = rng.integers(1, 90 * page, 24).tolist()
    past = rng.integers(0, 3 * page, 24).tolist()
    slots, pages = _slots(past, new, page, rng)
    cu = np.concatenate([[0], np.cumsum(new)]).tolist()
    g = torch.Generator(device="cuda").manual_seed(page)
    k, v = (torch.randn((cu[-1], kv, hd), generator=g, device="cuda").half() for _ in range(2))
    one = _cache(rng, pages, kv, hd, page)
    two = [t.clone() for t in one]
    s = _ints(slots)
    C.kv_write(k, v, _ints(cu), s, *one)
    for a, z in zip(cu, cu[1:]):
        C.kv_write(k[a:z], v[a:z], _ints([0, z - a]), s[a:z], *two)
    for a, b in zip(one, two):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_write_values_of_every_size():
    """Zeros, subnormals, the largest values, infinities and NaN; pages that grow past codes that fall below 2^-6."""
    rng = np.random.default_rng(0)
    hd, page = 64, 16
    x = np.zeros((16 * 6, 1, hd), np.float32)
    x[16:32] = 1e-30                                       # under the smallest scale
    x[32:48] = rng.standard_normal((16, 1, hd)) * 1e38     # near the largest float32
    x[48:64] = rng.standard_normal((16, 1, hd))
    x[50, 0, :4] = [np.inf, -np.inf, np.nan, 1.0]
    x[64:80] = [[np.inf] * hd]                             # nothing finite
    x[80:96] = 448.0
    x[80, 0, 0] = 449.0
    cu, slots = [0, 96], list(range(96))
    t = torch.from_numpy(x).cuda()
    _check_write(t, t, cu, slots, _cache(rng, 7, 1, hd, page))
    # token by token, each larger than the last: the earlier codes move down into the subnormals and to zero
    cache = _cache(rng, 2, 1, hd, page)
    for i in range(16):
        t = torch.from_numpy(rng.standard_normal((1, 1, hd)) * 4.0 ** i).to(torch.bfloat16).cuda()
        _check_write(t, t, [0, 1], [16 + i], cache)


def test_write_slots_that_are_not_a_plans():
    """Negative slots, pages past the cache, tokens whose slots do not follow, offsets past the tokens: what the
    documentation says is written, nothing else changes."""
    rng = np.random.default_rng(5)
    hd, page, pages = 128, 32, 4
    n = 40
    x = _rows(rng, (n, 2, hd), torch.float16)
    ok = list(range(8, 8 + n))
    for slots in ([-1] * n, [page * pages + i for i in range(n)], ok[:10] + [90] + ok[11:], ok[:5] + [-1] * (n - 5),
                  [3] * n, [2 ** 31 - 1] * n, [31 + 64 * (i > 0) + i for i in range(n)]):
        _check_write(x, x, [0, n], slots, _cache(rng, pages, 2, hd, page))
    cache = _cache(rng, pages, 2, hd, page)
    before = [t.clone() for t in cache]
    for cu in ([0, 0], [n, n + 5], [5, 5, 5]):
        C.kv_write(x, x, _ints(cu), _ints(ok), *cache)
    for a, b in zip(cache, before):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# ---- attention over the cache ------------------------------------------------------------------------


def _paged(rng, past, new, kv, hd, page, wide=None):
    total = [p + n for p, n in zip(past, new)]
    need = [-(-t // page) for t in total]
    wide = max(need) + 1 if wide is None else wide
    order = rng.permutation(sum(need) + 2)
    table = np.full((len(past), wide), 2 ** 30, np.int32)
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = order[at:at + k]
        at += k
    return table, _cache(rng, len(order), kv, hd, page)


def _want_cached(q, cu, lens, table, cache, causal, scale):
    """Outputs and bounds of every token (float64)."""
    kc, ks, vc, vs = cache
    page, hd, pages = kc.shape[2], kc.shape[3], kc.shape[0]
    kf = _host(kc) * _host(ks)[..., None, None]
    vf = _host(vc).transpose(0, 1, 3, 2) * _host(vs)[..., None, None]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    qh = _host(q)
    for b, (a, z) in enumerate(zip(cu, cu[1:])):
        n, total = z - a, min(int(lens[b]), table.shape[1] * page)
        ids = table[b][:-(-total // page)]
        seen = [t for t in range(total) if 0 <= ids[t // page] < pages]
        k = np.stack([kf[ids[t // page], :, t % page] for t in seen]) if seen else np.zeros((0,) + kf.shape[1:2] + (hd,))
        v = np.stack([vf[ids[t // page], :, t % page] for t in seen]) if seen else k
        limit = [int(lens[b]) - n + i + 1 if causal else int(lens[b]) for i in range(n)]
        limit = [int(np.searchsorted(seen, x)) for x in limit]
        o, mass, big = R.attend(qh[a:z], k, v, limit, scale)
        out[a:z] = o
        tiny = 2.0 ** -37 * 448 * float(vs.max())
        tol[a:z] = R.bound(o, mass, big, q.dtype, max(len(seen), 1), hd, torch.float16, tiny)
    return out, tol


def _check_cached(q, cu, lens, table, cache, causal, scale=None, **kw):
    want, tol = _want_cached(q, cu, lens, table, cache, causal, q.shape[2] ** -0.5 if scale is None else scale)
    got = C.kv_attention(q, _ints(cu), _ints(lens), torch.from_numpy(table).cuda(), *cache, causal=causal,
                         scale=scale, **kw)
    g = _host(got.torch)
    end = cu[-1]
    assert np.array_equal(np.isnan(g[:end]), np.isnan(want[:end]))
    off = np.abs(g[:end] - want[:end])
    fine = ~np.isnan(want[:end])
    worst = (off[fine] / tol[:end][fine]).max(initial=0)
    print(f"  {worst:.3f} of the bound", flush=True)
    assert worst <= 1
    return got


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,hd,page,past,new", [
    (8, 1, 256, 64, [0, 968, 63, 64, 500], [1, 1, 1, 1, 1]),        # single tokens, odd lengths, one key
    (8, 1, 256, 32, [100, 968, 0], [50, 50, 50]),                   # action suffixes
    (4, 4, 64, 16, [15, 16, 17, 1000], [1, 2, 33, 7]),              # a kv head per query head
    (32, 8, 128, 16, [300, 5], [1, 3]),
    (7, 1, 128, 128, [0, 260, 129], [63, 1, 20]),                   # seven heads: groups that end inside a row tile
    (16, 2, 64, 64, [700, 3], [1, 1]),
    (40, 2, 128, 32, [65, 90], [1, 2]),                             # twenty heads on a kv head: more than a row tile
])
def test_kv_attention(dt, heads, kv, hd, page, past, new):
    rng = np.random.default_rng(heads + hd + page)
    table, cache = _paged(rng, past, new, kv, hd, page)
    cu = np.concatenate([[0], np.cumsum(new)])
    q = _rows(rng, (cu[-1], heads, hd), TYPES[dt], spread=0.5)
    lens = [p + n for p, n in zip(past, new)]
    for causal in (True, False):
        a = _check_cached(q, cu, lens, table, cache, causal)
        # a wrong bound on the lengths changes the cut of the work, not the result
        _check_cached(q, cu, lens, table, cache, causal, max_kv=1)
        _check_cached(q, cu, lens, table, cache, causal, max_kv=10 ** 6)
        b = C.kv_attention(q, _ints(cu), _ints(lens), torch.from_numpy(table).cuda(), *cache, causal=causal)
        assert torch.equal(a.torch, b.torch)


def test_kv_attention_scales_of_every_size():
    """Page scales that are far apart, not powers of two, zero; a softmax scale of its own."""
    rng = np.random.default_rng(2)
    past, new = [400, 90], [3, 1]
    table, (kc, ks, vc, vs) = _paged(rng, past, new, 2, 128, 16)
    ks.copy_(torch.from_numpy(np.exp2(rng.uniform(-14, -9, ks.shape))))
    vs.copy_(torch.from_numpy(np.exp2(rng.uniform(-60, 40, vs.shape))))
    vs[::5] = 0.0
    q = _rows(rng, (4, 4, 128), torch.bfloat16, 0.5)
    _check_cached(q, [0, 3, 4], [403, 91], table, (kc, ks, vc, vs), True)
    _check_cached(q, [0, 3, 4], [403, 91], table, (kc, ks, vc, vs), True, scale=0.5)


@pytest.mark.parametrize("hd", [64, 256])
def test_kv_attention_lengths_and_pages_out_of_range(hd):
    """Refused and empty requests, lengths past the table, pages that are not there: zeros, or what is there."""
    rng = np.random.default_rng(8)
    page, past, new = 16, [30, 40, 0, 64, 100, 20], [2, 1, 3, 0, 1, 4]
    table, cache = _paged(rng, past, new, 1, hd, page, wide=8)
    cu = np.concatenate([[0], np.cumsum(new)])
    q = _rows(rng, (cu[-1] + 3, 8, hd), torch.float16, 0.5)
    lens = [32, 0, 1, 64, 10 ** 6, 24]     # request 1 refused, 2 shorter than its queries, 4 past its row
    table[4, :] = table[4, 0]
    table[0, 1] = -1
    table[5, 0] = 2 ** 31 - 1
    out = torch.full((cu[-1] + 3, 8, hd), 7.0, dtype=torch.float16, device="cuda")
    for causal in (True, False):
        got = _check_cached(q, cu, lens, table, cache, causal, out=out)
        assert got.torch.data_ptr() == out.data_ptr()
        assert (out[cu[-1]:] == 7).all()   # rows behind the last request
        assert (out[2] == 0).all()
    # no pages at all: every row is zero
    none = tuple(t[:0] for t in cache)
    o = C.kv_attention(q, _ints(cu), _ints(lens), torch.from_numpy(table).cuda(), *none)
    assert (o.torch[:cu[-1]] == 0).all()
    o = C.kv_attention(q[:0], _ints([0]), _ints([]), torch.zeros((0, 4), dtype=torch.int32, device="cuda"), *cache)
    assert o.shape == (0, 8, hd)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_kv_attention_nan_behind_the_mask(dt, hd):
    """NaN codes behind a request's last token, on pages that are not its own and in later tokens of its own:
    rows that do not see them are as if they were not there; rows that do are NaN."""
    rng = np.random.default_rng(9)
    page, past, new = 32, [50, 70], [5, 1]
    table, (kc, ks, vc, vs) = _paged(rng, past, new, 1, hd, page)
    q = _rows(rng, (6, 8, hd), TYPES[dt], 0.5)
    kr, vr = kc.view(torch.uint8), vc.view(torch.uint8)
    kr[table[0, 1], :, 55 - 32:] = 0x7f
    vr[table[0, 1], :, :, 55 - 32:] = 0xff
    kr[table[1, 2], :, 71 - 64:] = 0xff
    vr[table[1, 2], :, :, 71 - 64:] = 0x7f
    for causal in (True, False):
        got = _check_cached(q, [0, 5, 6], [55, 71], table, (kc, ks, vc, vs), causal)
        assert torch.isfinite(got.torch.float()).all()
    vr[table[0, 1], 0, 3, 53 - 32] = 0x7f  # the value of token 53, dim 3: seen by tokens 53 and 54
    got = _check_cached(q, [0, 5, 6], [55, 71], table, (kc, ks, vc, vs), True)
    bad = torch.isnan(got.torch.float())
    assert bad[3:5, :, 3].all() and int(bad.sum()) == 16
    kr[table[0, 1], 0, 54 - 32, 0] = 0x7f  # the key of token 54
    got = _check_cached(q, [0, 5, 6], [55, 71], table, (kc, ks, vc, vs), True)
    assert torch.isnan(got.torch[4].float()).all() and torch.isfinite(got.torch[:3].float()).all()


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("dt,hd", [("f16", 64), ("bf16", 128), ("f16", 256)])
def test_kv_attention_suffixes(dt, hd, page):
    """Many rows over long contexts, as action suffixes are: more waves to a workgroup, no splits."""
    rng = np.random.default_rng(40)
    past, new = [1018, 700, 0, 903, 65, 1200], [50, 50, 50, 0, 33, 50]
    table, (kc, ks, vc, vs) = _paged(rng, past, new, 1, hd, page)
    cu = np.concatenate([[0], np.cumsum(new)])
    lens = [p + n for p, n in zip(past, new)]
    table[1, 3] = -1
    kr, vr = kc.view(torch.uint8), vc.view(torch.uint8)
    last = table[5, (lens[5] - 1) // page], (lens[5] - 1) % page + 1   # NaN behind a request's end
    kr[last[0], :, last[1]:] = 0x7f
    vr[last[0], :, :, last[1]:] = 0xff
    q = _rows(rng, (cu[-1], 8, hd), TYPES[dt], 0.5)
    for causal in (True, False):
        got = _check_cached(q, cu, lens, table, (kc, ks, vc, vs), causal)
        assert torch.isfinite(got.torch.float()).all()
    vr[table[0, 0], 0, 5, 7] = 0x7f        # a value that every row of request 0 sees
    got = _check_cached(q, cu, lens, table, (kc, ks, vc, vs), False)
    bad = torch.isnan(got.torch.float())
    assert bad[:50, :, 5].all() and int(bad.sum()) == 50 * 8


def test_kv_attention_strides_and_workspace():
    rng = np.random.default_rng(4)
    past, new, hd = [900, 40], [2, 9], 128
    table, cache = _paged(rng, past, new, 2, hd, 64)
    cu, lens = [0, 2, 11], [902, 49]
    t = torch.from_numpy(table).cuda()
    q = _rows(rng, (11, 3 * 8, hd), torch.float16, 0.5)[:, 8:16]      # a slice of fused q/k/v rows
    want = C.kv_attention(q.contiguous(), _ints(cu), _ints(lens), t, *cache).torch
    out = torch.zeros((8, 11, hd + 2), dtype=torch.float16, device="cuda").transpose(0, 1)[:, :, 1:1 + hd]
    odd = torch.zeros((11, 8, hd + 1), dtype=torch.float16, device="cuda")[:, :, 1:]
    odd.copy_(q)
    need = C.kv_attention_workspace(11, 2, 8, 2, hd, table.shape[1] * 64)
    ws = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")
    for x in (q, odd):
        C.kv_attention(x, _ints(cu), _ints(lens), t, *cache, out=out, workspace=ws)
        assert torch.equal(out, want)
    assert need > 0 and (ws[need:] == 255).all()
    with pytest.raises(N.MlcvError, match="workspace"):
        C.kv_attention(q, _ints(cu), _ints(lens), t, *cache, workspace=ws[:need - 16])
    with pytest.raises(N.MlcvError, match="workspace"):
        C.kv_attention(q, _ints(cu), _ints(lens), t, *cache, workspace=ws[8:])


def test_cache_past_32_bit_offsets():
    """More than 4 GiB of pages on each side: writes to and reads from the last ones."""
    rng = np.random.default_rng(6)
    hd, page, pages = 256, 128, (1 << 32) // (256 * 128) + 40
    kc = torch.empty((pages, 1, page, hd), dtype=torch.uint8, device="cuda").view(F8)
    vc = torch.empty((pages, 1, hd, page), dtype=torch.uint8, device="cuda").view(F8)
    ks, vs = torch.empty((pages, 1), device="cuda"), torch.empty((pages, 1), device="cuda")
    ids = [pages - 1, 3, pages - 30, pages // 2]
    n = 4 * page
    slots = [ids[t // page] * page + t % page for t in range(n)]
    k, v = _rows(rng, (n, 1, hd), torch.float16, 1), _rows(rng, (n, 1, hd), torch.float16, 1)
    C.kv_write(k, v, _ints([0, n]), _ints(slots), kc, ks, vc, vs)
    ref = _cache(rng, 4, 1, hd, page, fill=False)
    C.kv_write(k, v, _ints([0, n]), _ints(range(n)), *ref)
    at = torch.tensor(ids, device="cuda")
    for a, b in zip((kc, ks, vc, vs), ref):
        a, b = (x.view(torch.uint8) if x.dtype == F8 else x for x in (a, b))
        assert torch.equal(a[at], b)
    q = _rows(rng, (2, 8, hd), torch.float16, 0.5)
    big = C.kv_attention(q, _ints([0, 2]), _ints([n - 3]), _ints(ids).view(1, 4), kc, ks, vc, vs).torch
    want = C.kv_attention(q, _ints([0, 2]), _ints([n - 3]), _ints(range(4)).view(1, 4), *ref).torch
    assert torch.equal(big, want)


# ---- attention over packed prompts -------------------------------------------------------------------


def _limits(n, causal, bidir):
    return [max(i + 1, min(max(bidir, 0), n)) if causal else n for i in range(n)]


def _check_prompts(q, k, v, cu, causal, bidir=None, scale=None, out=None):
    dt = q.dtype
    qh, kh, vh = _host(q), _host(k), _host(v)
    got = C.prompt_attention(q, k, v, _ints(cu), causal=causal, bidir=None if bidir is None else _ints(bidir),
                             scale=scale, out=out)
    g = _host(got.torch)
    worst = 0.0
    for b, (a, z) in enumerate(zip(cu, cu[1:])):
        n = z - a
        lim = _limits(n, causal, bidir[b] if bidir is not None else 0)
        o, mass, big = R.attend(qh[a:z], kh[a:z], vh[a:z], lim, q.shape[2] ** -0.5 if scale is None else scale)
        seen = np.abs(vh[a:z])
        top = seen[np.isfinite(seen)].max(initial=0)
        tol = R.bound(o, mass, big, dt, n, q.shape[2], dt, 2.0 ** -25 * top if dt == torch.float16 else 0.0)
        assert np.array_equal(np.isnan(g[a:z]), np.isnan(o))
        inf = np.isinf(o)
        assert np.array_equal(g[a:z][inf], o[inf])
        fine = np.isfinite(o)
        worst = max(worst, (np.abs(g[a:z] - o)[fine] / tol[fine]).max(initial=0))
    print(f"  {worst:.3f} of the bound", flush=True)
    assert worst <= 1
    return got


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,hd,lens", [
    (2, 1, 64, [1, 63, 64, 65, 130]),
    (8, 1, 256, [33, 300, 1, 128]),
    (8, 2, 128, [129, 0, 257, 5]),
    (7, 7, 64, [200]),
    (3, 1, 128, [2, 31, 32, 96]),
    (1, 1, 256, [31, 97]),
])
def test_prompt_attention(dt, heads, kv, hd, lens):
    rng = np.random.default_rng(heads + hd)
    cu = [0] + np.cumsum(lens).tolist()
    q, k, v = (_rows(rng, (cu[-1], h, hd), TYPES[dt], 0.5) for h in (heads, kv, kv))
    _check_prompts(q, k, v, cu, True)
    _check_prompts(q, k, v, cu, False)
    _check_prompts(q, k, v, cu, True, bidir=[(7 * i + 40) % (n + 2) - 1 for i, n in enumerate(lens)])
    _check_prompts(q, k, v, cu, True, bidir=[10 ** 6 * (i % 2) + 50 for i in range(len(lens))], scale=0.3)


@pytest.mark.parametrize("hd,kv", [(64, 8), (128, 1), (256, 2)])
def test_prompt_attention_of_many_heads(hd, kv):
    """More than 128 workgroups of 128 rows: no sharing of rows between waves."""
    rng = np.random.default_rng(hd)
    lens = [140, 1, 233]
    cu = [0] + np.cumsum(lens).tolist()
    q, k, v = (_rows(rng, (cu[-1], h, hd), torch.bfloat16 if hd == 64 else torch.float16, 0.5) for h in (48, kv, kv))
    _check_prompts(q, k, v, cu, True, bidir=[0, 1, 150])
    _check_prompts(q[:, :40], k, v, cu, False, scale=0.2)
    ramp = torch.linspace(0, 6, cu[-1], device="cuda").to(k.dtype)[:, None, None]  # maxima that come late
    _check_prompts(q, k * (1 + ramp), v, cu, True)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("hd,heads", [(64, 2), (128, 2), (256, 2), (64, 64), (128, 64), (256, 64)])
def test_prompt_attention_non_finite_behind_the_mask(dt, hd, heads):
    """NaN and infinities in tokens that a row does not see, of its own prompt and of its neighbours, do not reach it."""
    rng = np.random.default_rng(12)
    lens = [150, 70, 40]
    cu = [0] + np.cumsum(lens).tolist()
    q, k, v = (_rows(rng, (cu[-1], h, hd), TYPES[dt], 0.5) for h in (heads, 1, 1))
    v[100, 0, 5] = float("inf")
    v[101, 0, 6] = float("nan")
    v[120, 0, 5] = float("-inf")
    k[140] = float("nan")
    v[cu[1]:cu[2]] = float("nan")   # the whole middle prompt
    k[cu[1]:cu[2]] = float("inf")
    with np.errstate(all="ignore"):
        got = _check_prompts(q, k, v, cu, True).torch.float()
        assert torch.isfinite(got[:100]).all() and torch.isfinite(got[cu[2]:]).all()
        assert torch.isposinf(got[100:120, :, 5]).all() and torch.isnan(got[140:150]).all()
        _check_prompts(q, k, v, cu, True, bidir=[90, 3, 0])


def test_prompt_attention_strides_and_rows_behind():
    rng = np.random.default_rng(13)
    lens, hd = [45, 130], 128
    cu = [0] + np.cumsum(lens).tolist()
    n = cu[-1] + 6
    qkv = _rows(rng, (n, 8 + 2 + 2, hd), torch.float16, 0.5)
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    want = C.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), _ints(cu)).torch
    out = torch.full((n, 8, hd), 5.0, dtype=torch.float16, device="cuda")
    _check_prompts(q, k, v, cu, True, out=out)
    assert torch.equal(out[:cu[-1]], want[:cu[-1]]) and (out[cu[-1]:] == 5).all()
    # head-major tensors, rows at odd addresses (copied), one key and value for all tokens (stride 0, copied)
    hm = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    odd = [torch.zeros((n, x.shape[1], hd + 1), dtype=x.dtype, device="cuda")[:, :, 1:].copy_(x) for x in (q, k, v)]
    for a in (hm, odd, (q, odd[1], hm[2])):
        assert torch.equal(C.prompt_attention(*a, _ints(cu)).torch[:cu[-1]], want[:cu[-1]])
    one = k[:1].expand(n, 2, hd)
    _check_prompts(q, one, v, cu, True)
    assert C.prompt_attention(q[:0], k[:0], v[:0], _ints([0])).shape == (0, 8, hd)
    # offsets past the tokens are cut
    a = C.prompt_attention(q, k, v, _ints([0, 45, 10 ** 6])).torch
    b = C.prompt_attention(q, k, v, _ints([0, 45, n])).torch
    assert torch.equal(a, b)


def test_offsets_that_do_not_ascend():
    """cu_seqlens that overlap, descend or lie outside: nothing outside the tensors is touched, and a request whose
    offsets are sound and meet no other's is right."""
    rng = np.random.default_rng(17)
    n, hd = 300, 64
    q, k, v = (_rows(rng, (n, h, hd), torch.float16, 0.5) for h in (2, 1, 1))
    store = torch.full((n + 64, 2, hd), 9.0, dtype=torch.float16, device="cuda")
    out = store[32:32 + n]
    table, cache = _paged(rng, [500, 500, 500], [1, 1, 1], 1, hd, 16)
    t = torch.from_numpy(table).cuda()
    for cu in ([0, 290, 20, 300], [0, 300, 0, 300], [250, 100, 299, 10 ** 6], [-50, -1, 300, 2 ** 31 - 1],
               [2 ** 31 - 1, -2 ** 31, 300, 0]):
        out.fill_(9.0)
        C.prompt_attention(q, k, v, _ints(cu), out=out)
        C.kv_attention(q, _ints(cu), _ints([400, 2 ** 31 - 1, -5]), t, *cache, out=out)
        C.kv_attention(q, _ints(cu), _ints([400, 2 ** 31 - 1, -5]), t, *cache, max_kv=1, causal=False, out=out)
        C.kv_write(k, v, _ints(cu), _ints(range(n)), *cache)
        torch.cuda.synchronize()
        assert (store[:32] == 9).all() and (store[32 + n:] == 9).all()


def test_prompt_attention_large_logits():
    """Rows whose maximum comes late and is far above what came before, and weights that all underflow."""
    rng = np.random.default_rng(14)
    q, k, v = (_rows(rng, (300, h, 64), torch.float16, 0.5) for h in (2, 2, 2))
    ramp = torch.linspace(0, 12, 300, device="cuda").half()[:, None, None]
    _check_prompts(q, k * (1 + ramp), v, [0, 300], True, scale=1.0)
    _check_prompts(q, k * (1 + ramp.flip(0)), v, [0, 300], False, scale=4.0)
    _check_prompts(q * 0, k, v, [0, 300], True)


def test_prompt_attention_tokens_far_apart():
    """A token stride that puts the tensors past 4 GiB."""
    rng = np.random.default_rng(15)
    n, far = 600, 1 << 23
    store = torch.empty(n * far // 2, dtype=torch.float32, device="cuda").view(torch.float16)  # 10 GB
    k, v = (store[o:].as_strided((n, 1, 64), (far, 64, 1)) for o in (0, 4096))
    q, a, b = (_rows(rng, (n, 2 if i == 0 else 1, 64), torch.float16, 0.5) for i in range(3))
    k.copy_(a)
    v.copy_(b)
    got = C.prompt_attention(q, k, v, _ints([0, 70, n])).torch
    assert torch.equal(got, C.prompt_attention(q, a, b, _ints([0, 70, n])).torch)


# ---- together --------------------------------------------------------------------------------------


class _Server:
    """Three requests of a two-layer attention stack: prompts, then tokens one by one, on one cache."""

    def __init__(self, dt=torch.float16, seed=20, lens=(100, 7, 33), heads=8, kv=2, hd=64, page=16, layers=2):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.dt, self.h, self.kv, self.hd, self.page, self.layers = dt, heads, kv, hd, page, layers
        self.lens = list(lens)
        self.cache = C.PagedKVCache(64, page, kv, hd, layers)
        self.table = torch.full((len(lens), 12), -1, dtype=torch.int32, device="cuda")
        self.free = torch.arange(63, -1, -1, dtype=torch.int32, device="cuda")
        self.used = 0
        self.k = [[torch.zeros((0, kv, hd), dtype=dt, device="cuda") for _ in lens] for _ in range(layers)]
        self.v = [list(x) for x in self.k]

    def rand(self, n, h):
        return torch.randn((n, h, self.hd), generator=self.g, device="cuda").to(self.dt)

    def step(self, new, past):
        """Plan and write `new` tokens for each request; (plan, per-layer q, k, v)."""
        t = sum(new)
        plan = self.cache.plan(_ints(past), _ints(new), self.table, self.free[self.used:], t)
        assert plan.status.numpy()[1] == 0
        self.used += int(plan.status.numpy()[0])
        qkv = []
        for y in range(self.layers):
            q, k, v = (self.rand(t, h) for h in (self.h, self.kv, self.kv))
            self.cache.write(k, v, plan, y)
            at = 0
            for b, n in enumerate(new):
                self.k[y][b] = torch.cat([self.k[y][b], k[at:at + n]])
                self.v[y][b] = torch.cat([self.v[y][b], v[at:at + n]])
                at += n
            qkv.append((q, k, v))
        return plan, qkv

    def held(self, y, b):
        """What the cache holds of request b: K and V [len, KV, hd] in float64."""
        kc, ks, vc, vs = self.cache.pages(y)
        n = self.k[y][b].shape[0]
        ids = self.table[b].cpu().numpy()
        kf = _host(kc) * _host(ks)[..., None, None]
        vf = _host(vc).transpose(0, 1, 3, 2) * _host(vs)[..., None, None]
        return tuple(np.stack([x[ids[t // self.page], :, t % self.page] for t in range(n)]) for x in (kf, vf))


def test_serving_run():
    s = _Server()
    past = [0, 0, 0]
    plan, qkv = s.step(s.lens, past)
    cu = plan.cu_seqlens.numpy().tolist()
    for y, (q, k, v) in enumerate(qkv):
        _check_prompts(q, k, v, cu, True, bidir=[80, 7, 0])
    past = list(s.lens)
    for i in range(20):
        new = [1, 1, 1] if i != 7 else [5, 0, 17]  # and an action suffix in between
        plan, qkv = s.step(new, past)
        past = [p + n for p, n in zip(past, new)]
        cu = np.concatenate([[0], np.cumsum(new)])
        for y, (q, _, _) in enumerate(qkv):
            got = _host(s.cache.attention(q, plan, s.table, y).torch)
            for b, n in enumerate(new):
                if not n:
                    continue
                k, v = s.held(y, b)
                lim = [past[b] - n + j + 1 for j in range(n)]
                o, mass, big = R.attend(_host(q[cu[b]:cu[b + 1]]), k, v, lim, s.hd ** -0.5)
                tol = R.bound(o, mass, big, s.dt, past[b], s.hd, torch.float16, 2.0 ** -37 * 448 * 16)
                assert (np.abs(got[cu[b]:cu[b + 1]] - o) <= tol).all()
    # every cached value is the token's own under its page's scale: within half a step of e4m3, or of its
    # subnormals at the scale; rescaling a page rounds once more, then below 2^-6 of the scale only
    for y in range(s.layers):
        for b in range(3):
            k, v = s.held(y, b)
            for got, own in ((k, s.k[y][b]), (v, s.v[y][b])):
                x = _host(own)
                top = np.stack([np.abs(x[p:p + s.page]).max((0, 2)) for p in range(0, len(x), s.page)])
                top = np.repeat(top, s.page, 0)[:len(x)][..., None]
                # scale < 2 max / 224; a subnormal step is 2^-9 of it, half of that at each of two roundings
                assert (np.abs(got - x) <= 2.0 ** -4 * np.abs(x) + 2.0 ** -9 * top / 112).all()


def test_prefill_output_into_the_cache():
    """One layer of prefill's float32 keys and float16 values, in place, and the action suffix's queries over it:
    the joint attention over the dense cache, but for the 8 bits."""
    from mlc_vla.model.pi0 import Pi0Config
    from mlc_vla.sample import PiZeroRunner, make_prefix_mask_np
    from oracle import pi0_oracle as O

    cfg = Pi0Config(**TINY_KWARGS)
    d = O.dims_from_config(cfg)
    runner = PiZeroRunner(cfg, "rocm")
    p16 = O.make_params(O.param_specs(d), 0, "float16")
    params = runner.to_params([p16[n] for n, _ in runner.named_params])
    prefix = np.random.default_rng(3).standard_normal((1, cfg.prefix_len, cfg.vlm.width)).astype(np.float16)
    keys, values = runner.vm["prefill"](runtime.tensor(prefix), runtime.tensor(make_prefix_mask_np(cfg.prefix_len)),
                                        params)
    kv, hd, heads, p = cfg.vlm.num_kv_heads, cfg.vlm.head_dim, cfg.vlm.num_heads, cfg.prefix_len
    cache = C.PagedKVCache(4, 16, kv, hd, layers=cfg.vlm.depth)
    table = torch.full((1, 3), -1, dtype=torch.int32, device="cuda")
    plan = cache.plan(_ints([0]), _ints([p]), table, _ints([2, 0, 3]), p)
    t = 8
    q = torch.randn((t, heads, hd), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").half()
    for y in range(cfg.vlm.depth):
        k, v = keys.torch[y, 0].transpose(0, 1), values.torch[y, 0].transpose(0, 1)  # [P, KV, hd] views
        cache.write(k, v, plan, y)
        look = C.KVPlan(_ints([0, t]), plan.kv_lens, plan.slot_map, plan.status)
        got = cache.attention(q, look, table, y, causal=False).torch
        dense = torch.empty((t, heads * hd), dtype=torch.float16, device="cuda")
        qs = (q.float() * hd ** -0.5).half().reshape(t, heads * hd)
        ptr = lambda x: ctypes.c_void_p(x.data_ptr())  # noqa: E731
        N.call("mlcv_joint_attention", ptr(qs), t, heads, kv, hd, ptr(keys.torch[y]), 1, ptr(values.torch[y]), p, None,
               None, None, 0, ptr(dense), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        # a key is off by at most 2^-4 of itself (or of 2^-6 of its page's largest): the logits move by at most
        # 2^-4 sum |q||k| (and that floor), the weights by twice that, the values by 2^-4 of themselves
        kf, vf, qf = _host(k), _host(v), _host(q)
        o, mass, big = R.attend(qf, kf, vf, [p] * t, hd ** -0.5)
        move = 2 * (2.0 ** -4 * big + 2.0 ** -9 / 112 * np.abs(kf).max() * np.abs(qf).sum(-1, keepdims=True) * hd ** -0.5)
        tol = (np.expm1(move) + 2.0 ** -4 + 2.0 ** -9) * mass + 2.0 ** -4 * np.abs(vf).max() * 2.0 ** -3 + 1e-3
        assert (np.abs(_host(got) - _host(dense).reshape(o.shape)) <= tol).all()


def test_captured_step_replays():
    """Plan, write and attention of a decode step as one graph: new inputs before each replay, eager work and
    synchronization between them, every replay against the eager result."""
    s = _Server(torch.bfloat16, lens=(40, 90, 3))
    s.step(s.lens, [0, 0, 0])
    past, new = _ints(s.lens), _ints([1, 1, 1])
    q, k, v = s.rand(3, s.h), s.rand(3, s.kv), s.rand(3, s.kv)
    free = s.free[s.used:].clone()

    def step():
        plan = s.cache.plan(past, new, s.table, free, 3)
        s.cache.write(k, v, plan, 1)
        return plan, s.cache.attention(q, plan, s.table, 1).torch, C.prompt_attention(q, k, v, plan.cu_seqlens).torch

    start = [t.clone() for t in s.cache.pages(1)] + [s.table.clone()]

    def restore():
        for a, b in zip(list(s.cache.pages(1)) + [s.table], start):
            (a.view(torch.uint8) if a.dtype == F8 else a).copy_(b.view(torch.uint8) if b.dtype == F8 else b)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs, each with its own plan and workspace
        restore()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, got))
    for i in range(4):
        for graph, (plan, out, own) in graphs:
            for x in (q, k, v):
                x.copy_(torch.randn(x.shape, generator=s.g, device="cuda") * 2.0 ** i)
            restore()
            want_plan, want, want_own = step()
            pages = [t.clone() for t in s.cache.pages(1)]
            torch.cuda.synchronize()
            restore()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(own, want_own)
            for a, b in zip(plan, want_plan):
                assert torch.equal(a.torch, b.torch)
            for a, b in zip(s.cache.pages(1), pages):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_two_streams_at_once():
    """Calls of two streams that overlap: each has its own workspace."""
    rng = np.random.default_rng(30)
    past = [3000, 2500]
    jobs = []
    for i in range(2):
        table, cache = _paged(rng, past, [1, 1], 1, 256, 64)
        q = _rows(rng, (2, 8, 256), torch.float16, 0.5)
        args = (q, _ints([0, 1, 2]), _ints([3001, 2501]), torch.from_numpy(table).cuda(), *cache)
        jobs.append((args, C.kv_attention(*args).torch, torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i, (args, _, st) in enumerate(jobs):
            with torch.cuda.stream(st):
                outs[i].append(C.kv_attention(*args).torch)
    torch.cuda.synchronize()
    for i, (_, want, _) in enumerate(jobs):
        for o in outs[i]:
            assert torch.equal(o, want)


def test_arguments_are_checked():
    """Refusals that need device tensors (the others: test_kv_cache_args.py)."""
    rng = np.random.default_rng(31)
    table, cache = _paged(rng, [20], [1], 2, 64, 16)
    kc, ks, vc, vs = cache
    t = torch.from_numpy(table).cuda()
    q = _rows(rng, (1, 4, 64), torch.float16)
    cu, lens = _ints([0, 1]), _ints([21])
    C.kv_attention(q, cu, lens, t, *cache)
    for args, kw, what in (
            ((q.float(), cu, lens, t, *cache), {}, "dtype"),
            ((q[0], cu, lens, t, *cache), {}, "shape"),
            ((q[:, :, :32], cu, lens, t, *cache), {}, "argument q expects shape"),
            ((q.transpose(1, 2), cu, lens, t, *cache), {}, "argument q expects shape"),
            ((q, cu.long(), lens, t, *cache), {}, "cu_seqlens"),
            ((q, cu, lens, t[:, ::2], *cache), {}, "contiguous"),
            ((q, cu, lens, t, kc, ks, kc, vs), {}, "v_cache"),
            ((q, cu, lens, t, kc, ks[:1], vc, vs), {}, "k_scale"),
            ((q, cu, lens.cpu(), t, *cache), {}, "device"),
            ((q, cu, lens, t, *cache), {"out": q[:0]}, "out")):
        with pytest.raises(ValueError, match=what):
            C.kv_attention(*args, **kw)
    with pytest.raises(N.MlcvError, match="multiple of the kv heads"):
        C.kv_attention(q[:, :3], cu, lens, t, *cache)
    with pytest.raises(N.MlcvError, match="scale"):
        C.kv_attention(q, cu, lens, t, *cache, scale=0.0)
    x = _rows(rng, (1, 2, 64), torch.float16)
    with pytest.raises(N.MlcvError, match="bidir"):
        C.prompt_attention(q, x, x, cu, causal=False, bidir=_ints([1]))
    with pytest.raises(ValueError, match="dtype"):
        C.prompt_attention(q, x.bfloat16(), x, cu)
    with pytest.raises(ValueError, match="slot_map"):
        C.kv_write(x, x, cu, _ints([0, 1]), *cache)
    with pytest.raises(ValueError, match="argument k expects shape"):
        C.kv_write(x[:, :1], x, cu, _ints([0]), *cache)
    with pytest.raises(ValueError, match="new_lens"):
        C.kv_plan(_ints([0]), _ints([1, 2]), t, _ints([1]), num_pages=4, page_size=16, tokens=3)
