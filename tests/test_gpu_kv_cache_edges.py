"""The request entry points where their inputs touch what is not theirs: pages that no request uses, page numbers that
are not there.  Plain 64-bit forms and bounds as in test_gpu_kv_cache.py."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import kvref as R
from mlc_vla import _native as N
from mlc_vla import kv_cache as C
from test_gpu_kv_cache import F8, TYPES, _cache, _host, _ints, _rows, _say, _want_cached

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _named(request):
    _say(request)


def _own_pages(rng, lens, kv, hd, page, wide, unused=4):
    """A cache whose pages 0 and, `unused` in all, its last ones belong to no request, and a table whose entries behind
    the requests' own are -1, such pages, and numbers past the cache."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + unused
    order = rng.permutation(sum(need)) + 1
    table = np.zeros((len(lens), wide), np.int32)
    at = 0
    for i, k in enumerate(need):
        table[i] = [(-1, 0, total - 1, 2 ** 31 - 1, total)[(i + j) % 5] for j in range(wide)]
        table[i, :k] = order[at:at + k]
        at += k
    return table, _cache(rng, total, kv, hd, page), [0] + list(range(total - unused + 1, total))


def _check(q, cu, lens, table, cache, causal, want, tol, **kw):
    got = C.kv_attention(q, _ints(cu), _ints(lens), torch.from_numpy(table).cuda(), *cache, causal=causal, **kw)
    g = _host(got.torch)
    assert np.isfinite(g).all()
    worst = (np.abs(g - want) / tol).max()
    print(f"  {worst:.3f} of the bound", flush=True)
    assert worst <= 1


# ---- attention over the cache ------------------------------------------------------------------------


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 64, 128])
def test_kv_attention_scales_of_pages_not_in_use(dt, hd, page):
    """Page scales that are NaN, infinite or negative wherever no request has its tokens: behind a request's last page,
    at page 0 (which stands in for numbers that are not there) and in holes.  No row sees them."""
    rng = np.random.default_rng(page + hd)
    past, new = [5, 70, 900, 2 * page - 1], [1, 3, 2, 1]
    lens, cu = [p + n for p, n in zip(past, new)], np.concatenate([[0], np.cumsum(new)])
    table, (kc, ks, vc, vs), unused = _own_pages(rng, lens, 2, hd, page, 2 + -(-902 // page))
    table[2, 3] = -1                                      # a hole
    table[2, 5] = 2 ** 31 - 1
    q = _rows(rng, (cu[-1], 8, hd), TYPES[dt], 0.5)
    for causal in (True, False):
        want, tol = _want_cached(q, cu, lens, table, (kc, ks, vc, vs), causal, hd ** -0.5)
        for x in (float("nan"), float("inf"), float("-inf"), -1.0):
            bad_k, bad_v = ks.clone(), vs.clone()
            bad_k[unused], bad_v[unused] = x, x
            for most in (None, 1, 10 ** 6):                # other cuts of the keys
                _check(q, cu, lens, table, (kc, bad_k, vc, bad_v), causal, want, tol, max_kv=most)


# ---- write -----------------------------------------------------------------------------------------


def _check_only(x, cu, slots, written, cache):
    """kv_write of x as keys and values under `slots`: what writing the token runs `written` (first token, first slot,
    tokens; each within a page) one by one gives, and nothing else changes."""
    kc, ks, vc, vs = cache
    page = kc.shape[2]
    k, v = (_host(kc), _host(ks)), (_host(vc).transpose(0, 1, 3, 2).copy(), _host(vs))
    xh = _host(x)
    for t, slot, n in written:
        for data, scale in (k, v):
            R.write(xh[t:t + n], [0, n], range(slot, slot + n), data, scale, page)
    C.kv_write(x, x, _ints(cu), _ints(slots), *cache)
    for got, want in ((kc, k[0]), (ks, k[1]), (vc, v[0].transpose(0, 1, 3, 2)), (vs, v[1])):
        np.testing.assert_array_equal(_host(got), want)


@pytest.mark.parametrize("hd,kv", [(64, 2), (128, 1), (256, 1)])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_write_behind_pages_that_are_not_there(hd, kv, page):
    """A request whose first pages have numbers outside of the cache: its later tokens go where their slots say."""
    rng = np.random.default_rng(page + hd)
    for past, ids in ((0, [-1, 2]), (5, [-1, 3, -1, 1]), (page - 1, [-1, -1, 0, 2]), (0, [-1, -1, -1, 3]), (0, [1, -1, 2]),
                      (3, [-1, -1])):
        for n in (len(ids) * page - past, len(ids) * page - past - page + 1):
            own = [ids[(past + t) // page] for t in range(n)]
            slots = [-1 if i < 0 else i * page + (past + t) % page for t, i in enumerate(own)]
            # two more requests around it, so that its tokens and pages do not begin at 0
            slots = [4 * page, 4 * page + 1] + slots + [5 * page + 7]
            written, t = [(0, 4 * page, 2), (2 + n, 5 * page + 7, 1)], 0
            while t < n:
                run = min(n - t, page - (past + t) % page)
                if own[t] >= 0:
                    written.append((2 + t, slots[2 + t], run))
                t += run
            x = _rows(rng, (n + 3, kv, hd), torch.float16)
            _check_only(x, [0, 2, 2 + n, 3 + n], slots, written, _cache(rng, 6, kv, hd, page))


def test_plan_write_and_attention_behind_a_page_that_is_not_there():
    """The free list begins with a page outside of the cache: the plan gives its tokens no slots, the writer fills the
    request's other page, and the attention sees that page alone."""
    rng = np.random.default_rng(3)
    hd, page = 64, 16
    cache = _cache(rng, 4, 1, hd, page)
    table = torch.full((1, 2), -1, dtype=torch.int32, device="cuda")
    plan = C.kv_plan(_ints([0]), _ints([32]), table, _ints([99, 2]), num_pages=4, page_size=page, tokens=32)
    assert plan.slot_map.numpy().tolist() == [-1] * 16 + list(range(32, 48)) and plan.kv_lens.numpy().tolist() == [32]
    x = _rows(rng, (32, 1, hd), torch.float16, 0.5)
    _check_only(x, [0, 32], plan.slot_map.numpy().tolist(), [(16, 32, 16)], cache)
    q = _rows(rng, (32, 2, hd), torch.float16, 0.5)
    want, tol = _want_cached(q, [0, 32], [32], table.cpu().numpy(), cache, True, hd ** -0.5)
    _check(q, [0, 32], [32], table.cpu().numpy(), cache, True, want, tol)
    assert (want[:16] == 0).all() and (want[16:] != 0).all()


@pytest.mark.parametrize("hd", [64, 256])
def test_write_keeps_nan_codes_of_a_page_that_grows(hd):
    """NaN codes among the tokens that a page keeps stay NaN when its scale grows, and do not raise it."""
    rng = np.random.default_rng(hd)
    page = 32
    kc, ks, vc, vs = _cache(rng, 3, 2, hd, page)
    kr, vr = kc.view(torch.uint8), vc.view(torch.uint8)
    kr[1, 0, 3, 5], kr[1, 1, 6, hd - 1], kr[1, 0, 20, 2] = 0x7f, 0xff, 0x7f    # the last one behind the new tokens
    vr[1, 0, 5, 3], vr[1, 1, hd - 1, 6], vr[1, 0, 2, 20] = 0xff, 0x7f, 0xff
    for size in (1.0, 1e4):                                                    # the second grows the page
        x = _rows(rng, (9, 2, hd), torch.float32) * size
        _check_only(x, [0, 9], range(page + 7, page + 16), [(0, page + 7, 9)], (kc, ks, vc, vs))
    assert int(torch.isnan(kc.float()).sum()) == 3 and int(torch.isnan(vc.float()).sum()) == 3


# ---- plan ------------------------------------------------------------------------------------------


def test_plans_in_turn():
    """A plan's kv_lens as the next step's past_lens: into another plan, not over itself."""
    lens, page, free = [15, 16, 40], 16, _ints(range(20))
    table = torch.full((3, 8), -1, dtype=torch.int32, device="cuda")
    cache = C.PagedKVCache(20, page, 1, 64)
    plan = cache.plan(_ints([0, 0, 0]), _ints(lens), table, free, sum(lens))
    used, new = int(plan.status.numpy()[0]), _ints([1, 1, 1])
    plans = [C.KVPlan(*(torch.zeros(n, dtype=torch.int32, device="cuda") for n in (4, 3, 3, 2))) for _ in range(2)]
    past = plan.kv_lens.torch
    for i in range(18):
        at = plans[i & 1]
        cache.plan(past, new, table, free[used:], 3, out=at)
        past, lens = at.kv_lens, [n + 1 for n in lens]
        with pytest.raises(N.MlcvError, match="overlap"):
            cache.plan(past, new, table, free[used:], 3, out=at)
        used += int(at.status[0])
        assert past.tolist() == lens and int(at.status[1]) == 0
        want = [int(table[b, (n - 1) // page]) * page + (n - 1) % page for b, n in enumerate(lens)]
        assert at.slot_map.tolist() == want and min(want) >= 0


# ---- attention over the cache: every form of the kernel -------------------------------------------------


def _plan(*sizes):
    s, w = ctypes.c_int32(), ctypes.c_int32()
    N.call("mlcv_kv_attention_plan", *sizes, ctypes.byref(s), ctypes.byref(w))
    return s.value, w.value


def _wanted(q, cu, lens, table, cache, causal):
    """_want_cached by matrix products, for many rows: (outputs, bounds, seen [tokens][n keys of the request])."""
    kc, ks, vc, vs = cache
    page, kv, hd = kc.shape[2], kc.shape[1], kc.shape[3]
    kf, vf = _host(kc) * _host(ks)[..., None, None], _host(vc).transpose(0, 1, 3, 2) * _host(vs)[..., None, None]
    qh, scale, grp = _host(q), hd ** -0.5, q.shape[1] // kv
    out, tol, seen = np.zeros(q.shape), np.zeros(q.shape), []
    tiny = 2.0 ** -37 * 448 * float(vs.max())
    for b, (a, z) in enumerate(zip(cu, cu[1:])):
        n, total = z - a, int(lens[b])
        ids = table[b][:-(-total // page)]
        there = np.array([0 <= ids[t // page] < kc.shape[0] for t in range(total)], bool)
        at = [(ids[t // page] if there[t] else 0, t % page) for t in range(total)]
        limit = np.array([total - n + i + 1 if causal else total for i in range(n)])
        see = (np.arange(total)[None, :] < limit[:, None]) & there[None, :]
        seen.append(see)
        for h in range(q.shape[1]):
            k, v = (np.array([x[p, h // grp, o] for p, o in at]).reshape(total, hd) for x in (kf, vf))
            k[~there], v[~there] = 0, 0
            with np.errstate(invalid="ignore"):
                x = np.where(see, qh[a:z, h] @ k.T * scale, -np.inf)
                p = np.where(see.any(1)[:, None], np.exp(x - x.max(1, keepdims=True, initial=-np.inf)), 0)
                p = np.where(see, p, 0) / np.maximum(p.sum(1, keepdims=True), 1e-300)
            o, mass = p @ v, p @ np.abs(v)
            big = np.where(see, np.abs(qh[a:z, h]) @ np.abs(k).T * scale, 0).max(1, initial=0)[:, None]
            out[a:z, h] = o
            tol[a:z, h] = R.bound(o, mass, big, q.dtype, max(int(there.sum()), 1), hd, torch.float16, tiny)
    return out, tol, seen


# new tokens of each request, their past, a bound on the lengths, and what the call is cut into
FORMS = {
    "four": ([50, 33, 0, 50, 1], [200, 250, 77, 0, 5], 300, (1, 4)),
    "eight": ([50, 33, 50, 0, 17, 50], [968, 700, 0, 903, 65, 400], 1018, (1, 8)),
    "few splits": ([1, 1, 2], [900, 1017, 63], 1018, None),
    "many splits": ([1, 2], [9000, 3000], 9001, None),
}


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("hd,page", [(64, 16), (64, 128), (128, 64), (128, 32), (256, 16), (256, 128)])
def test_kv_attention_every_form(form, dt, hd, page):
    """Four waves per workgroup and eight, no splits, up to 16 of them and more: lengths of every kind, a hole, page
    scales and codes that are not numbers in what no row sees, and then in what some do."""
    new, past, most, cut = FORMS[form]
    rng = np.random.default_rng(hd + page)
    lens, cu = [p + n for p, n in zip(past, new)], [0] + np.cumsum(new).tolist()
    splits, waves = _plan(cu[-1], len(new), 8, 1, hd, most)
    assert (splits, waves) == cut if cut else (waves == 4 and (splits > 16 if form == "many splits" else 1 < splits <= 16))
    table, (kc, ks, vc, vs), unused = _own_pages(rng, lens, 1, hd, page, 1 + -(-most // page))
    table[1, 1] = -1
    q = _rows(rng, (cu[-1], 8, hd), TYPES[dt], 0.5)
    kr, vr = kc.view(torch.uint8), vc.view(torch.uint8)
    want = {causal: _wanted(q, cu, lens, table, (kc, ks, vc, vs), causal) for causal in (True, False)}
    ks[unused], vs[unused] = float("nan"), float("inf")
    kr[unused], vr[unused] = 0x7f, 0xff
    for b, n in enumerate(lens):                          # behind each request's end, on its last page
        if n % page:
            kr[table[b, n // page], :, n % page:] = 0xff
            vr[table[b, n // page], :, :, n % page:] = 0x7f
    for causal in (True, False):
        _check(q, cu, lens, table, (kc, ks, vc, vs), causal, *want[causal][:2], max_kv=most)
    # values that rows see: the last key of request 0 (its last row's alone, if causal) and its first key
    for key, dim in ((lens[0] - 1, 3), (0, hd - 1)):
        vr[table[0, key // page], 0, dim, key % page] = 0x7f
        for causal in (True, False):
            got = C.kv_attention(q, _ints(cu), _ints(lens), torch.from_numpy(table).cuda(), kc, ks, vc, vs, causal=causal,
                                 max_kv=most)
            out, tol, seen = want[causal]
            bad = np.zeros(out.shape, bool)
            for k, d in ((lens[0] - 1, 3), (0, hd - 1)) if key == 0 else ((key, dim),):
                bad[:cu[1], :, d] |= seen[0][:, k][:, None]
            g = _host(got.torch)
            np.testing.assert_array_equal(np.isnan(g), bad)
            assert (np.abs(g - out)[~bad] <= tol[~bad]).all()


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,hd,page,past,new", [
    (4, 1, 64, 16, [1000, 300, 7], [64, 200, 130]),
    (8, 2, 128, 64, [1000, 0, 129], [65, 128, 257]),
    (8, 1, 256, 32, [2000, 63], [64, 100]),
    (6, 6, 128, 16, [15, 1], [513, 64]),
    (20, 1, 64, 128, [500], [300]),
])
def test_kv_attention_chunks(dt, heads, kv, hd, page, past, new):
    """64 and more new tokens of a request over its cached ones: a prompt that comes in pieces."""
    rng = np.random.default_rng(hd + page)
    lens, cu = [p + n for p, n in zip(past, new)], [0] + np.cumsum(new).tolist()
    table, cache, _ = _own_pages(rng, lens, kv, hd, page, 2 + -(-max(lens) // page))
    q = _rows(rng, (cu[-1], heads, hd), TYPES[dt], 0.5)
    for causal in (True, False):
        want, tol, _ = _wanted(q, cu, lens, table, cache, causal)
        for most in (max(lens), 1, 10 ** 6):
            _check(q, cu, lens, table, cache, causal, want, tol, max_kv=most)


def test_wanted_is_the_plain_form():
    """The products above against the rows one by one."""
    rng = np.random.default_rng(1)
    lens, cu = [40, 3, 70], [0, 5, 8, 9]
    table, cache, _ = _own_pages(rng, lens, 2, 64, 16, 6)
    table[2, 1] = -1
    q = _rows(rng, (9, 4, 64), torch.float16)
    for causal in (True, False):
        a, at = _want_cached(q, cu, lens, table, cache, causal, 64 ** -0.5)
        b, bt, _ = _wanted(q, cu, lens, table, cache, causal)
        np.testing.assert_allclose(b, a, rtol=1e-10, atol=1e-10)
        assert (bt >= at * (1 - 1e-9)).all()  # it counts every key of the request


def test_requests_of_sound_offsets_beside_others():
    """Offsets that descend or lie outside before and behind a request: its rows are what it alone gives, with splits of
    the keys and without, and its tokens are written; nothing around the outputs and the cache is."""
    rng = np.random.default_rng(17)
    n, hd, page = 300, 64, 16
    q, k, v = (_rows(rng, (n, h, hd), torch.float16, 0.5) for h in (2, 1, 1))
    table, cache, _ = _own_pages(rng, [500, 500, 500], 1, hd, page, 32)
    t = torch.from_numpy(table).cuda()
    cu, lens, own = [250, 100, 299, 10 ** 6], [400, 450, 3], slice(100, 299)
    store = torch.full((n + 64, 2, hd), 9.0, dtype=torch.float16, device="cuda")
    out = store[32:32 + n]
    C.prompt_attention(q, k, v, _ints(cu), out=out)
    assert torch.equal(out[own], C.prompt_attention(q[own], k[own], v[own], _ints([0, 199])).torch)
    assert (out[:100] == 9).all()
    for most in (1, 512, 10 ** 6):
        for causal in (True, False):
            out.fill_(9.0)
            C.kv_attention(q, _ints(cu), _ints(lens), t, *cache, out=out, max_kv=most, causal=causal)
            want, tol, _ = _wanted(q[own], [0, 199], lens[1:2], table[1:2], cache, causal)
            assert (np.abs(_host(out[own]) - want) <= tol).all()
            assert (out[:100] == 9).all()
    assert (store[:32] == 9).all() and (store[32 + n:] == 9).all()
    # the writer: request 1's tokens to pages of their own, and a guard on both sides of each cache
    whole = [torch.full((32 + 40 + 32,) + x.shape[1:], 3, dtype=torch.uint8, device="cuda").view(F8) if x.dtype == F8 else
             torch.full((32 + 40 + 32,) + x.shape[1:], 3.0, device="cuda") for x in cache]
    held = [x[32:72] for x in whole]
    slots = [-1] * 100 + [16 * 3 + 5 + i for i in range(199)] + [16 * 30]
    C.kv_write(k, v, _ints(cu), _ints(slots), *held)
    alone = [x.clone() for x in whole]
    for x in alone:
        (x.view(torch.uint8) if x.dtype == F8 else x).fill_(3)
    C.kv_write(k[own], v[own], _ints([0, 199]), _ints(slots[own]), *(x[32:72] for x in alone))
    C.kv_write(k[299:], v[299:], _ints([0, 1]), _ints(slots[299:]), *(x[32:72] for x in alone))
    for a, b in zip(whole, alone):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# ---- together ----------------------------------------------------------------------------------------


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_kv_attention_over_its_own_queries(form, hd):
    """out = q, as the documentation allows, in every form of the kernel."""
    new, past, most, _ = FORMS[form]
    rng = np.random.default_rng(hd)
    lens, cu = [p + n for p, n in zip(past, new)], [0] + np.cumsum(new).tolist()
    table, cache, _ = _own_pages(rng, lens, 1, hd, 64, 1 + -(-most // 64))
    wide = _rows(rng, (cu[-1], 12, hd), torch.float16, 0.5)
    args = (_ints(cu), _ints(lens), torch.from_numpy(table).cuda(), *cache)
    want = C.kv_attention(wide[:, 2:10], *args, max_kv=most).torch
    rest = wide[:, 10:].clone()
    q = wide[:, 2:10]                                    # a slice of wider rows
    assert torch.equal(C.kv_attention(q, *args, max_kv=most, out=q).torch, want) and torch.equal(q, want)
    assert torch.equal(wide[:, 10:], rest)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("heads", [4, 64])               # few rows: shared by two waves; many
def test_prompt_attention_over_its_own_queries(hd, heads):
    rng = np.random.default_rng(hd)
    lens = [1, 130, 200, 63]
    cu = _ints([0] + np.cumsum(lens).tolist())
    q, k, v = (_rows(rng, (sum(lens) + 2, h, hd), torch.bfloat16, 0.5) for h in (heads, 2, 2))
    want, rest = C.prompt_attention(q, k, v, cu).torch[:-2], q[-2:].clone()
    assert torch.equal(C.prompt_attention(q, k, v, cu, out=q).torch[:-2], want) and torch.equal(q[-2:], rest)


def test_captured_step_whose_lengths_grow():
    """One graph of a decode step, replayed as its requests grow over page ends: the lengths, the table and the list of
    free pages stay on the device and are the next replay's; every replay against eager calls on caches of their own."""
    g = torch.Generator(device="cuda").manual_seed(5)
    page, kv, heads, hd, lens = 16, 2, 8, 64, [30, 1, 47]
    rand = lambda n, h: torch.randn((n, h, hd), generator=g, device="cuda").half()  # noqa: E731
    caches = [C.PagedKVCache(40, page, kv, hd) for _ in range(2)]
    tables = [torch.full((3, 8), -1, dtype=torch.int32, device="cuda") for _ in range(2)]
    free, new, past = _ints(range(39, -1, -1)), _ints([1, 1, 1]), _ints(lens)
    k, v = rand(sum(lens), kv), rand(sum(lens), kv)
    for cache, table in zip(caches, tables):
        plan = cache.plan(_ints([0, 0, 0]), past, table, free, sum(lens))
        cache.write(k, v, plan)
    used = int(plan.status.numpy()[0])
    left = torch.cat([free[used:], free[:used]])          # the list that the graph takes pages from the front of
    at = torch.arange(left.numel(), device="cuda")
    q, k, v = rand(3, heads), rand(3, kv), rand(3, kv)

    def step(cache, table, past, left):
        plan = cache.plan(past, new, table, left, 3)
        cache.write(k, v, plan)
        return plan, cache.attention(q, plan, table).torch

    spare = [t.clone() for t in (caches[0].k.view(torch.uint8), caches[0].v.view(torch.uint8), caches[0].k_scale,
                                 caches[0].v_scale, tables[0])]
    step(caches[0], tables[0], past, left)                # as a capture asks for; then back
    for a, b in zip((caches[0].k.view(torch.uint8), caches[0].v.view(torch.uint8), caches[0].k_scale, caches[0].v_scale,
                     tables[0]), spare):
        a.copy_(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, out = step(caches[0], tables[0], past, left)
        past.copy_(plan.kv_lens.torch)
        left.copy_(left[(at + plan.status.torch[:1]) % left.numel()])
    own_past, own_left = past.clone(), left.clone()
    for i in range(40):
        for x in (q, k, v):
            x.copy_(rand(3, x.shape[1]))
        want_plan, want = step(caches[1], tables[1], own_past, own_left)
        own_past, own_left = want_plan.kv_lens.torch, own_left.roll(-int(want_plan.status.torch[0]))
        graph.replay()
        torch.cuda.synchronize()
        assert past.tolist() == [n + i + 1 for n in lens] and want_plan.status.torch[1] == 0
        assert torch.equal(out, want) and torch.equal(tables[0], tables[1]) and torch.equal(left, own_left)
        for a, b in zip(caches[0].pages(), caches[1].pages()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
