"""Pages of the cache that change hands, on the GPU (mlc_vla.kv_cache): free, fork, compact, copy, and plans over a
counted free list, against plain implementations (stepref.py); bytes and numbers have to be equal."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import kvref as R
import stepref as S
from mlc_vla import _native as N
from mlc_vla import kv_cache as C

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def _named(request):
    print(request.node.name, flush=True)


def _ints(v):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(v, np.int32))).cuda()


def _pool(rng, layers, pages, kv, page, hd):
    """Any bytes, NaN codes too: pages are copied as they are."""
    raw = [torch.from_numpy(rng.integers(0, 256, s, dtype=np.uint8)).cuda().view(F8)
           for s in ((layers, pages, kv, page, hd), (layers, pages, kv, hd, page))]
    scale = [torch.from_numpy(rng.standard_normal((layers, pages, kv)).astype(np.float32)).cuda() for _ in range(2)]
    return raw[0], scale[0], raw[1], scale[1]


def _bytes(cache):
    return [t.view(torch.uint8).cpu().numpy().copy() if t.dtype == F8 else t.cpu().numpy().copy() for t in cache]


def _moved(before, pairs):
    """The pool's bytes after copying all pairs at once."""
    out = [x.copy() for x in before]
    if pairs:
        src, dst = (np.array(x) for x in zip(*pairs))
        for x, y in zip(out, before):
            x[:, dst] = y[:, src]
    return out


def _same(cache, want):
    for got, w in zip(_bytes(cache), want):
        np.testing.assert_array_equal(got, w)


def _requests(rng, b, most, page, pages, wide=None, shared=True):
    """A table of b requests over a pool, some sharing pages, and their lengths."""
    lens = rng.integers(0, most + 1, b)
    need = -(-lens // page)
    wide = int(need.max(initial=0)) + 1 if wide is None else wide
    table = rng.integers(-3, pages + 3, (b, wide))  # entries not in use may hold anything
    order = rng.permutation(pages)
    at = 0
    for i in range(b):
        s = int(min(need[i], need[i - 1]) // 2) if shared and i % 3 == 2 else 0
        table[i, :s] = table[i - 1, :s]
        table[i, s:need[i]] = order[at:at + need[i] - s]
        at += need[i] - s
    assert at <= pages
    return table, lens


# ---- free --------------------------------------------------------------------------------------------


def _check_free(table, lens, pages, page):
    want, n = S.free(table, lens, pages, page)
    got = C.kv_free(_ints(table), _ints(lens), num_pages=pages, page_size=page)
    assert got.free_count.numpy().tolist() == [n]
    np.testing.assert_array_equal(got.free_pages.numpy(), want)


@pytest.mark.parametrize("b,most,page,pages", [
    (1, 1, 16, 1), (3, 100, 16, 30), (16, 1168, 64, 1024), (5, 300, 128, 64), (7, 2000, 32, 4095), (9, 1000, 16, 4096),
    (64, 1000, 16, 4097), (300, 500, 16, 12000), (4096, 33, 16, 70001), (2, 131072, 64, 300000)])
def test_free(b, most, page, pages):
    rng = np.random.default_rng(pages)
    table, lens = _requests(rng, b, most, page, pages)
    _check_free(table, lens, pages, page)


def test_free_of_a_pool_of_many_slices():
    """Over 1024 * 4096 pages a workgroup marks more than one block of them."""
    rng = np.random.default_rng(0)
    pages = 2 ** 23 + 77
    table = rng.integers(0, pages, (50, 300))
    table[3, :5] = [0, pages - 1, 4095, 4096, 8191]
    _check_free(table, np.full(50, 300 * 16), pages, 16)


def test_free_lengths_and_numbers_out_of_range():
    rng = np.random.default_rng(1)
    table = rng.integers(-5, 50, (6, 8))
    table[0, 0], table[1, 1] = 2 ** 31 - 1, -2 ** 31
    _check_free(table, np.array([-3, 10 ** 9, 128, 0, 2 ** 31 - 1, -2 ** 31]), 40, 16)
    _check_free(table, np.full(6, 128), 40, 16)


def test_free_without_requests_pages_or_entries():
    t = torch.empty((0, 4), dtype=torch.int32, device="cuda")
    got = C.kv_free(t, _ints([]), num_pages=5, page_size=16)
    assert got.free_pages.numpy().tolist() == [0, 1, 2, 3, 4] and got.free_count.numpy().tolist() == [5]
    got = C.kv_free(_ints([[1, 2]]), _ints([20]), num_pages=0, page_size=16)
    assert got.free_count.numpy().tolist() == [0] and got.free_pages.shape == (0,)
    got = C.kv_free(torch.empty((2, 0), dtype=torch.int32, device="cuda"), _ints([9, 9]), num_pages=3, page_size=16)
    assert got.free_pages.numpy().tolist() == [0, 1, 2]


@pytest.mark.parametrize("count", [0, 1, 5, 9, 12, 99, -4])
def test_plan_over_a_counted_free_list(count):
    """As if the list ended there; counts outside of it are brought into range."""
    rng = np.random.default_rng(count + 9)
    page, past, new = 16, np.array([3, 16, 0, 40]), np.array([30, 1, 20, 3])
    table = np.full((4, 6), -1)
    table[0, 0], table[1, 0], table[3, :3] = 20, 21, [22, 23, 24]
    free = rng.permutation(12)
    tokens = int(new.sum())
    want_table = table.copy()
    want = R.plan(past, new, want_table, free[:max(0, min(count, 12))], 30, page, tokens)
    t = _ints(table)
    got = C.kv_plan(_ints(past), _ints(new), t, _ints(free), num_pages=30, page_size=page, tokens=tokens,
                    free_count=_ints([count]))
    for name, x, w in zip(got._fields, got, want):
        np.testing.assert_array_equal(x.numpy(), w, err_msg=name)
    np.testing.assert_array_equal(t.cpu().numpy(), want_table)


# ---- copy --------------------------------------------------------------------------------------------


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("hd,kv,layers", [(64, 1, 3), (128, 3, 2), (256, 1, 18), (64, 130, 1), (256, 9, 1)])
def test_copy(page, hd, kv, layers):
    rng = np.random.default_rng(page + hd)
    pages, n = 13, 5
    cache = _pool(rng, layers, pages, kv, page, hd)
    before, order = _bytes(cache), rng.permutation(pages)
    C.kv_copy(_ints(order[:n]), _ints(order[n:2 * n]), *cache)
    _same(cache, _moved(before, list(zip(order[:n], order[n:2 * n]))))
    # into another pool; a page may be read twice; numbers outside of either pool are passed over
    before, into = _bytes(cache), _pool(rng, layers, 7, kv, page, hd)
    want = _bytes(into)
    C.kv_copy(_ints([3, 3, 12, -1, 13, 0, 1]), _ints([6, 0, 2, 3, 4, 7, -2]), *cache, into=into)
    for w, x in zip(want, before):
        w[:, [6, 0, 2]] = x[:, [3, 3, 12]]
    _same(into, want)
    _same(cache, before)


def test_copy_of_one_layer_and_of_nothing():
    rng = np.random.default_rng(2)
    cache = _pool(rng, 3, 6, 2, 16, 64)
    before = _bytes(cache)
    C.kv_copy(_ints([4]), _ints([1]), *(t[1] for t in cache))
    want = [x.copy() for x in before]
    for w in want:
        w[1, 1] = w[1, 4]
    _same(cache, want)
    C.kv_copy(_ints([]), _ints([]), *cache)
    _same(cache, want)
    mine, more = C.PagedKVCache(4, 32, 2, 64, layers=2), C.PagedKVCache(9, 32, 2, 64, layers=2)
    mine.k.view(torch.uint8).fill_(7)
    mine.v_scale.fill_(2.0)
    mine.copy(_ints([0, 1, 2, 3]), _ints([5, 6, 7, 8]), into=more)
    assert (more.k.view(torch.uint8)[:, 5:] == 7).all() and (more.k.view(torch.uint8)[:, :5] == 0).all()
    assert (more.v_scale[:, 5:] == 2).all() and (more.v_scale[:, :5] == 0).all()


def test_copy_past_32_bit_offsets():
    pages, kv, page, hd = 2 ** 17 + 3, 2, 128, 256  # 8.6 GB a side
    k = torch.zeros((1, pages, kv, page, hd), dtype=torch.uint8, device="cuda")
    v = torch.zeros((1, pages, kv, hd, page), dtype=torch.uint8, device="cuda")
    ks, vs = (torch.zeros((1, pages, kv), device="cuda") for _ in range(2))
    k[0, -1], v[0, -1], ks[0, -1], vs[0, -2] = 5, 6, 3.0, 4.0
    k[0, 70000] = 9
    C.kv_copy(_ints([pages - 1, 70000]), _ints([1, pages - 2]), k.view(F8), ks, v.view(F8), vs)
    assert (k[0, 1] == 5).all() and (v[0, 1] == 6).all() and (ks[0, 1] == 3).all() and (k[0, pages - 2] == 9).all()
    assert (vs[0, pages - 2] == 0).all() and (k[0, 0] == 0).all() and (k[0, 2] == 0).all()
    del k, v
    torch.cuda.empty_cache()


# ---- fork --------------------------------------------------------------------------------------------


def _check_fork(rng, parents, table, lens, free, pages, page, kv=1, hd=64, layers=2, count=None):
    want_table, want_lens, status, pairs = S.fork(parents, table, lens, free if count is None else free[:count], page)
    cache = _pool(rng, layers, pages, kv, page, hd)
    before = _bytes(cache)
    old = _ints(table)
    got = C.kv_fork(_ints(parents), old, _ints(lens), _ints(free), *cache,
                    free_count=None if count is None else _ints([count]))
    np.testing.assert_array_equal(got.block_table.numpy(), want_table)
    np.testing.assert_array_equal(got.kv_lens.numpy(), want_lens)
    np.testing.assert_array_equal(got.status.numpy(), status)
    np.testing.assert_array_equal(old.cpu().numpy(), table)
    _same(cache, _moved(before, [p for p in pairs if 0 <= p[0] < pages and 0 <= p[1] < pages]))


@pytest.mark.parametrize("b,n,most,page", [(1, 1, 40, 16), (1, 8, 100, 64), (4, 16, 1168, 64), (7, 3, 50, 128), (3, 300, 70, 16),
                                           (64, 512, 300, 32), (300, 299, 64, 16)])
def test_fork(b, n, most, page):
    rng = np.random.default_rng(b + n)
    pages = int(b * (most // page + 1)) + n + 3
    table, lens = _requests(rng, b, most, page, pages - n, shared=False)
    used, _ = S.used_pages(table, lens, pages, page)
    free = rng.permutation(np.setdiff1d(np.arange(pages), used))
    _check_fork(rng, rng.integers(-1, b + 1, n), table, lens, free, pages, page)
    _check_fork(rng, rng.integers(0, b, n), table, lens, free, pages, page, kv=3, hd=128, layers=1)


@pytest.mark.parametrize("count", [0, 1, 3, 4, 5, 50, None])
def test_fork_where_the_free_pages_do_not_last(count):
    """The rows behind are refused; those that need no page are not."""
    rng = np.random.default_rng(5)
    table, lens = np.array([[3, 4, 9], [5, 6, 9], [7, 9, 9]]), np.array([20, 32, 5])
    _check_fork(rng, [0, 1, 2, 0, 1, 2, 0, 1, -1, 3, 2, 0], table, lens, np.array([12, 10, 11, 13, 8]), 16, 16, count=count)


def test_fork_odd_arguments():
    """Lengths outside of the table, page numbers outside of the pool, no rows, no pages, the same row many times."""
    rng = np.random.default_rng(6)
    table = np.array([[3, 4], [-1, 20], [7, 40]])
    _check_fork(rng, [0, 0, 1, 1, 2, 2, 2], table, np.array([10 ** 9, 17, 20]), np.array([12, 50, 10, -3, 8]), 16, 16)
    _check_fork(rng, [0, 0, 1, 2], table, np.array([-5, 0, 16]), np.array([12]), 16, 16)
    _check_fork(rng, [], table, np.array([20, 17, 20]), np.array([12]), 16, 16)
    _check_fork(rng, [0, 0], table, np.array([20, 17, 20]), np.zeros(0, int), 16, 16)
    _check_fork(rng, [1, 0], np.zeros((0, 2), int), np.zeros(0, int), np.array([3]), 16, 16)
    _check_fork(rng, [2] * 4096, table, np.array([20, 17, 20]), np.arange(100, 5000), 5000, 16)


# ---- compact -----------------------------------------------------------------------------------------


def _check_compact(rng, table, lens, pages, page, kv=1, hd=64, layers=2, place=False):
    want, status, pairs = S.compact(table, lens, pages, page)
    cache = _pool(rng, layers, pages, kv, page, hd)
    before, t = _bytes(cache), _ints(table)
    out = C.KVCompact(t, torch.zeros(2, dtype=torch.int32, device="cuda")) if place else None
    got = C.kv_compact(t, _ints(lens), *cache, out=out)
    new = t if place else got.block_table.torch
    np.testing.assert_array_equal(new.cpu().numpy(), want)
    np.testing.assert_array_equal(C._t(got.status).cpu().numpy(), status)
    if not place:
        np.testing.assert_array_equal(t.cpu().numpy(), table)
    _same(cache, _moved(before, pairs))


@pytest.mark.parametrize("b,most,page,pages,hd,kv", [
    (1, 1, 16, 1, 64, 1), (2, 40, 16, 9, 64, 1), (16, 300, 16, 512, 256, 1), (5, 300, 128, 64, 128, 3), (40, 90, 32, 400, 64, 2),
    (64, 900, 16, 4096, 64, 1), (300, 300, 16, 9001, 64, 1), (17, 4000, 64, 20000, 64, 1), (200, 60, 16, 900, 64, 1), (3, 14000, 16, 3000, 64, 1)])
@pytest.mark.parametrize("place", [False, True])
def test_compact(b, most, page, pages, hd, kv, place):
    rng = np.random.default_rng(pages + b)
    table, lens = _requests(rng, b, most, page, pages)
    _check_compact(rng, table, lens, pages, page, kv, hd, 1 if pages > 4096 else 3, place)


def test_compact_full_empty_and_dense():
    rng = np.random.default_rng(8)
    _check_compact(rng, rng.permutation(4096).reshape(8, 512), np.full(8, 512 * 16), 4096, 16, layers=1)  # all in use
    _check_compact(rng, rng.permutation(50)[None], np.zeros(1, int), 50, 16)                               # none
    _check_compact(rng, np.arange(20)[None], np.array([20 * 16]), 50, 16)                                  # dense already
    _check_compact(rng, 30 + np.arange(20)[None], np.array([20 * 16 - 3]), 50, 16)                         # all move
    _check_compact(rng, np.zeros((0, 3), int), np.zeros(0, int), 50, 16)
    _check_compact(rng, np.array([[-1, 60, 49, 7], [49, 2 ** 31 - 1, 3, 0]]), np.array([10 ** 9, 48]), 50, 16)  # odd numbers
    _check_compact(rng, np.concatenate([np.arange(4096), [8191]])[None], np.array([4097 * 16]), 8192, 16, layers=1)


def test_a_compacted_pool_serves_as_before():
    """Attention over the cache before and after, bit for bit, and the free list behind the dense part."""
    rng = np.random.default_rng(9)
    cache = C.PagedKVCache(40, 16, 2, 64)
    table, lens = _requests(rng, 4, 100, 16, 40, wide=8)
    lens[0] = 100
    table[0, :7] = np.setdiff1d(np.arange(40), S.used_pages(table[1:], lens[1:], 40, 16)[0])[:7]
    cache.k.view(torch.uint8).copy_(torch.from_numpy(rng.integers(0, 126, cache.k.shape, dtype=np.uint8)))
    cache.v.view(torch.uint8).copy_(torch.from_numpy(rng.integers(0, 126, cache.v.shape, dtype=np.uint8)))
    cache.k_scale.fill_(2.0 ** -9)
    cache.v_scale.copy_(torch.rand(cache.v_scale.shape))
    t, m = _ints(np.clip(table, 0, 39)), _ints(lens)
    q = torch.randn((4, 4, 64), device="cuda").half()
    plan = C.KVPlan(_ints(range(5)), m, _ints([0] * 4), _ints([0, 0]))
    want = cache.attention(q, plan, t).torch
    got = cache.compact(t, m)
    assert torch.equal(cache.attention(q, plan, got.block_table).torch, want)
    n = int(got.status.numpy()[0])
    free = cache.free(got.block_table, m)
    assert free.free_count.numpy().tolist() == [40 - n]
    assert free.free_pages.numpy().tolist() == list(range(n, 40)) + [-1] * n


def test_page_arguments():
    rng = np.random.default_rng(10)
    cache = _pool(rng, 2, 8, 1, 16, 64)
    t, m, p, f = _ints([[1, 2], [3, 4]]), _ints([20, 32]), _ints([0, 0, 1]), _ints([5, 6, 7])
    k, ks, v, vs = cache
    one = tuple(x[0] for x in cache)
    made = C.kv_fork(p, t, m, f, *cache)
    small = torch.zeros(16, dtype=torch.uint8, device="cuda")
    for fn, args, kw, what in (
            (C.kv_free, (t, m), dict(num_pages=-1, page_size=16), "num_pages"),
            (C.kv_free, (t[0], m), dict(num_pages=8, page_size=16), "block_table expects"),
            (C.kv_free, (t, m[:1]), dict(num_pages=8, page_size=16), "kv_lens expects"),
            (C.kv_free, (t.long(), m), dict(num_pages=8, page_size=16), "block_table has dtype"),
            (C.kv_free, (t[:, ::2], m), dict(num_pages=8, page_size=16), "contiguous"),
            (C.kv_free, (t, m.cpu()), dict(num_pages=8, page_size=16), "kv_lens is not on"),
            (C.kv_free, (t, m), dict(num_pages=8, page_size=16, out=C.KVFree(f, _ints([0]))), "out.free_pages expects"),
            (C.kv_free, (t, m), dict(num_pages=8, page_size=16, workspace=m), "workspace has dtype"),
            (C.kv_copy, (p, f[:2], *cache), {}, "dst expects"), (C.kv_copy, (p.long(), f, *cache), {}, "src has dtype"),
            (C.kv_copy, (p, f, k, ks, v, vs[0]), {}, "v_scale expects"), (C.kv_copy, (p, f, k, ks, k, vs), {}, "v_cache expects"),
            (C.kv_copy, (p, f, k.view(torch.uint8), ks, v, vs), {}, "k_cache has dtype"),
            (C.kv_copy, (p, f, k[:, ::2], ks[:, ::2], v[:, ::2], vs[:, ::2]), {}, "contiguous"),
            (C.kv_copy, (p, f, k[0, 0], ks, v, vs), {}, "k_cache expects"),
            (C.kv_copy, (p, f, *cache), dict(into=one), "other layers"),
            (C.kv_fork, (p[None], t, m, f, *cache), {}, "parents expects"),
            (C.kv_fork, (p, t, m, f.long(), *cache), {}, "free_pages has dtype"),
            (C.kv_fork, (p, t, m, f, *cache), dict(free_count=m), "free_count expects"),
            (C.kv_fork, (p[:2], t, m, f, *cache), dict(out=made), "out.block_table expects"),
            (C.kv_plan, (m, m, t, f), dict(num_pages=8, page_size=16, tokens=9, free_count=3), "tensor"),
            (C.kv_compact, (t, m, *cache), dict(out=C.KVCompact(t, m[:1])), "out.status expects")):
        with pytest.raises((ValueError, TypeError), match=what):
            fn(*args, **kw)
    for fn, args, kw, what in (
            (C.kv_free, (t, m), dict(num_pages=8, page_size=24), "page must"),
            (C.kv_free, (t, m), dict(num_pages=8, page_size=16, workspace=small), "workspace"),
            (C.kv_compact, (t, m, *cache), dict(workspace=small), "workspace"),
            (C.kv_fork, (p, t, m, f, *cache), dict(out=C.KVFork(made.block_table, p, made.status)), "overlap"),
            (C.kv_compact, (t, m, *cache), dict(out=C.KVCompact(t, m)), "overlap")):
        with pytest.raises(N.MlcvError, match=what):
            fn(*args, **kw)
