"""The request entry points where their inputs touch what is not theirs: pages that no request uses, page numbers that
are not there.  Plain 64-bit forms and bounds as in test_gpu_kv_cache.py."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import kvref as R
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
