"""The operators around a decode step's attention where their ordinary tests do not reach: masks of every finite size, scaled
logits past 2^31, rows that are almost certain, against plain implementations in 64 bits (stepref.py)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import stepref as S
from mlc_vla import _native as N
from mlc_vla import kv_cache as C
from mlc_vla import logits as L
from test_gpu_request_step import _check_logprobs, _check_rope, _host, _tokens

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(autouse=True)
def _named(request):
    print(request.node.name, flush=True)


def _ints(v):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(v, np.int32))).cuda()


# ---- log probabilities: finite masks and large logits ------------------------------------------------------


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("mask", [-1e9, -1e10, -1e12, -1e20, -1e30, -1e35])
def test_token_logprobs_finite_masks(dt, mask):
    """Masks that cover a wave's first round, all of a wave, a split, a row; scores, no and many alternatives, four waves for
    a row and one."""
    rng = np.random.default_rng(int(-np.log10(-mask)) % 97)
    for rows, vocab in ((7, 16384), (7, 40000), (1000, 4000)):
        x = rng.standard_normal((rows, vocab)) * 2
        x[0, 40:] = mask                      # only the first wave of the first split meets anything else
        x[1, :vocab - 40] = mask              # only the last does, and late
        x[2] = mask                           # nothing is left: uniform
        x[3, 512:2048] = mask                 # other waves' first rounds
        x[4, rng.random(vocab) < 0.999] = mask
        x[5, vocab // 2:] = -np.inf           # beside masks of -inf
        x[5, :vocab // 2 - 3] = mask
        x = torch.from_numpy(x).to(TYPES[dt]).cuda()
        for scale in ((0.5, 1.0, 4.0) if rows < 10 else (1.0,)):
            for top in (0, 20) if rows < 10 else (20,):
                _check_logprobs(x, scale, _tokens(rng, rows, 2, vocab), top)


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("scale", [1e3, 1e6])
def test_token_logprobs_of_large_scaled_logits(dt, scale):
    """Logits around 1e3 and 1e4 of either sign at the smallest temperatures."""
    rng = np.random.default_rng(int(scale) % 1009)
    for vocab in (1500, 9001, 30000):
        x = rng.standard_normal((6, vocab))
        x[:2] += 3000
        x[2:4] -= 12000
        x[4] = -12000
        x[5] = 20000
        _check_logprobs(torch.from_numpy(x).to(TYPES[dt]).cuda(), scale, _tokens(rng, 6, 2, vocab), 9)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [1.0, 4.0])
def test_token_logprobs_of_rising_maxima(dt, scale):
    """A row's largest logit grows from round to round through every size up to the type's largest."""
    vocab = 30000
    up = np.linspace(90, 127.9, vocab)
    x = np.stack([2.0 ** up, -2.0 ** up[::-1], 2.0 ** np.linspace(118, 122, vocab), 2.0 ** np.linspace(20, 40, vocab),
                  np.where(np.arange(vocab) < vocab // 2, -2.0 ** 127, 2.0 ** 127)])
    _check_logprobs(torch.from_numpy(x).to(TYPES[dt]).cuda(), scale, _tokens(np.random.default_rng(1), 5, 2, vocab), 5)


@pytest.mark.parametrize("vocab", [1000, 5000, 40000])
def test_token_logprobs_keep_the_entropy_of_certain_rows(vocab):
    """One other logit of probability t: the entropy is ln(1 + t) + t / (1 + t) ln(1 / t).
    1 + t as float32 is off by at most t and by at most half a step, 2^-24: so is its logarithm.  The other sum has one term but
    zeros: the difference, the scale, their product, the exponential (of an argument of up to 48, each of three roundings
    counts 48 half steps), and where it is rebased the same again; the logarithm and the sums 16 half steps."""
    gaps = np.array([0.5, 1.0, 3.0, 8.0, 12.0, 15.0, 17.0, 18.0, 20.0, 24.0, 28.0, 33.0])
    rel = (2 * 3 * 48 + 16) * S.E32
    for at, other in ((17, 18), (17, 17 + 512 % (vocab - 30)), (vocab - 1, 3), (2, vocab - 1), (600, 80)):
        for top in (1.977, 30.0, -5e3, 1e6):
            x = np.full((len(gaps), vocab), -np.inf, np.float32)
            x[:, at] = top
            x[:, other] = np.float32(top) - gaps.astype(np.float32)
            d = x[:, at].astype(np.float64) - x[:, other]  # what float32 holds
            t = np.exp(-d)
            want = np.log1p(t) + t / (1 + t) * d
            got = L.token_logprobs(torch.from_numpy(x).cuda(), _ints([at] * len(gaps)), top=1)
            h, lp = _host(got.entropy.torch), _host(got.logprobs.torch)
            ends = 1.01 * np.minimum(t, S.E32)
            assert (h >= 0).all() and (np.abs(h - want) <= ends + rel * want).all(), (at, other, top, h, want)
            assert (lp <= 0).all() and (np.abs(lp + np.log1p(t)) <= ends + rel * np.log1p(t)).all()


def test_token_logprobs_entropy_is_not_negative():
    """Rows of one token that nothing else comes near, at many sizes of the largest logit."""
    rng = np.random.default_rng(2)
    x = np.full((400, 3000), -np.inf, np.float32)
    top = np.linspace(1, 40, 400)
    x[np.arange(400), rng.integers(0, 1500, 400)] = top
    x[np.arange(400), rng.integers(1500, 3000, 400)] = top - rng.uniform(17, 50, 400)
    for scale in (0.7, 1.0, 1.3):
        h = L.token_logprobs(torch.from_numpy(x).cuda(), scale=scale).entropy.torch
        assert (h >= 0).all() and (h < 1e-4).all()


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
def test_token_logprobs_order_beside_nan(dt):
    """Quiet and signalling NaN next to the largest logits: the alternatives are the numbers, in their order."""
    rng = np.random.default_rng(5)
    bits = {"f16": (np.uint16, 0x7e00, 0x7c01), "bf16": (np.uint16, 0x7fc0, 0x7f81), "f32": (np.uint32, 0x7fc00000, 0x7f800001)}
    kind, quiet, loud = bits[dt]
    for vocab in (1500, 9001, 40000):
        x = torch.from_numpy(rng.standard_normal((6, vocab)) * 3).to(TYPES[dt])
        raw = x.view(torch.int16 if dt != "f32" else torch.int32).numpy().view(kind)
        best = _host(x).argsort(1)[:, -30:]
        for r, nan in ((0, quiet), (1, loud)):
            near = (best[r][:, None] // 8 * 8 + np.arange(8)).ravel()  # the eight logits that a lane takes at once
            raw[r, [i for i in near if i < vocab and i not in best[r]]] = nan
            raw[2 + r, rng.random(vocab) < 0.3] = nan
            raw[4 + r, rng.integers(0, vocab)] = nan
        for top in (1, 20, 64):
            _check_logprobs(x.cuda(), 1.0, _tokens(rng, 6, 2, vocab), top)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [1e-6, 1e-3, 0.25, 0.5, 1.0])
def test_token_logprobs_of_the_largest_distances(dt, scale):
    """Logits further apart than the largest float32, whose log probabilities are within it, or just past it."""
    for vocab in (100, 9001):
        x = np.full((3, vocab), -3.2e38)
        x[0, 7], x[1, ::3], x[2, 50:] = 3e38, 2.1e38, -1e38
        ids = torch.tensor([[0, 7], [1, 3], [3, 60]], dtype=torch.int32, device="cuda")
        _check_logprobs(torch.from_numpy(x).to(TYPES[dt]).cuda(), scale, ids, 60)


def test_token_logprobs_within_one_buffer():
    """Results in a padded vocabulary's padding are taken, results over the logits are not."""
    rng = np.random.default_rng(6)
    x = torch.from_numpy(rng.standard_normal((5, 600))).float().cuda()
    pad = x.view(torch.int32)
    tokens = _tokens(rng, 5, 1, 500)
    want = L.token_logprobs(x[:, :500], tokens, top=4)
    given = L.TokenLogprobs(x[4, 500:505], x[0, 520:525], pad[1, 540:560].view(5, 4), x[2, 570:590].view(5, 4))
    L.token_logprobs(x[:, :500], tokens, top=4, out=given)
    assert all(torch.equal(a, b.torch) for a, b in zip(given, want))
    for bad in (dict(logprobs=x[2, 497:502]), dict(entropy=given.logprobs), dict(top_ids=pad[3, 490:510].view(5, 4)),
                dict(top_logprobs=given.top_ids.view(torch.float32)), dict(logprobs=tokens.view(torch.float32))):
        before = x.clone()
        with pytest.raises(N.MlcvError, match="overlap the inputs or one another"):
            L.token_logprobs(x[:, :500], tokens, top=4, out=given._replace(**bad))
        assert torch.equal(x, before)


# ---- pages -------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("pages", [0, 2, 500, 4097, 20000, 300000])
def test_results_do_not_keep_a_large_workspace(pages):
    """What kv_free and kv_compact return holds no more beside itself than 64 KB or a quarter of its size."""
    rng = np.random.default_rng(pages)
    table = _ints(rng.permutation(pages)[:min(pages, 40)].reshape(2, -1))
    lens = _ints([table.shape[1] * 16] * 2)
    cache = C.PagedKVCache(pages, 16, 1, 64)
    for t, m in ((table, lens), (torch.cat([table] * 400, 1), lens)):
        got = cache.free(t, m)
        want, n = S.free(t.cpu().numpy(), m.cpu().numpy(), pages, 16)
        np.testing.assert_array_equal(got.free_pages.numpy(), want)
        assert got.free_count.numpy().tolist() == [n]
        size = 4 * (pages + 1)
        assert got.free_pages.torch.untyped_storage().nbytes() <= size + max(1 << 16, size // 4) + 16
        dense = cache.compact(t, m)
        assert dense.status.numpy()[0] == pages - n
        size = 4 * (t.numel() + 2)
        assert dense.block_table.torch.untyped_storage().nbytes() <= size + max(1 << 16, size // 4) + 16
        # into given tensors, with and without a given workspace
        for kw in ({}, dict(workspace=torch.zeros(C.kv_compact_workspace(pages), dtype=torch.uint8, device="cuda"))):
            np.testing.assert_array_equal(cache.free(t, m, out=got, **kw).free_pages.numpy(), want)
            assert cache.compact(t, m, out=dense, **kw).status.numpy()[0] == pages - n


# ---- norm and rotation -------------------------------------------------------------------------------------


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("hd,rd", [(64, 64), (128, 96), (256, 256)])
@pytest.mark.parametrize("eps", [0.0, 1e-44, 1e-38, 1e-20, 1e-6])
def test_qk_rope_norms_heads_of_every_size(dt, hd, rd, eps):
    """Heads whose squares sum past the largest float32 or below the smallest, beside ordinary ones, with every size of eps."""
    rng = np.random.default_rng(hd)
    sizes = 10.0 ** (np.arange(-7, 4.5, 0.5) if dt == "f16" else np.arange(-37, 38, 1.5))
    x = rng.uniform(0.5, 1, (len(sizes), 3, hd)) * rng.choice([-1, 1], (len(sizes), 3, hd))
    x *= np.stack([sizes, sizes[::-1], np.ones(len(sizes))], 1)[..., None]
    x[:, :2, 5] *= 1e-3
    x = torch.from_numpy(x).to(TYPES[dt]).cuda()
    pos = rng.integers(0, 5000, len(sizes))
    w = torch.from_numpy(0.3 * rng.standard_normal(hd)).float().cuda()
    got = C.qk_rope(x, x[:, :1], positions=_ints(pos), rotary_dim=rd, norm=True, q_weight=w, k_weight=w, eps=eps)
    there = np.ones(len(sizes), bool)
    _check_rope(x, x[:, :1], pos, there, got, rd, 10000.0, True, (w, w), 1.0, float(np.float32(eps)))


@pytest.mark.parametrize("dt", ["f16", "f32"])
def test_qk_rope_within_one_buffer(dt):
    """Outs beside their inputs, between their rows and in their place are taken where no element is shared, and refused where
    one is."""
    rng = np.random.default_rng(8)
    t, h, kv, hd = 21, 6, 2, 64
    pos = _ints(rng.integers(0, 9000, t))
    base = torch.from_numpy(rng.standard_normal((t, 2 * (h + kv) + 1, hd))).to(TYPES[dt]).cuda()
    q, k = base[:, :h], base[:, h:h + kv]
    want = [x.torch.clone() for x in C.qk_rope(q.contiguous(), k.contiguous(), positions=pos)]

    def check(q, k, out):
        got = C.qk_rope(q, k, positions=pos, out=out)
        assert all(torch.equal(g.torch, w) and torch.equal(o, w) for g, o, w in zip(got, out, want))

    for made in (lambda b: (b[:, h + kv:2 * h + kv], b[:, 2 * h + kv:-1]),      # each token's outs behind its inputs
                 lambda b: (b[:, h + kv:2 * h + kv], b[:, h:h + kv]),          # k in place
                 lambda b: (b[:, :h], b[:, -kv:]),                              # q in place
                 lambda b: (b[:, :h], b[:, h:h + kv]),                          # both
                 lambda b: (b.new_zeros(t, h, hd), b[:, h + kv::4][:, :kv])):     # every fourth head
        b = base.clone()
        check(b[:, :h], b[:, h:h + kv], made(b))
    wide = torch.zeros((t, 3, h, hd), dtype=TYPES[dt], device="cuda")  # outs of other strides than the inputs, rows between rows
    wide[:, 0] = q
    check(wide[:, 0], k, (wide[:, 1], wide[:, 2, :kv]))
    for made in (lambda b: (b[:, 1:h + 1], b[:, -kv:]), lambda b: (b[:, h:2 * h], b[:, -kv:]),
                 lambda b: (b[:, -h:], b[:, -kv:]), lambda b: (b[:, :h], b[:, h - 1:h - 1 + kv]),
                 lambda b: (b[:, h + kv:2 * h + kv], b[:, :kv])):
        b = base.clone()
        with pytest.raises(N.MlcvError, match="overlaps an input or the other out"):
            C.qk_rope(b[:, :h], b[:, h:h + kv], positions=pos, out=made(b))
        assert torch.equal(b, base)


def test_refused_requests_keep_their_pages_over_a_fork():
    """A plan refuses a request that does not fit; the step goes on with the lengths that the requests hold: no page of the
    refused one is free, no copy goes there, and its row goes on as it was."""
    cache = C.PagedKVCache(12, 16, 1, 64, layers=2)
    table = torch.full((3, 8), -1, dtype=torch.int32, device="cuda")
    lens = _ints([0, 0, 0])
    x = torch.from_numpy(np.random.default_rng(3).standard_normal((200, 1, 64))).half().cuda()

    def step(new):
        free = cache.free(table, lens)
        plan = cache.plan(lens, _ints(new), table, free.free_pages, sum(new), free_count=free.free_count)
        for y in range(2):
            cache.write(x[:sum(new)], x[:sum(new)], plan, y)
        return plan

    plan = step([50, 33, 70])  # 4, 3 and 5 pages: none is free
    assert plan.status.numpy().tolist() == [12, 0]
    lens = plan.kv_lens.torch.clone()
    lens[2] = 0                # the last one has ended
    plan = step([1, 100, 1])   # the second would need 6 more; the third starts anew
    assert plan.kv_lens.numpy().tolist() == [51, 0, 1] and plan.status.numpy().tolist() == [1, 1]
    held = torch.where(plan.kv_lens.torch > 0, plan.kv_lens.torch, lens)
    assert held.cpu().tolist() == [51, 33, 1]
    mine = table[1, :3].long()
    before = [t.view(torch.uint8)[:, mine].clone() for t in cache.all_layers()]
    free = cache.free(table, held)
    n = int(free.free_count.numpy()[0])
    assert n == 4 and not set(free.free_pages.numpy()[:n].tolist()) & set(mine.cpu().tolist())
    fork = cache.fork(_ints([0, 0, 1, 1, 2]), table, held, *free)
    assert fork.kv_lens.numpy().tolist() == [51, 51, 33, 33, 1] and fork.status.numpy().tolist() == [2, 0]
    assert torch.equal(fork.block_table.torch[2, :3], table[1, :3])
    for t, b in zip(cache.all_layers(), before):
        assert torch.equal(t.view(torch.uint8)[:, mine], b)
        assert torch.equal(t.view(torch.uint8)[:, fork.block_table.torch[3, 2].long()], b[:, 2])  # the copy of its last page
