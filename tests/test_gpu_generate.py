"""Generating text for several requests with all of it together: plan over the counted free list, rotation, cache writer,
attention, log probabilities, forks of beams, a pool made dense and one moved into a larger, eager and captured."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import kvref as R
import stepref as S
from mlc_vla import kv_cache as C
from mlc_vla import logits as L

pytestmark = pytest.mark.gpu

H, KV, HD, PAGE, LAYERS, VOCAB = 4, 2, 64, 16, 2, 3001
DT = torch.float16


@pytest.fixture(autouse=True)
def _named(request):
    print(request.node.name, flush=True)


def _ints(v):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(v, np.int32))).cuda()


def _host(t):
    return t.detach().cpu().to(torch.float64).numpy()


class _Beams:
    """A server's state, and beside it each row's own keys and values as they were written."""

    def __init__(self, rows, seed=0, pages=80):
        self.rng = np.random.default_rng(seed)
        self.cache = C.PagedKVCache(pages, PAGE, KV, HD, layers=LAYERS)
        self.table = torch.full((rows, 8), -1, dtype=torch.int32, device="cuda")
        self.lens = _ints([0] * rows)
        self.own = [[np.zeros((0, 2, KV, HD)) for _ in range(LAYERS)] for _ in range(rows)]

    def rand(self, t, h):
        return torch.from_numpy(self.rng.standard_normal((t, h, HD))).to(DT).cuda()

    def step(self, new):
        """One step of `new` tokens for each row; every layer's attention is checked."""
        tokens = sum(new)
        free = self.cache.free(self.table, self.lens)
        plan = self.cache.plan(self.lens, _ints(new), self.table, free.free_pages, tokens, free_count=free.free_count)
        assert plan.status.numpy()[1] == 0
        pos, _ = S.places(plan.cu_seqlens.numpy(), plan.kv_lens.numpy(), tokens)
        cu = np.concatenate([[0], np.cumsum(new)])
        for y in range(LAYERS):
            x = self.rand(tokens, H + 2 * KV)  # a fused projection
            q, k = C.qk_rope(x[:, :H], x[:, H:H + KV], plan.cu_seqlens, plan.kv_lens, norm=True)
            want, size = S.rope(_host(x[:, H:H + KV]), pos, HD, 10000.0, True)
            assert (np.abs(_host(k.torch) - want) <= S.rope_bound(want, size, DT, HD, pos, True)).all()
            self.cache.write(k, x[:, H + KV:], plan, y)
            for b, n in enumerate(new):
                at = slice(cu[b], cu[b + 1])
                kv = np.stack([_host(k.torch)[at], _host(x[:, H + KV:])[at]], 1)
                self.own[b][y] = np.concatenate([self.own[b][y], kv])
            got = _host(self.cache.attention(q, plan, self.table, y).torch)
            for b, n in enumerate(new):
                k64, v64 = self.held(y, b, int(plan.kv_lens.numpy()[b]))
                lim = [len(k64) - n + i + 1 for i in range(n)]
                o, mass, big = R.attend(_host(q.torch)[cu[b]:cu[b + 1]], k64, v64, lim, HD ** -0.5)
                tol = R.bound(o, mass, big, DT, len(k64), HD, torch.float16, 2.0 ** -37 * 448 * 16)
                assert (np.abs(got[cu[b]:cu[b + 1]] - o) <= tol).all()
        self.lens = plan.kv_lens.torch
        return plan

    def held(self, y, b, n):
        """What the cache holds of row b, checked against what was written: within half a step of e4m3, or of its subnormals
        at the page's scale (below 2 max / 448), twice where the page grew."""
        if n == 0:
            return [np.zeros((0, KV, HD))] * 2
        kc, ks, vc, vs = self.cache.pages(y)
        ids = self.table[b].cpu().numpy()
        kf = _host(kc) * _host(ks)[..., None, None]
        vf = _host(vc).transpose(0, 1, 3, 2) * _host(vs)[..., None, None]
        got = [np.stack([x[ids[t // PAGE], :, t % PAGE] for t in range(n)]) for x in (kf, vf)]
        for z in range(2):
            x = self.own[b][y][:, z]
            assert len(x) == n
            top = np.stack([np.abs(x[p:p + PAGE]).max((0, 2)) for p in range(0, n, PAGE)])
            top = np.repeat(top, PAGE, 0)[:n][..., None]
            assert (np.abs(got[z] - x) <= 2.0 ** -4 * np.abs(x) + 2.0 ** -9 * top / 112).all()
        return got

    def fork(self, parents):
        free = self.cache.free(self.table, self.lens)
        r = self.cache.fork(_ints(parents), self.table, self.lens, *free)
        assert r.status.numpy()[1] == 0
        self.table, self.lens = r.block_table.torch, r.kv_lens.torch
        self.own = [[x.copy() for x in self.own[p]] for p in parents]

    def score(self, rows):
        """Made-up logits of each row, their best tokens checked."""
        x = torch.from_numpy(3 * self.rng.standard_normal((rows, VOCAB))).bfloat16().cuda()
        got = L.token_logprobs(x, top=4)
        _, _, ids, lp = S.logprobs(_host(x), 1.0, None, 4)
        np.testing.assert_array_equal(got.top_ids.numpy(), ids)
        return got.top_logprobs.torch


def test_beams():
    s = _Beams(3)
    s.step([40, 17, 32])
    s.fork([0, 0, 1, 1, 2, 2])
    total = torch.zeros(6, device="cuda")
    for i in range(24):
        s.step([1] * 6)
        # two beams of each request go on: the best of their alternatives
        lp = (s.score(6) + total[:, None]).view(3, 8)
        best = lp.topk(2, -1)
        total = best.values.flatten()
        parents = (torch.arange(3, device="cuda")[:, None] * 2 + best.indices // 4).flatten().cpu().tolist()
        s.fork(parents)
        if i == 8:  # the pool becomes dense
            r = s.cache.compact(s.table, s.lens)
            s.table, live = r.block_table.torch, int(r.status.numpy()[0])
            free = s.cache.free(s.table, s.lens)
            assert free.free_pages.numpy()[:80 - live].tolist() == list(range(live, 80))
        if i == 13:  # and moves into a larger one, its pages in another order
            more = C.PagedKVCache(100, PAGE, KV, HD, layers=LAYERS)
            to = np.random.default_rng(5).permutation(100)[:80]
            s.cache.copy(_ints(np.arange(80)), _ints(to), into=more)
            held = torch.arange(8, device="cuda")[None] < ((s.lens + PAGE - 1) // PAGE)[:, None]
            s.table = torch.where(held, _ints(to)[s.table.clamp(min=0).long()], s.table)
            s.cache = more
        if i == 17:  # one request ends, another takes its place, and the other's beams stay
            s.lens = s.lens * _ints([1, 1, 0, 0, 1, 1])
            for b in (2, 3):
                s.own[b] = [np.zeros((0, 2, KV, HD)) for _ in range(LAYERS)]
            s.step([1, 1, 20, 20, 1, 1])
    pages = int(s.cache.free(s.table, s.lens).free_count.numpy()[0])
    used, _ = S.used_pages(s.table.cpu().numpy(), s.lens.cpu().numpy(), 100, PAGE)
    assert pages == 100 - len(used)


def test_beams_of_a_small_pool_are_refused_and_go_on():
    """Where the free pages do not last, a fork refuses rows, and those that are left still are right."""
    s = _Beams(2, seed=3, pages=7)
    s.step([40, 20])  # 3 and 2 pages: two are free
    free = s.cache.free(s.table, s.lens)
    r = s.cache.fork(_ints([0, 0, 0, 1, 1]), s.table, s.lens, *free)
    assert r.status.numpy().tolist() == [2, 1] and r.kv_lens.numpy().tolist() == [40, 40, 40, 20, 0]
    s.table, s.lens = r.block_table.torch, r.kv_lens.torch
    s.own = [[x.copy() for x in s.own[p]] for p in (0, 0, 0, 1)] + [[np.zeros((0, 2, KV, HD))] * LAYERS]
    s.step([8, 1, 1, 12, 0])
    assert s.cache.free(s.table, s.lens).free_count.numpy().tolist() == [0]
    free = s.cache.free(s.table, s.lens)  # none: a request that would need a page is refused
    plan = s.cache.plan(s.lens, _ints([1, 1, 1, 1, 1]), s.table, free.free_pages, 5, free_count=free.free_count)
    assert plan.status.numpy().tolist() == [0, 3] and plan.kv_lens.numpy().tolist() == [0, 42, 42, 0, 0]


def test_captured_decode_step():
    """A whole step as one graph: free, plan, rotation, write, attention, log probabilities, fork.  Two graphs, new inputs
    before each replay, eager work and synchronization between them; every replay against the eager result."""
    s = _Beams(4, seed=1)
    s.step([40, 17, 32, 5])
    parents = _ints([0, 0, 2, 1])
    x = [s.rand(4, H + 2 * KV) for _ in range(LAYERS)]
    z = torch.zeros((4, 40000), dtype=torch.bfloat16, device="cuda")  # split, and joined by a second launch
    given = _ints([1, 2, 3, 4])
    ones = _ints([1] * 4)
    lens, start = s.lens.clone(), s.table.clone()

    def step():
        free = s.cache.free(s.table, lens)
        plan = s.cache.plan(lens, ones, s.table, free.free_pages, 4, free_count=free.free_count)
        out = []
        for y in range(LAYERS):
            q, k = C.qk_rope(x[y][:, :H], x[y][:, H:H + KV], plan.cu_seqlens, plan.kv_lens)
            s.cache.write(k, x[y][:, H + KV:], plan, y)
            out.append(s.cache.attention(q, plan, s.table, y))
        best = L.token_logprobs(z, given, top=6)
        free = s.cache.free(s.table, plan.kv_lens)
        fork = s.cache.fork(parents, s.table, plan.kv_lens, *free)
        dense = s.cache.compact(fork.block_table, fork.kv_lens)
        return [*plan, *out, *best, *fork, *dense]

    saved = [t.clone() for t in s.cache.all_layers()]

    def restore():
        for a, b in zip(list(s.cache.all_layers()) + [s.table], saved + [start]):
            (a.view(torch.uint8) if a.dtype == C._F8 else a).copy_(b.view(torch.uint8) if b.dtype == C._F8 else b)

    def state():
        return [(t.view(torch.uint8) if t.dtype == C._F8 else t).clone() for t in s.cache.all_layers()] + [s.table.clone()]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # each with its own outputs and workspaces
        restore()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, got))
    for i in range(4):
        for graph, got in graphs:
            for t in x:
                t.copy_(torch.from_numpy(s.rng.standard_normal(t.shape)) * 2.0 ** i)
            z.copy_(torch.from_numpy(4 * s.rng.standard_normal(z.shape)))
            parents.copy_(_ints(s.rng.integers(-1, 4, 4)))
            lens.copy_(_ints([40 - i, 16 + i, 32, 5 + 5 * i]))
            restore()
            want = [t.torch.clone() for t in step()]
            held = state()
            torch.cuda.synchronize()
            restore()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a.torch, b)
            for a, b in zip(state(), held):
                assert torch.equal(a, b)


def test_two_streams_at_once():
    """Calls that overlap on two streams, each with its own data: no call shares anything with another."""
    rng = np.random.default_rng(4)
    jobs = []
    for i in range(2):
        table = rng.permutation(9000)[:4 * 1000].reshape(4, 1000)
        t, m = _ints(table), _ints([15000, 900, 0, 16000 - i])
        cache = C.PagedKVCache(9000, PAGE, 1, HD)
        cache.k.view(torch.uint8).copy_(torch.from_numpy(rng.integers(0, 120, cache.k.shape, dtype=np.uint8)))
        z = torch.from_numpy(rng.standard_normal((5, 60000))).half().cuda()
        q, k = (torch.from_numpy(rng.standard_normal((300, h, HD))).half().cuda() for h in (8, 2))
        jobs.append((t, m, cache, z, q, k, torch.cuda.Stream()))

    def calls(t, m, cache, z, q, k):
        free = cache.free(t, m)
        out = [*free, *L.token_logprobs(z, top=9)[1:], *C.qk_rope(q, k, positions=m[:1].expand(300).contiguous())]
        out += cache.fork(_ints([0, 0, 3, 3, 3]), t, m, *free)
        return [x.torch for x in out + list(cache.compact(t, m))] + [cache.k.view(torch.uint8).clone()]

    before = [job[2].k.view(torch.uint8).clone() for job in jobs]
    want = [calls(*job[:-1]) for job in jobs]
    for job, x in zip(jobs, before):
        job[2].k.view(torch.uint8).copy_(x)
    torch.cuda.synchronize()
    for _ in range(5):
        outs = []
        for job in jobs:
            with torch.cuda.stream(job[-1]):
                outs.append(calls(*job[:-1]))
        torch.cuda.synchronize()
        for job, x, got, w in zip(jobs, before, outs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, w))
            job[2].k.view(torch.uint8).copy_(x)
        torch.cuda.synchronize()
