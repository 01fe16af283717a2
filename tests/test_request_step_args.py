"""Argument checks of the entry points around a decode step's attention, all answered on the host before any device
call."""

from __future__ import annotations

import ctypes

import pytest
import torch

from mlc_vla import _native as N
from mlc_vla import kv_cache as C
from mlc_vla import logits as L

P = 4096  # a pointer that is never followed


def _rope(**kw):
    a = dict(q=P, q_tok=256, q_head=64, k=P, k_tok=128, k_head=64, dtype=1, tokens=5, cu=P, B=2, lens=P, pos=None, H=4,
             KV=2, hd=64, rotary=64, theta=1e4, norm=0, qw=None, kw=None, w_dtype=1, w_offset=1.0, eps=1e-6, qo=2 * P,
             qo_tok=256, qo_head=64, ko=3 * P, ko_tok=128, ko_head=64, stream=None)
    a.update(kw)
    N.call("mlcv_qk_rope", *a.values())


def _logprobs(**kw):
    a = dict(logits=P, dtype=1, stride=100, rows=3, vocab=100, scale=1.0, tokens=P, given=1, lp=P, entropy=P, top=4, ids=P,
             tlp=P, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    N.call("mlcv_token_logprobs", *a.values())


def _free(**kw):
    a = dict(table=P, B=2, max_pages=4, lens=2 * P, num_pages=8, page=16, free=3 * P, count=4 * P, ws=5 * P, ws_bytes=1 << 40,
             stream=None)
    a.update(kw)
    N.call("mlcv_kv_free", *a.values())


def _copy(**kw):
    a = dict(src=P, dst=P, n=2, k=P, ks=P, v=P, vs=P, num_pages=8, k2=P, ks2=P, v2=P, vs2=P, pages2=8, layers=2, page=16, KV=1,
             hd=64, stream=None)
    a.update(kw)
    N.call("mlcv_kv_copy", *a.values())


def _fork(**kw):
    a = dict(parents=P, n=3, table=2 * P, B=2, max_pages=4, lens=3 * P, free=4 * P, n_free=5, count=5 * P, k=P, ks=P, v=P, vs=P,
             layers=2, num_pages=8, page=16, KV=1, hd=64, out=6 * P, out_lens=7 * P, status=8 * P, stream=None)
    a.update(kw)
    N.call("mlcv_kv_fork", *a.values())


def _compact(**kw):
    a = dict(table=P, B=2, max_pages=4, lens=2 * P, k=P, ks=P, v=P, vs=P, layers=2, num_pages=8, page=16, KV=1, hd=64, out=3 * P,
             status=4 * P, ws=5 * P, ws_bytes=1 << 40, stream=None)
    a.update(kw)
    N.call("mlcv_kv_compact", *a.values())


@pytest.mark.parametrize("fn,bad,what", [
    (_free, dict(page=48), "page"), (_free, dict(num_pages=-1), "negative"), (_free, dict(B=4097), "4096"),
    (_free, dict(num_pages=2 ** 28), "slots"), (_free, dict(max_pages=2 ** 28), "slots"), (_free, dict(free=None), "null"),
    (_free, dict(count=None), "null"), (_free, dict(lens=None), "null"), (_free, dict(table=None), "null"),
    (_free, dict(ws=None), "workspace"), (_free, dict(ws=P + 8), "workspace"), (_free, dict(ws_bytes=64), "workspace"),
    (_free, dict(free=P), "overlap"), (_free, dict(count=2 * P + 4), "overlap"), (_free, dict(free=3 * P, count=3 * P + 28), "overlap"),
    (_copy, dict(page=8), "page"), (_copy, dict(hd=96), "head_dim"), (_copy, dict(n=-1), "negative"),
    (_copy, dict(layers=0), "layers"), (_copy, dict(KV=0), "layers"), (_copy, dict(k=None), "null"),
    (_copy, dict(vs2=None), "null"), (_copy, dict(src=None), "null"), (_copy, dict(v=P + 8), "aligned"),
    (_copy, dict(k2=P + 1), "aligned"), (_copy, dict(num_pages=2 ** 28), "slots"), (_copy, dict(pages2=-1), "negative"),
    (_copy, dict(KV=65535, page=128, hd=256), "2\\^30"),
    (_fork, dict(n=-1), "negative"), (_fork, dict(n=4097), "4096"), (_fork, dict(B=4097), "4096"), (_fork, dict(page=24), "page"),
    (_fork, dict(status=None), "null"), (_fork, dict(parents=None), "null"), (_fork, dict(out=None), "null"),
    (_fork, dict(out_lens=None), "null"), (_fork, dict(lens=None), "null"),
    (_fork, dict(free=None), "free_pages"), (_fork, dict(k=None), "null"), (_fork, dict(hd=32), "head_dim"),
    (_fork, dict(out=2 * P + 28), "overlap"), (_fork, dict(out_lens=P), "overlap"), (_fork, dict(out=4 * P - 8), "overlap"),
    (_fork, dict(status=5 * P), "overlap"), (_fork, dict(out_lens=8 * P), "overlap"),
    (_compact, dict(page=24), "page"), (_compact, dict(ws_bytes=8), "workspace"), (_compact, dict(out=None), "null"),
    (_compact, dict(status=None), "null"), (_compact, dict(lens=None), "null"), (_compact, dict(v=None), "null"),
    (_compact, dict(out=P + 4), "overlap"), (_compact, dict(status=2 * P), "overlap"), (_compact, dict(ws=P), "overlap"),
    (_compact, dict(layers=70000), "layers"), (_compact, dict(B=5000), "4096"),
    (_logprobs, dict(dtype=0), "float"), (_logprobs, dict(rows=-1), "size"), (_logprobs, dict(vocab=0), "size"),
    (_logprobs, dict(vocab=2 ** 31 - 1), "vocab"), (_logprobs, dict(top=65), "top"), (_logprobs, dict(vocab=3), "top"),
    (_logprobs, dict(top=-1), "top"), (_logprobs, dict(given=-1), "size"), (_logprobs, dict(scale=0.0), "scale"),
    (_logprobs, dict(scale=float("inf")), "scale"), (_logprobs, dict(scale=float("nan")), "scale"),
    (_logprobs, dict(logits=None), "null"), (_logprobs, dict(tokens=None), "null"), (_logprobs, dict(lp=None), "null"),
    (_logprobs, dict(ids=None), "null"), (_logprobs, dict(tlp=None), "null"), (_logprobs, dict(logits=P + 1), "aligned"),
    (_logprobs, dict(vocab=257152), "workspace"), (_logprobs, dict(vocab=257152, ws=P + 8, ws_bytes=1 << 40), "workspace"),
    (_logprobs, dict(vocab=257152, ws=P, ws_bytes=100), "workspace"), (_logprobs, dict(rows=2 ** 30), "rows"),
    (_rope, dict(dtype=4), "float"), (_rope, dict(tokens=-1), "size"), (_rope, dict(H=0), "size"),
    (_rope, dict(KV=0), "size"), (_rope, dict(B=-1), "size"), (_rope, dict(hd=80), "head_dim"),
    (_rope, dict(rotary=40), "rotary"), (_rope, dict(rotary=80), "rotary"), (_rope, dict(theta=0.0), "theta"),
    (_rope, dict(theta=float("inf")), "theta"), (_rope, dict(qw=P), "weights go with norm"),
    (_rope, dict(norm=1, eps=float("inf")), "eps"), (_rope, dict(norm=1, kw=P, w_dtype=3), "weights are"),
    (_rope, dict(norm=1, kw=P, w_offset=float("nan")), "w_offset"), (_rope, dict(pos=P), "positions"),
    (_rope, dict(cu=None, lens=None), "positions"), (_rope, dict(lens=None), "null"), (_rope, dict(q=None), "null"),
    (_rope, dict(ko=None), "null"), (_rope, dict(tokens=2 ** 31 - 1), "2\\^31"), (_rope, dict(B=2 ** 31 - 1), "requests"),
    (_rope, dict(qo=P, qo_tok=512), "strides"), (_rope, dict(ko=P, ko_head=-64), "strides"),
    (_rope, dict(H=2 ** 30), "heads"), (_rope, dict(qo_tok=0), "out overlap"), (_rope, dict(ko_head=32), "out overlap"),
])
def test_refused(fn, bad, what):
    with pytest.raises(N.MlcvError, match=what):
        fn(**bad)


def test_empty_calls_do_nothing():
    _rope(tokens=0)
    _rope(B=0)
    _logprobs(rows=0)
    _copy(n=0)
    _copy(num_pages=0)
    _copy(pages2=0)


def test_host_tensors_are_refused():
    x = torch.zeros((2, 4, 64), dtype=torch.float16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="device"):
        C.qk_rope(x, x, positions=i)
    with pytest.raises(ValueError, match="device"):
        L.token_logprobs(x[0])


def test_workspace_of_logprobs():
    assert L.token_logprobs_workspace(0, 257152, 5) == 0 and L.token_logprobs_workspace(2000, 257152, 5) == 0
    one = L.token_logprobs_workspace(1, 257152, 0)
    assert one > 0 and L.token_logprobs_workspace(1, 257152, 64) == one // 16 * (16 + 8 * 64)
    assert L.token_logprobs_workspace(1, 4096, 64) == 0
    with pytest.raises(N.MlcvError, match="null"):
        N.call("mlcv_token_logprobs_workspace", 1, 100, 1, None)


def test_workspaces_of_the_pages():
    for n in (0, 1, 4096, 4097, 2 ** 22, 2 ** 22 + 1, 2 ** 26):
        blocks = max(1, -(-n // 4096))
        assert blocks * 516 <= C.kv_free_workspace(n) <= 4 * blocks * 516 + 16
        assert C.kv_compact_workspace(n) == C.kv_free_workspace(n) + 12 * n
    for name in ("mlcv_kv_free_workspace", "mlcv_kv_compact_workspace"):
        with pytest.raises(N.MlcvError, match="null"):
            N.call(name, 5, None)
        with pytest.raises(N.MlcvError, match="num_pages"):
            N.call(name, -1, ctypes.byref(ctypes.c_size_t()))


@pytest.mark.parametrize("bad", [
    dict(qo=P + 128), dict(ko=P), dict(qo=2 * P, ko=2 * P + 2048), dict(k=2 * P + 2558), dict(ko=P + 2558), dict(ko=2 * P - 1278),
    dict(qo=P, k=P + 384, k_tok=256), dict(qo=P, k=P + 500, k_tok=256, H=3),                    # in place in a fused row, k in q's
    dict(qo=P, ko=P + 768 - 2, ko_tok=384, q_tok=384, qo_tok=384, H=6),
    dict(lens=2 * P + 4), dict(cu=3 * P + 8), dict(cu=None, lens=None, pos=2 * P), dict(norm=1, qw=2 * P), dict(norm=1, kw=3 * P + 126),
    dict(tokens=4, q_tok=-256, q=P + 6 * 512, ko=P + 3 * 512)])
def test_outs_of_rope_over_other_arrays_are_refused(bad):
    with pytest.raises(N.MlcvError, match="overlaps an input or the other out"):
        _rope(**bad)


@pytest.mark.parametrize("bad", [
    dict(lp=P + 598), dict(lp=2 * P), dict(entropy=3 * P), dict(ids=4 * P + 8), dict(tlp=5 * P - 44), dict(tlp=P),
    dict(stride=200, lp=P + 588), dict(stride=-100, entropy=P - 200), dict(given=3, lp=4 * P - 4),
    dict(rows=3, vocab=257152, stride=257152, ws=P + 16, ws_bytes=1 << 40)])
def test_outputs_of_logprobs_over_other_arrays_are_refused(bad):
    a = dict(tokens=2 * P, lp=3 * P, entropy=4 * P, ids=5 * P, tlp=6 * P)
    with pytest.raises(N.MlcvError, match="overlap the inputs or one another"):
        _logprobs(**{**a, **bad})


def test_rope_refuses_tokens_whose_next_round_passes_an_int():
    with pytest.raises(N.MlcvError, match="2\\^31 - 40961"):
        _rope(tokens=2 ** 31 - 1 - 40960 + 1)
