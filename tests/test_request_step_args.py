"""Argument checks of the entry points around a decode step's attention, all answered on the host before any device
call."""

from __future__ import annotations

import pytest
import torch

from mlc_vla import _native as N
from mlc_vla import kv_cache as C
from mlc_vla import logits as L

P = 4096  # a pointer that is never followed


def _rope(**kw):
    a = dict(q=P, q_tok=256, q_head=64, k=P, k_tok=128, k_head=64, dtype=1, tokens=5, cu=P, B=2, lens=P, pos=None, H=4,
             KV=2, hd=64, rotary=64, theta=1e4, norm=0, qw=None, kw=None, w_dtype=1, w_offset=1.0, eps=1e-6, qo=P,
             qo_tok=256, qo_head=64, ko=P, ko_tok=128, ko_head=64, stream=None)
    a.update(kw)
    N.call("mlcv_qk_rope", *a.values())


def _logprobs(**kw):
    a = dict(logits=P, dtype=1, stride=100, rows=3, vocab=100, scale=1.0, tokens=P, given=1, lp=P, entropy=P, top=4, ids=P,
             tlp=P, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    N.call("mlcv_token_logprobs", *a.values())


@pytest.mark.parametrize("fn,bad,what", [
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
    (_rope, dict(H=2 ** 30), "heads"), (_rope, dict(qo_tok=0), "out overlap"), (_rope, dict(ko_head=32), "out overlap"),
])
def test_refused(fn, bad, what):
    with pytest.raises(N.MlcvError, match=what):
        fn(**bad)


def test_empty_calls_do_nothing():
    _rope(tokens=0)
    _rope(B=0)
    _logprobs(rows=0)


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
