"""Argument checks of the request entry points, all answered on the host before any device call."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import kvref as R
from mlc_vla import _native as N
from mlc_vla import kv_cache as C

P = 4096  # a pointer that is never followed


def _plan(**kw):
    a = dict(past=P, new=P, B=2, free=P, n_free=4, num_pages=8, page=16, table=P, max_pages=4, cu=P, lens=P, slots=P,
             tokens=5, status=P, stream=None)
    a.update(kw)
    N.call("mlcv_kv_plan", *a.values())


def _write(**kw):
    a = dict(k=P, k_dtype=1, k_tok=64, k_head=64, v=P, v_dtype=1, v_tok=64, v_head=64, tokens=5, cu=P, B=2, slots=P,
             kc=P, ks=P, vc=P, vs=P, num_pages=8, page=16, KV=1, hd=64, stream=None)
    a.update(kw)
    N.call("mlcv_kv_write", *a.values())


def _attn(**kw):
    a = dict(q=P, dtype=1, q_tok=64, q_head=64, tokens=5, cu=P, B=2, lens=P, table=P, max_pages=4, kc=P, ks=P, vc=P,
             vs=P, num_pages=8, page=16, H=4, KV=2, hd=64, scale=0.1, causal=1, max_kv=10 ** 6, out=P, o_tok=256,
             o_head=64, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    N.call("mlcv_kv_attention", *a.values())


def _prompt(**kw):
    a = dict(q=P, q_tok=256, q_head=64, k=P, k_tok=128, k_head=64, v=P, v_tok=128, v_head=64, dtype=1, tokens=5, cu=P,
             B=2, H=4, KV=2, hd=64, scale=0.1, causal=1, bidir=None, out=P, o_tok=256, o_head=64, stream=None)
    a.update(kw)
    N.call("mlcv_prompt_attention", *a.values())


@pytest.mark.parametrize("fn,bad,what", [
    (_plan, dict(B=-1), "negative"), (_plan, dict(page=48), "page"), (_plan, dict(B=4097), "4096"),
    (_plan, dict(cu=None), "null"), (_plan, dict(past=None), "null"), (_plan, dict(free=None), "free_pages"),
    (_plan, dict(slots=None), "slot_map"), (_plan, dict(num_pages=2 ** 28), "slots"), (_plan, dict(num_pages=2 ** 27 - 1), "slots"),
    (_plan, dict(max_pages=2 ** 28), "slots"), (_plan, dict(status=None), "null"),
    (_write, dict(hd=96), "head_dim"), (_write, dict(page=8), "page"), (_write, dict(k_dtype=0), "float"),
    (_write, dict(v_dtype=4), "float"), (_write, dict(kc=P + 8), "aligned"), (_write, dict(v=None), "null"),
    (_write, dict(KV=0), "size"), (_write, dict(KV=70000), "65535"), (_write, dict(tokens=-1), "size"),
    (_write, dict(num_pages=2 ** 28), "slots"), (_write, dict(B=2 ** 30), "requests"),
    (_attn, dict(), "workspace"), (_attn, dict(ws=P, ws_bytes=64), "workspace"),
    (_attn, dict(ws=P + 4, ws_bytes=1 << 40), "workspace"), (_attn, dict(dtype=2), "float16 or bfloat16"),
    (_attn, dict(H=3), "kv heads"), (_attn, dict(hd=80), "head_dim"), (_attn, dict(page=24), "page"),
    (_attn, dict(scale=0.0), "scale"), (_attn, dict(scale=float("nan")), "scale"),
    (_attn, dict(scale=float("inf")), "scale"), (_attn, dict(scale=-1.0), "scale"), (_attn, dict(q=None), "null"),
    (_attn, dict(vc=P + 1), "aligned"), (_attn, dict(ks=None), "null"), (_attn, dict(max_kv=-1), "negative"),
    (_attn, dict(tokens=2 ** 31 - 1), "2\\^31"), (_attn, dict(max_pages=-1), "slots"),
    (_prompt, dict(dtype=2), "float16 or bfloat16"), (_prompt, dict(H=5), "kv heads"), (_prompt, dict(hd=72), "head_dim"),
    (_prompt, dict(scale=0.0), "scale"), (_prompt, dict(causal=0, bidir=P), "bidir"), (_prompt, dict(k=P + 2), "aligned"),
    (_prompt, dict(q_tok=257), "aligned"), (_prompt, dict(out=P + 4), "aligned"), (_prompt, dict(k_tok=32), "apart"),
    (_prompt, dict(v_tok=1 << 24), "apart"), (_prompt, dict(q=None), "null"), (_prompt, dict(B=-3), "negative"),
    (_prompt, dict(B=2 ** 31 - 1), "workgroups"),
])
def test_refused(fn, bad, what):
    with pytest.raises(N.MlcvError, match=what):
        fn(**bad)


def test_empty_calls_do_nothing():
    for fn in (_write, _attn, _prompt):
        fn(tokens=0)
        fn(B=0)
    _write(num_pages=0)


def test_workspace_query():
    n = ctypes.c_size_t(7)
    with pytest.raises(N.MlcvError, match="head_dim"):
        N.call("mlcv_kv_attention_workspace", 1, 1, 8, 1, 100, 10, ctypes.byref(n))
    with pytest.raises(N.MlcvError, match="null"):
        N.call("mlcv_kv_attention_workspace", 1, 1, 8, 1, 128, 10, None)
    for tokens, b, kv in ((0, 0, 10 ** 6), (0, 3, 100), (5, 0, 100)):
        assert C.kv_attention_workspace(tokens, b, 8, 1, 128, kv) == 0
    assert C.kv_attention_workspace(1, 1, 8, 1, 256, 131072) > 0
    # a pass over a short cache has no splits to join
    assert C.kv_attention_workspace(1, 1, 8, 1, 256, 64) == 0


def test_host_tensors_are_refused():
    x = torch.zeros((2, 4, 64), dtype=torch.float16)
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="device"):
        C.prompt_attention(x, x, x, i)
    with pytest.raises(ValueError, match="device"):
        C.kv_plan(i, i, i.view(3, 1), i, num_pages=1, page_size=16, tokens=1)
    with pytest.raises(TypeError, match="tensor"):
        C.prompt_attention(np.zeros((2, 4, 64), np.float16), x, x, i)


def test_plain_write_is_what_the_format_says():
    """The reference that the GPU is held to: torch's own conversion, and known codes."""
    x = np.random.default_rng(0).standard_normal(20000) * np.exp2(np.random.default_rng(1).uniform(-12, 8, 20000))
    x = np.clip(x, -448, 448).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(R.e4m3(x.astype(np.float64)), want)
    assert R.scale_for(448.0) == 1.0 and R.scale_for(448.1) == 2.0 and R.scale_for(0.0) == 2.0 ** -64


@pytest.mark.parametrize("a,b", [("lens", "past"), ("cu", "past"), ("table", "new"), ("slots", "free"), ("status", "free"),
                                 ("lens", "new"), ("table", "free"), ("cu", "lens"), ("slots", "table"), ("status", "cu")])
def test_a_plan_over_its_own_lengths_is_refused(a, b):
    """Every workgroup reads the lengths while one writes the plan's."""
    ints = dict(past=2, new=2, free=4, table=8, cu=3, lens=2, slots=5, status=2)
    at, p = {}, P
    for name, n in ints.items():
        at[name], p = p, p + 4 * n
    for shift in (0, 4 * (ints[b] - 1), -4 * (ints[a] - 1)):
        with pytest.raises(N.MlcvError, match="overlap"):
            _plan(**{**at, a: at[b] + shift})


@pytest.mark.parametrize("fn,bad", [
    (_write, dict(tokens=2 ** 31 - 255)), (_write, dict(tokens=2 ** 31 - 1)), (_prompt, dict(tokens=2 ** 31 - 255)),
    (_prompt, dict(tokens=2 ** 31 - 1)), (_attn, dict(tokens=2 ** 30 - 100, ws=P, ws_bytes=1 << 62)),
    (_attn, dict(tokens=2 ** 31 - 255, H=2, ws=P, ws_bytes=1 << 62)),
])
def test_tokens_near_the_largest_int_are_refused(fn, bad):
    """The last tile or page reaches past the last token: its positions have to be ints as well.  (Tensors of a stride
    of 0 have such sizes without the memory.)"""
    with pytest.raises(N.MlcvError, match="2\\^31 - 256"):
        fn(**bad)


@pytest.mark.parametrize("fn,bad", [
    (_prompt, dict(o_tok=0)), (_prompt, dict(o_head=0)), (_prompt, dict(o_tok=60)), (_prompt, dict(o_head=-32)),
    (_attn, dict(o_tok=0, ws=P, ws_bytes=1 << 62)), (_attn, dict(o_head=0, ws=P, ws_bytes=1 << 62)),
    (_prompt, dict(o_tok=64, o_head=64)), (_prompt, dict(o_tok=192, o_head=128)), (_prompt, dict(o_tok=-256, o_head=300)),
    (_attn, dict(o_tok=-63, ws=P, ws_bytes=1 << 62)), (_attn, dict(o_head=32, ws=P, ws_bytes=1 << 62)),
])
def test_rows_of_out_that_overlap_are_refused(fn, bad):
    """An expanded tensor as out: rows of several tokens or heads would be written to one place."""
    with pytest.raises(N.MlcvError, match="out overlap"):
        fn(**bad)


def test_attention_plan_query():
    s, w = ctypes.c_int32(), ctypes.c_int32()
    ask = lambda *a: N.call("mlcv_kv_attention_plan", *a, ctypes.byref(s), ctypes.byref(w)) or (s.value, w.value)  # noqa: E731
    with pytest.raises(N.MlcvError, match="head_dim"):
        ask(1, 1, 8, 1, 100, 10)
    with pytest.raises(N.MlcvError, match="null"):
        N.call("mlcv_kv_attention_plan", 1, 1, 8, 1, 64, 10, None, None)
    assert ask(0, 0, 8, 1, 64, 0) == (1, 4)
    for hd in (64, 128, 256):
        assert ask(400, 8, 8, 1, hd, 1018) == (1, 8)                            # action suffixes: no splits, no workspace
        assert C.kv_attention_workspace(400, 8, 8, 1, hd, 1018) == 0
        assert ask(1, 1, 8, 1, hd, 9000)[0] > 16 and ask(2, 2, 8, 1, hd, 1018)[0] in range(2, 17)
        assert ask(16 * 300, 300, 8, 1, hd, 4096) == (1, 4)


@pytest.mark.parametrize("fn,bad,what", [
    (_prompt, dict(scale=3e38), "scale"), (_attn, dict(scale=2.4e38, ws=P, ws_bytes=1 << 62), "scale"),
    (_prompt, dict(tokens=1 << 27, H=64, KV=64, o_tok=4096), "workgroups"),
    (_attn, dict(tokens=1 << 22, H=64, KV=64, o_tok=4096, max_kv=64), "workgroups"),
    (_write, dict(B=1 << 23, tokens=1 << 20), "requests"),
])
def test_what_a_launch_cannot_hold_is_refused(fn, bad, what):
    """A scale whose product with log2(e) is infinite; grids of 2^32 threads and more."""
    with pytest.raises(N.MlcvError, match="invalid argument.*" + what):
        fn(**bad)
