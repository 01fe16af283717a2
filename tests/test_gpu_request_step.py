"""What a decode step of several requests needs around its attention, on the GPU: norm and rotation of queries and keys
(kv_cache.qk_rope), log probabilities (logits.token_logprobs), against plain implementations in 64 bits (stepref.py, which derives the tolerances)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import stepref as S
from mlc_vla import _native as N
from mlc_vla import kv_cache as C
from mlc_vla import logits as L

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(autouse=True)
def _named(request):
    print(request.node.name, flush=True)


def _ints(v):
    return torch.tensor(list(v), dtype=torch.int32, device="cuda")


def _host(t):
    return t.detach().cpu().to(torch.float64).numpy()


def _randn(rng, shape, dt, scale=1.0):
    return torch.from_numpy(scale * rng.standard_normal(shape)).to(dt).cuda()


# ---- norm and rotation ---------------------------------------------------------------------------------


def _check_rope(q, k, pos, there, got, rd, theta, norm, ws, offset, eps):
    for x, y, w in zip((q, k), got, ws):
        hd = x.shape[2]
        want, size = S.rope(_host(x), pos, rd, theta, norm, None if w is None else _host(w), offset, eps)
        tol = S.rope_bound(want, size, x.dtype, hd, pos, norm)
        y = _host(y.torch)
        assert (np.abs(y - want) <= tol)[there].all(), np.max((np.abs(y - want) / tol)[there])


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("hd,heads,kv,rd", [(64, 1, 1, 64), (64, 14, 2, 32), (128, 8, 8, 128), (128, 5, 1, 112),
                                            (256, 8, 1, 256), (256, 3, 3, 16), (256, 2, 1, 0), (64, 1, 1, 48), (64, 2, 1, 16),
                                            (128, 2, 1, 96), (256, 1, 1, 256)])
@pytest.mark.parametrize("norm", [False, True])
def test_qk_rope(dt, hd, heads, kv, rd, norm):
    rng = np.random.default_rng(hd + heads + rd + norm)
    past, new = [0, 131071, 5, 700, 3], [3, 1, 0, 70, 2]
    cu = np.concatenate([[0], np.cumsum(new)])
    lens = [p + n for p, n in zip(past, new)]
    tokens = int(cu[-1]) + 2  # two rows behind the last request
    q, k = _randn(rng, (tokens, heads, hd), TYPES[dt], 3.0), _randn(rng, (tokens, kv, hd), TYPES[dt])
    ws = [None, None]
    if norm:
        ws = [_randn(rng, hd, TYPES[dt], 0.3), None if rd == 16 else _randn(rng, hd, TYPES[dt], 0.3)]
    got = C.qk_rope(q, k, _ints(cu), _ints(lens), theta=500000.0, rotary_dim=rd, norm=norm, q_weight=ws[0], k_weight=ws[1])
    pos, there = S.places(cu, lens, tokens)
    _check_rope(q, k, pos, there, got, rd, 500000.0, norm, ws, 1.0, 1e-6)


@pytest.mark.parametrize("dt", ["f16", "f32"])
def test_qk_rope_given_positions(dt):
    """Any int32: far, negative, the same twice; weights in float32, no offset, another eps."""
    rng = np.random.default_rng(1)
    pos = np.array([0, 1, -1, 7, 7, 131072, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31] + list(range(100, 600)))
    q, k = _randn(rng, (len(pos), 4, 128), TYPES[dt]), _randn(rng, (len(pos), 2, 128), TYPES[dt])
    ws = [torch.from_numpy(1 + 0.1 * rng.standard_normal(128)).float().cuda() for _ in range(2)]
    for norm, w in ((False, [None, None]), (True, ws), (True, [None, None])):
        got = C.qk_rope(q, k, positions=_ints(pos), norm=norm, q_weight=w[0], k_weight=w[1], weight_offset=0.0, eps=1e-3)
        _check_rope(q, k, pos, np.ones(len(pos), bool), got, 128, 10000.0, norm, w, 0.0, 1e-3)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dt", ["f16", "f32"])
def test_qk_rope_strides(hd, dt):
    """Views of a fused projection, rows off 16 bytes, head-major tensors, in place, into given tensors."""
    rng = np.random.default_rng(hd)
    t, h, kv = 37, 6, 2
    pos = _ints(range(1000, 1000 + t))
    base = _randn(rng, (t, h + 2 * kv, hd), TYPES[dt])
    q, k = base[:, :h], base[:, h:h + kv]
    want = [x.torch.clone() for x in C.qk_rope(q.contiguous(), k.contiguous(), positions=pos, norm=True)]
    assert all(torch.equal(a.torch, b) for a, b in zip(C.qk_rope(q, k, positions=pos, norm=True), want))
    odd = torch.zeros(t * (h + kv) * hd + 3, dtype=TYPES[dt], device="cuda")[3:].view(t, h + kv, hd)
    odd.copy_(base[:, :h + kv])
    assert all(torch.equal(a.torch, b) for a, b in zip(C.qk_rope(odd[:, :h], odd[:, h:], positions=pos, norm=True), want))
    qh, kh = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k))
    outs = [torch.zeros((n, t, hd + 8), dtype=TYPES[dt], device="cuda").transpose(0, 1)[..., 8:] for n in (h, kv)]
    got = C.qk_rope(qh, kh, positions=pos, norm=True, out=outs)
    assert all(torch.equal(a.torch, b) and a.torch.data_ptr() == o.data_ptr() for a, b, o in zip(got, want, outs))
    v = base[:, h + kv:].clone()
    C.qk_rope(q, k, positions=pos, norm=True, out=(q, k))  # in place
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(base[:, h + kv:], v)


def test_qk_rope_rows_behind_the_last_request():
    """They stay as they were; so does everything where no offset says whose a token is."""
    rng = np.random.default_rng(3)
    q, k = _randn(rng, (9, 2, 64), torch.float16), _randn(rng, (9, 1, 64), torch.float16)
    outs = [torch.full_like(x, 7.0) for x in (q, k)]
    C.qk_rope(q, k, _ints([0, 2, 5]), _ints([2, 9]), out=outs)
    assert all((o[5:] == 7).all() and (o[:5] != 7).any(-1).all() for o in outs)
    for cu in ([9, 9, 9], [-5, -1, 0]):
        outs = [torch.full_like(x, 7.0) for x in (q, k)]
        C.qk_rope(q, k, _ints(cu), _ints([2, 9]), out=outs)
        assert all((o == 7).all() for o in outs)
    # no tokens, no requests
    C.qk_rope(q[:0], k[:0], _ints([0, 0]), _ints([4]))
    outs = [torch.full_like(x, 7.0) for x in (q, k)]
    C.qk_rope(q, k, _ints([0]), _ints([]), out=outs)
    assert all((o == 7).all() for o in outs)


@pytest.mark.parametrize("b", [1, 63, 64, 65, 127, 4095, 4097, 9000])
def test_qk_rope_of_many_requests(b):
    """The search for a token's request; some bring no tokens."""
    rng = np.random.default_rng(b)
    new = rng.integers(0, 3, b)
    new[0] = 1
    cu = np.concatenate([[0], np.cumsum(new)])
    lens = rng.integers(0, 5000, b) + new
    tokens = int(cu[-1])
    q, k = _randn(rng, (tokens, 1, 64), torch.float32), _randn(rng, (tokens, 1, 64), torch.float32)
    pos, there = S.places(cu, lens, tokens)
    got = C.qk_rope(q, k, _ints(cu), _ints(lens))
    same = C.qk_rope(q, k, positions=_ints(pos))
    assert all(torch.equal(x.torch, y.torch) for x, y in zip(got, same))
    _check_rope(q, k, pos, there, got, 64, 10000.0, False, (None, None), 1.0, 1e-6)


def test_qk_rope_values_of_every_size():
    """Zeros, subnormals, the largest values, infinities and NaN stay within their head."""
    q = torch.zeros((6, 2, 64), dtype=torch.float16, device="cuda")
    q[1], q[2, 0], q[3, 0, 5], q[4, 0, 5] = 6e-8, 6e4, float("inf"), float("nan")
    k = torch.ones((6, 1, 64), dtype=torch.float16, device="cuda")
    pos = _ints([0] * 6)
    got = C.qk_rope(q, k, positions=pos)[0].torch
    assert torch.equal(got[:3], q[:3]) and torch.isfinite(got[3:, 1]).all()
    assert got[3, 0, 5].isinf() and got[4, 0, 5].isnan()
    got = C.qk_rope(q, k, positions=pos, norm=True)[0].torch
    assert (got[0] == 0).all() and torch.isfinite(got[:3]).all() and (got[2, 0] == 1).all()
    # 6e-8^2 is far below eps: x / sqrt(eps)
    assert (got[1] - 5.96e-8 * 1e3).abs().max() < 1e-6


@pytest.mark.parametrize("norm", [False, True])
def test_qk_rope_dims_that_are_not_turned(norm):
    """They know nothing of one another: an infinity stays where it is (but for the norm, which is its head's)."""
    x = torch.ones((3, 2, 128), device="cuda")
    x[0, 0, 40], x[1, 1, 127], x[2, 0, 3] = float("inf"), float("nan"), float("inf")
    got = C.qk_rope(x, x[:, :1], positions=_ints([5, 6, 0]), rotary_dim=32, norm=norm)[0].torch
    bad = ~torch.isfinite(got)
    if norm:
        assert not bad[0, 1].any() and not bad[1, 0].any() and not bad[2, 1].any()
    else:
        want = torch.zeros_like(bad)
        want[0, 0, 40] = want[1, 1, 127] = want[2, 0, 3] = want[2, 0, 19] = True  # 3 and 19 are a pair: inf * 0
        assert torch.equal(bad, want) and torch.equal(got[..., 32:].nan_to_num(7.0), x[..., 32:].nan_to_num(7.0))


def test_qk_rope_rotates_as_the_model_does():
    """The rotation of the joint attention's oracle."""
    from oracle import pi0_oracle as O

    rng = np.random.default_rng(5)
    x = rng.standard_normal((40, 8, 256)).astype(np.float32)
    cos, sin = O.make_rope_np(40, 256, 10000.0, 0)
    want = O.apply_rope(x, cos, sin, O.Prec("f64"))
    t = torch.from_numpy(x).cuda()
    got = C.qk_rope(t, t[:, :1], positions=_ints(range(40)))[0].torch
    # its table holds float32 angles: at position 39 half a step is 2^-19
    assert np.abs(_host(got) - want).max() <= 2.0 ** -18 * 2 * np.abs(x).max()


def test_qk_rope_arguments():
    rng = np.random.default_rng(9)
    q, k = _randn(rng, (4, 4, 64), torch.float16), _randn(rng, (4, 2, 64), torch.float16)
    cu, lens, pos, w = _ints([0, 4]), _ints([4]), _ints(range(4)), _randn(rng, 64, torch.float16)
    C.qk_rope(q, k, cu, lens)
    for args, kw, what in (
            ((q, k), {}, "positions"), ((q, k, cu), {}, "positions"), ((q, k, cu, lens), dict(positions=pos), "exclude"),
            ((q, k.float(), cu, lens), {}, "k has dtype"), ((q, k[:3], cu, lens), {}, "k expects shape"),
            ((q, k[..., :32], cu, lens), {}, "k expects shape"), ((q[0], k, cu, lens), {}, "q expects shape"),
            ((q.int(), k, cu, lens), {}, "q has dtype"), ((q[..., ::2], k[..., ::2], cu, lens), {}, "contiguous rows"),
            ((q, k, cu, _ints([4, 4])), {}, "cu_seqlens expects"), ((q, k, cu.long(), lens), {}, "cu_seqlens has dtype"),
            ((q, k, cu.cpu(), lens), {}, "cu_seqlens is not on"), ((q, k), dict(positions=pos[:3]), "positions expects"),
            ((q, k), dict(positions=pos.long()), "positions has dtype"),
            ((q, k, cu, lens), dict(q_weight=w), "goes with norm"),
            ((q, k, cu, lens), dict(norm=True, q_weight=w[:32]), "q_weight expects"),
            ((q, k, cu, lens), dict(norm=True, q_weight=w, k_weight=w.float()), "q_weight has dtype"),
            ((q, k, cu, lens), dict(norm=True, k_weight=w.bfloat16()), "k_weight has dtype"),
            ((q, k, cu, lens), dict(out=(q, k[:3])), "out expects"),
            ((q, k, cu, lens), dict(out=(q, k, k)), "two tensors")):
        with pytest.raises(ValueError, match=what):
            C.qk_rope(*args, **kw)
    for kw, what in ((dict(rotary_dim=24), "rotary"), (dict(rotary_dim=80), "rotary"), (dict(rotary_dim=-16), "rotary"),
                     (dict(theta=0.5), "theta"), (dict(theta=float("nan")), "theta"), (dict(norm=True, eps=-1.0), "eps"),
                     (dict(norm=True, eps=float("nan")), "eps"),
                     (dict(norm=True, q_weight=w, weight_offset=float("inf")), "w_offset"),
                     (dict(out=(q[:1].expand(4, 4, 64), k)), "must have its strides"),
                     (dict(out=(q.clone()[:1].expand(4, 4, 64), k)), "out overlap"),
                     (dict(out=(q.transpose(0, 1), k)), "must have its strides")):
        with pytest.raises(N.MlcvError, match=what):
            C.qk_rope(q, k, cu, lens, **kw)


# ---- log probabilities -----------------------------------------------------------------------------------


def _check_logprobs(x, scale, tokens, top, **kw):
    host, vocab = _host(x), x.shape[1]
    ids = None if tokens is None else tokens.cpu().numpy().reshape(len(host), -1)
    want, h, top_ids, top_lp = S.logprobs(host, float(np.float32(scale)), ids, top)
    tol, tol_h = S.logprobs_bound(host, scale, vocab)
    got = L.token_logprobs(x, tokens, top=top, scale=scale, **kw)

    def near(g, w, t):
        g = g.torch.cpu().double().numpy().reshape(w.shape)
        fin = np.isfinite(w)
        np.testing.assert_array_equal(g[~fin], w[~fin])
        with np.errstate(invalid="ignore"):
            assert (np.abs(g - w) <= t)[fin].all(), np.max((np.abs(g - w) / t)[fin])

    near(got.entropy, h, tol_h)
    assert (got.logprobs is None) == (tokens is None) and (got.top_ids is None) == (not top)
    if tokens is not None:
        assert got.logprobs.shape == tuple(tokens.shape)
        near(got.logprobs, want, tol(np.where(np.isfinite(want), want, 0.0)))
    if top:
        np.testing.assert_array_equal(got.top_ids.numpy(), top_ids)
        near(got.top_logprobs, top_lp, tol(np.where(np.isfinite(top_lp), top_lp, 0.0)))
    return got


def _tokens(rng, rows, n, vocab):
    t = rng.integers(-1, vocab + 1, (rows, n) if n > 1 else rows)
    return torch.from_numpy(t.astype(np.int32)).cuda()


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,vocab,top,n", [
    (1, 1, 1, 1), (3, 2, 2, 2), (1, 7, 5, 1), (9, 64, 64, 1), (5, 333, 20, 3), (130, 4096, 1, 1), (2, 4097, 64, 1),
    (3, 16391, 20, 5), (1, 50257, 20, 1), (40, 50257, 8, 1), (2, 257152, 64, 70), (1, 1000, 0, 1), (3, 70001, 0, 0),
    (1100, 5001, 3, 1), (4100, 4500, 3, 1), (1000, 4000, 20, 0), (17, 16385, 2, 1)])
def test_token_logprobs(dt, rows, vocab, top, n):
    rng = np.random.default_rng(vocab + rows)
    x = rng.standard_normal((rows, vocab)) * 3
    x[np.arange(rows), rng.integers(0, vocab, rows)] += 9
    x = torch.from_numpy(x).to(TYPES[dt]).cuda()
    _check_logprobs(x, 1.0 if rows != 5 else 0.7, _tokens(rng, rows, n, vocab) if n else None, top)


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("vocab", [100, 5000, 33000])
def test_token_logprobs_order(dt, vocab):
    """Ascending, descending, all equal, two values, zeros of both signs: ties go to the lowest index."""
    rng = np.random.default_rng(vocab)
    up = np.arange(vocab) / vocab * 20 - 10
    x = np.stack([up, -up, np.full(vocab, 1.5), rng.integers(0, 2, vocab) * 1.0, np.where(rng.random(vocab) < 0.5, 0.0, -0.0),
                  np.sort(rng.standard_normal(vocab)), np.where(np.arange(vocab) % 64 < 8, up, -20.0)])
    x = torch.from_numpy(x).to(TYPES[dt]).cuda()
    for top in (1, 20, 64):
        _check_logprobs(x, 1.0, _tokens(rng, len(x), 2, vocab), top)


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("vocab", [50, 9001])
def test_token_logprobs_masks(dt, vocab):
    """-inf and the type's lowest value as masks: of some logits, of all but a few, of all; NaN and +inf in a row."""
    rng = np.random.default_rng(vocab)
    low, t = torch.finfo(TYPES[dt]).min, vocab - 3
    x = torch.from_numpy(rng.standard_normal((14, vocab)) * 2).to(TYPES[dt])
    x[0, 5:] = -np.inf
    x[1, :t] = -np.inf
    x[2] = -np.inf
    x[3, 5:] = low
    x[4, :t] = low
    x[5] = low
    x[6] = torch.finfo(TYPES[dt]).max
    x[7, 3] = np.nan
    x[8, t] = np.inf
    x[9] = np.nan
    x[10, ::2], x[10, 1::2] = -np.inf, np.nan
    x[11, 2], x[11, 3:] = low, -np.inf
    x[12, 0] = np.nan
    x[12, 1:] = -np.inf
    x[13, :7], x[13, 7:] = torch.finfo(TYPES[dt]).max, -np.inf
    x = x.cuda()
    for scale in (1.0, 4.0):
        for top in (0, 1, 20, 50):
            _check_logprobs(x, scale, _tokens(rng, len(x), 3, vocab), top)


@pytest.mark.parametrize("dt", ["f16", "f32"])
@pytest.mark.parametrize("scale", [1e-6, 1e-3, 30.0, 1e6])
def test_token_logprobs_temperatures(dt, scale):
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.standard_normal((3, 6000)) * 5).to(TYPES[dt]).cuda()
    _check_logprobs(x, scale, _tokens(rng, 3, 4, 6000), 10)


def test_token_logprobs_of_certain_rows():
    """A row that is almost certain keeps the digits of its entropy: every term has one sign."""
    x = torch.full((8, 5000), -30.0, device="cuda")
    gap = torch.tensor([4.0, 8, 12, 16, 20, 24, 28, 30], device="cuda")
    x[:, 17] = gap
    got = _check_logprobs(x, 1.0, torch.full((8,), 17, dtype=torch.int32, device="cuda"), 2)
    _, h, _, _ = S.logprobs(_host(x), 1.0, None, 2)
    # ln s: the largest term's exponential is off by 2^-23, s by 2^-24 of about 1; every other term by (5000 / 256 + 200) 2^-24
    np.testing.assert_allclose(got.entropy.numpy(), h, rtol=1e-4, atol=2.0 ** -22)


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("vocab", [37, 4099, 30011])
def test_token_logprobs_strides(dt, vocab):
    """Rows at every offset from 16 bytes, a padded vocabulary, one row for all, rows backwards; given outputs."""
    rng = np.random.default_rng(vocab)
    whole = torch.from_numpy(rng.standard_normal((9, vocab + 13)) * 3).to(TYPES[dt]).cuda()
    whole[:, vocab:] = float("nan")  # never looked at
    tokens = _tokens(rng, 9, 1, vocab)
    for off in range(9):
        _check_logprobs(whole[:, off:vocab], 1.0, tokens, 7)
    flat = whole.flatten()[13:]
    flat = torch.where(torch.isnan(flat), 0.0, flat).to(TYPES[dt])
    _check_logprobs(flat[:8 * (vocab + 13)].view(8, vocab + 13)[:, 5:vocab + 5], 1.0, tokens[:8], 7)
    _check_logprobs(whole[:1, :vocab].expand(9, vocab), 1.0, tokens, 7)
    made = _check_logprobs(whole[:, :vocab], 1.0, tokens, 7)
    n = L.token_logprobs_workspace(9, vocab, 7)
    given = L.TokenLogprobs(*(torch.zeros_like(t.torch) for t in made))
    ws = torch.zeros(n + 64, dtype=torch.uint8, device="cuda")
    again = L.token_logprobs(whole[:, :vocab], tokens, top=7, out=given, workspace=ws)
    assert again is given and all(torch.equal(a, b.torch) for a, b in zip(given, made)) and (ws[n:] == 0).all()


def test_token_logprobs_past_32_bit_offsets():
    """Rows behind 2^32 bytes and 2^31 elements."""
    rows, vocab = 8400, 257152
    x = torch.empty((rows, vocab), dtype=torch.float16, device="cuda")
    x.fill_(-5.0)
    hot = torch.arange(rows, device="cuda") * 29 % vocab
    x[torch.arange(rows, device="cuda"), hot] = 9.0
    got = L.token_logprobs(x, hot.to(torch.int32), top=2)
    want = -np.log1p((vocab - 1) * np.exp(-14.0))
    assert torch.equal(got.top_ids.torch[:, 0], hot.to(torch.int32))
    assert torch.equal(got.top_ids.torch[:, 1], (hot == 0).to(torch.int32))
    assert (got.logprobs.torch - want).abs().max() < 1e-4 and torch.equal(got.logprobs.torch, got.top_logprobs.torch[:, 0])
    del x
    torch.cuda.empty_cache()


def test_token_logprobs_arguments():
    x = torch.zeros((3, 100), dtype=torch.float16, device="cuda")
    t = _ints([1, 2, 3])
    made = L.token_logprobs(x, t, top=4)
    for args, kw, what in (
            ((x[0],), {}, "logits expects"), ((x.int(),), {}, "logits has dtype"), ((x[:, ::2],), {}, "contiguous rows"),
            ((x.cpu(),), {}, "device"), ((x, t[:2]), {}, "tokens expects"), ((x, t.long()), {}, "tokens has dtype"),
            ((x, t.cpu()), {}, "tokens is not on"), ((x, t), dict(top=-1), "top"),
            ((x,), dict(top=4, out=made), "nothing to hold"), ((x, t), dict(out=made), "nothing to hold"),
            ((x, t), dict(top=3, out=made), "top_ids expects"),
            ((x, t), dict(top=4, out=made._replace(entropy=None)), "entropy is missing")):
        with pytest.raises(ValueError, match=what):
            L.token_logprobs(*args, **kw)
    for kw, what in ((dict(top=65), "top must"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
                     (dict(scale=-1.0), "scale")):
        with pytest.raises(N.MlcvError, match=what):
            L.token_logprobs(x, t, **kw)
    with pytest.raises(N.MlcvError, match="bad size"):
        L.token_logprobs(x[:, :0])
    big = torch.zeros((2, 50000), device="cuda")
    assert L.token_logprobs_workspace(2, 50000, 5) > 64
    with pytest.raises(N.MlcvError, match="workspace"):
        L.token_logprobs(big, workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"), top=5)
    assert L.token_logprobs(x[:0], t[:0], top=2).top_ids.shape == (0, 2)


def test_token_logprobs_refuses_one_token_without_a_row():
    x = torch.zeros((1, 100), dtype=torch.float16, device="cuda")
    for t in (_ints([3])[0], _ints([3]).reshape(1, 1, 1)):
        with pytest.raises(ValueError, match="tokens expects"):
            L.token_logprobs(x, t)
