"""Several requests at once: packed prompts and a paged 8-bit key/value cache.

No counterpart in the reference, which serves one request over a dense cache.  Tokens of the
requests are packed one after another, ``cu_seqlens`` [B + 1] int32 says where each begins, and every
length stays on the device: nothing here synchronizes, so a serving step can be captured into a graph.

    plan = kv_plan(past, new, table, free, num_pages=..., page_size=64, tokens=T)   # slots of the new tokens
    q, k = qk_rope(q, k, plan.cu_seqlens, plan.kv_lens)                             # turned to their positions
    out = prompt_attention(q, k, v, plan.cu_seqlens)                                # a prompt's own attention
    cache.write(k, v, plan, layer)                                                  # into the pages
    out = cache.attention(q, plan, table, layer)                                    # later tokens
    free = cache.free(table, lens)                                                  # pages that no request holds
    fork = cache.fork(parents, table, lens, *free)                                  # beams: who goes on from whom

Every function body is one call into ``libmlcvla_hip.so`` (include/mlcvla.h says what each computes);
tensors are ``runtime.Tensor`` or torch tensors on one HIP device, on whose current stream the work runs.
Keys and values of any strides with contiguous rows are taken in place.
"""

from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple, Optional, Tuple

import torch

from . import _native as N
from .runtime import Tensor, device

_F16, _BF16, _F32, _I32, _U8 = torch.float16, torch.bfloat16, torch.float32, torch.int32, torch.uint8
_F8 = torch.float8_e4m3fn
_CODE = {_F16: N.MLCV_DTYPE_F16, _F32: N.MLCV_DTYPE_F32, _BF16: N.MLCV_DTYPE_BF16}
_NAME = {_F16: "float16", _BF16: "bfloat16"}
_ANY_NAME = {_F16: "float16", _BF16: "bfloat16", _F32: "float32"}


class KVPlan(NamedTuple):
    """What ``kv_plan`` made: see mlcv_kv_plan."""

    cu_seqlens: Tensor  # [B + 1] first token of each request
    kv_lens: Tensor     # [B] cached tokens after the new ones are written; 0: the request was refused
    slot_map: Tensor    # [tokens] slot of each new token, -1: none
    status: Tensor      # [2] pages taken from the front of the free list; requests refused


class KVFree(NamedTuple):
    """What ``kv_free`` made: see mlcv_kv_free."""

    free_pages: Tensor  # [num_pages] the free pages, ascending, then -1
    free_count: Tensor  # [1] how many there are


class KVFork(NamedTuple):
    """What ``kv_fork`` made: see mlcv_kv_fork."""

    block_table: Tensor  # [N, max_pages]
    kv_lens: Tensor      # [N]; 0: the row was refused, or its parent is none
    status: Tensor       # [2] pages taken from the front of the free list; rows refused


class KVCompact(NamedTuple):
    """What ``kv_compact`` made: see mlcv_kv_compact."""

    block_table: Tensor  # [B, max_pages] with the pages' new numbers
    status: Tensor       # [2] pages in use, now the first of the pool; pages moved


# A call's checks take longer than the kernels of its smallest sizes: each function first looks at everything it
# needs in one expression, and only where that fails are the arguments gone through one by one for the message.
def _t(x) -> torch.Tensor:
    if type(x) is Tensor:
        return x.torch
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"expected a device tensor, got {type(x).__name__}")
    return x


def _bad(fn: str, name: str, what: str):
    raise ValueError(f"{fn}: argument {name} {what}")


def _refuse(fn: str, dev: int, wanted) -> None:
    """Raises for the first of ``wanted`` (name, tensor, dtypes, shape with None for any size, contiguous) that is not
    as said or not on HIP device ``dev``."""
    for name, t, dtypes, shape, dense in wanted:
        if t.dtype not in dtypes:
            _bad(fn, name, f"has dtype {t.dtype}")
        if t.dim() != len(shape) or any(w is not None and w != s for w, s in zip(shape, t.shape)):
            _bad(fn, name, f"expects shape {tuple(shape)}, got {tuple(t.shape)}")
        if t.get_device() < 0 or t.get_device() != dev:
            _bad(fn, name, "is not on the HIP device of the other tensors")
        if dense and not t.is_contiguous():
            _bad(fn, name, "must be contiguous")
        if not dense and t.stride(-1) != 1 and t.numel() > 0:
            _bad(fn, name, "must have contiguous rows")
    _bad(fn, wanted[0][0], "and the others do not go together")


_lib = None


def _call(name: str, dev: int, *args) -> None:
    """One native call on HIP device ``dev`` and its current stream."""
    global _lib
    if _lib is None:
        _lib = N.load()
    if dev == torch._C._cuda_getDevice():
        rc = getattr(_lib, name)(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = getattr(_lib, name)(*args, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        N.check(rc)


def _aligned(t: torch.Tensor, low: int) -> torch.Tensor:
    """``t`` [tokens, heads, hd] of 16-bit elements with 16-byte aligned rows, its tokens ``low`` to 2^24 elements
    apart: itself, or a copy."""
    a, b, _ = t.stride()
    if not (t.data_ptr() | 2 * a | 2 * b) & 15 and low <= a < 1 << 24:
        return t
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


def _like(q: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(q, memory_format=torch.contiguous_format)


def _given(fn: str, out, q: torch.Tensor, dev: int) -> torch.Tensor:
    o = _t(out)
    if not (o.shape == q.shape and o.dtype is q.dtype and o.get_device() == dev
            and (o.stride(2) == 1 or not o.numel())):
        _refuse(fn, dev, (("out", o, (q.dtype,), q.shape, False),))
    return o


def _count(fn: str, free_count, dev: int) -> int:
    c = _t(free_count)
    if not (c.dtype is _I32 and c.shape == (1,) and c.get_device() == dev):
        _refuse(fn, dev, (("free_count", c, (_I32,), (1,), True),))
    return c.data_ptr()


def kv_plan(past_lens, new_lens, block_table, free_pages, *, num_pages: int, page_size: int, tokens: int,
            free_count=None, out: Optional[KVPlan] = None) -> KVPlan:
    """Block tables and slot maps from request lengths (mlcv_kv_plan).

    past_lens, new_lens [B], block_table [B, max_pages] (its new entries are written), free_pages [F], all int32;
    ``tokens``: the packed tokens of the call.  ``free_count`` [1] int32: how many of free_pages are free, as ``kv_free``
    leaves it (mlcv_kv_plan_counted; default: all).  ``out``: a plan of the same sizes to write into; not the one whose
    ``kv_lens`` are the call's past_lens (two plans in turn do)."""
    past, new, table, free = _t(past_lens), _t(new_lens), _t(block_table), _t(free_pages)
    dev = past.get_device()
    shape = table.shape
    n, wide = shape if len(shape) == 2 else (-1, 0)
    if not (past.dtype is _I32 and new.dtype is _I32 and table.dtype is _I32 and free.dtype is _I32
            and past.shape == (n,) and new.shape == (n,) and free.dim() == 1 and past.is_contiguous()
            and new.is_contiguous() and table.is_contiguous() and free.is_contiguous()
            and dev >= 0 and new.get_device() == table.get_device() == free.get_device() == dev
            and 0 <= tokens < 1 << 31 and 0 <= num_pages < 1 << 31):
        if not (0 <= tokens < 1 << 31 and 0 <= num_pages < 1 << 31):
            _bad("kv_plan", "tokens or num_pages", "is negative or past 2^31 - 1")
        i32, b = (_I32,), past.shape[0] if past.dim() == 1 else None
        _refuse("kv_plan", dev, (("past_lens", past, i32, (None,), True), ("new_lens", new, i32, (b,), True),
                                 ("block_table", table, i32, (b, None), True),
                                 ("free_pages", free, i32, (None,), True)))
    if out is None:
        cu, lens, slots, status = torch.empty(tokens + 2 * n + 3, dtype=_I32, device=past.device).split(
            (n + 1, n, tokens, 2))
        out = KVPlan(Tensor(cu, "int32"), Tensor(lens, "int32"), Tensor(slots, "int32"), Tensor(status, "int32"))
    else:
        cu, lens, slots, status = (_t(x) for x in out)
        if not (cu.shape == (n + 1,) and lens.shape == (n,) and slots.shape == (tokens,) and status.shape == (2,)
                and all(t.dtype is _I32 and t.is_contiguous() and t.get_device() == dev
                        for t in (cu, lens, slots, status))):
            _refuse("kv_plan", dev, tuple(("out." + f, t, (_I32,), (k,), True) for f, t, k in
                                          zip(KVPlan._fields, (cu, lens, slots, status), (n + 1, n, tokens, 2))))
    _call("mlcv_kv_plan_counted", dev, past.data_ptr(), new.data_ptr(), n, free.data_ptr(), free.shape[0],
          None if free_count is None else _count("kv_plan", free_count, dev), num_pages, page_size, table.data_ptr(), wide, cu.data_ptr(),
          lens.data_ptr(), slots.data_ptr(), tokens, status.data_ptr())
    return out


def qk_rope(q, k, cu_seqlens=None, kv_lens=None, *, positions=None, theta: float = 10000.0,
            rotary_dim: Optional[int] = None, norm: bool = False, q_weight=None, k_weight=None,
            weight_offset: float = 1.0, eps: float = 1e-6, out=None) -> Tuple[Tensor, Tensor]:
    """Norm of each head (optional) and rotation of queries [tokens, H, hd] and keys [tokens, KV, hd] (float16, bfloat16 or
    float32, any strides with contiguous rows), in one pass (mlcv_qk_rope).

    The tokens' places in the cache, from a plan's ``cu_seqlens`` and ``kv_lens``, or ``positions`` [tokens] int32.
    ``rotary_dim``: the first dims of a head that are turned (default: all); ``norm``: each head is divided by its root mean
    square, and times ``weight_offset`` + its weight [hd] (of the type of q or float32) where there is one.  ``out``: two
    tensors; they may be q and k themselves, but share no other element with an input or one another.  Rows behind the
    last request are left as they were, so by default they are not initialized."""
    q, k = _t(q), _t(k)
    dev, dt = q.get_device(), q.dtype
    code = _CODE.get(dt)
    tokens, heads, hd = q.shape if q.dim() == 3 else (-1,) * 3
    kv = k.shape[1] if k.dim() == 3 else -1
    if not (code and k.dtype is dt and k.shape == (tokens, kv, hd) and dev >= 0 and k.get_device() == dev
            and (q.stride(2) == k.stride(2) == 1 or not tokens * hd)):
        t, d = (tokens, hd) if q.dim() == 3 else (None, None)
        _refuse("qk_rope", dev, (("q", q, _CODE, (None,) * 3, False), ("k", k, (dt,), (t, None, d), False)))
    n, cu, lens, pos = 0, None, None, None
    if positions is None:
        if cu_seqlens is None or kv_lens is None:
            _bad("qk_rope", "positions", "or cu_seqlens and kv_lens are needed")
        c, m = _t(cu_seqlens), _t(kv_lens)
        n = m.shape[0] if m.dim() == 1 else -1
        if not (c.dtype is _I32 and m.dtype is _I32 and c.shape == (n + 1,) and c.is_contiguous() and m.is_contiguous()
                and c.get_device() == m.get_device() == dev):
            _refuse("qk_rope", dev, (("kv_lens", m, (_I32,), (None,), True), ("cu_seqlens", c, (_I32,), (n + 1,), True)))
        cu, lens = c.data_ptr(), m.data_ptr()
    else:
        if cu_seqlens is not None or kv_lens is not None:
            _bad("qk_rope", "positions", "and cu_seqlens or kv_lens exclude one another")
        p = _t(positions)
        if not (p.dtype is _I32 and p.shape == (tokens,) and p.is_contiguous() and p.get_device() == dev):
            _refuse("qk_rope", dev, (("positions", p, (_I32,), (tokens,), True),))
        pos = p.data_ptr()
    wt, at = code, [None, None]
    if q_weight is not None or k_weight is not None:
        if not norm:
            _bad("qk_rope", "q_weight" if q_weight is not None else "k_weight", "goes with norm")
        ws = [None if w is None else _t(w) for w in (q_weight, k_weight)]
        wt = _F32 if any(w is not None and w.dtype is _F32 for w in ws) else dt
        for i, w in enumerate(ws):
            if w is None:
                continue
            if not (w.dtype is wt and w.shape == (hd,) and w.is_contiguous() and w.get_device() == dev):
                _refuse("qk_rope", dev, (("qk"[i] + "_weight", w, (wt,), (hd,), True),))
            at[i] = w.data_ptr()
        wt = _CODE[wt]
    if out is None:
        qo, ko = _like(q), _like(k)
    else:
        if len(out) != 2:
            _bad("qk_rope", "out", "is not two tensors")
        qo, ko = _given("qk_rope", out[0], q, dev), _given("qk_rope", out[1], k, dev)
    qt, qh, _ = q.stride()
    kt, kh, _ = k.stride()
    qot, qoh, _ = qo.stride()
    kot, koh, _ = ko.stride()
    _call("mlcv_qk_rope", dev, q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, code, tokens, cu, n, lens, pos, heads, kv, hd,
          hd if rotary_dim is None else rotary_dim, theta, norm, at[0], at[1], wt, weight_offset, eps, qo.data_ptr(), qot,
          qoh, ko.data_ptr(), kot, koh)
    return Tensor(qo, _ANY_NAME[dt]), Tensor(ko, _ANY_NAME[dt])


def _cache_wanted(kc, ks, vc, vs):
    pages, kv, page, hd = kc.shape if kc.dim() == 4 else (None,) * 4
    return (("k_cache", kc, (_F8,), (None,) * 4, True), ("k_scale", ks, (_F32,), (pages, kv), True),
            ("v_cache", vc, (_F8,), (pages, kv, hd, page), True), ("v_scale", vs, (_F32,), (pages, kv), True))


def kv_write(k, v, cu_seqlens, slot_map, k_cache, k_scale, v_cache, v_scale) -> None:
    """Write new keys and values [tokens, KV, hd] (float16, bfloat16 or float32, any strides with contiguous rows)
    into their slots of the cache (mlcv_kv_write): k_cache [pages, KV, page, hd] and v_cache [pages, KV, hd, page]
    float8_e4m3fn, their scales [pages, KV] float32."""
    k, v, cu, slots = _t(k), _t(v), _t(cu_seqlens), _t(slot_map)
    kc, ks, vc, vs = _t(k_cache), _t(k_scale), _t(v_cache), _t(v_scale)
    dev, shape = k.get_device(), kc.shape
    pages, kv, page, hd = shape if len(shape) == 4 else (-1,) * 4
    tokens = k.shape[0] if k.dim() == 3 else -1
    kt, vt = _CODE.get(k.dtype), _CODE.get(v.dtype)
    if not (kt and vt and kc.dtype is _F8 and vc.dtype is _F8 and ks.dtype is _F32 and vs.dtype is _F32
            and cu.dtype is _I32 and slots.dtype is _I32 and k.shape == (tokens, kv, hd) and v.shape == k.shape
            and vc.shape == (pages, kv, hd, page) and ks.shape == (pages, kv) and vs.shape == (pages, kv)
            and slots.shape == (tokens,) and cu.dim() == 1 and cu.shape[0] > 0
            and (k.stride(2) == v.stride(2) == 1 or not tokens * kv * hd) and kc.is_contiguous() and vc.is_contiguous()
            and ks.is_contiguous() and vs.is_contiguous() and cu.is_contiguous() and slots.is_contiguous()
            and dev >= 0 and v.get_device() == kc.get_device() == ks.get_device() == vc.get_device()
            == vs.get_device() == cu.get_device() == slots.get_device() == dev):
        rows, i32 = (tokens, kv, hd) if len(shape) == 4 else (None,) * 3, (_I32,)
        _refuse("kv_write", dev, _cache_wanted(kc, ks, vc, vs)
                + (("k", k, _CODE, (None,) + rows[1:], False), ("v", v, _CODE, rows, False),
                   ("slot_map", slots, i32, (tokens,), True), ("cu_seqlens", cu, i32, (None,), True)))
    ks0, ks1, _ = k.stride()
    vs0, vs1, _ = v.stride()
    _call("mlcv_kv_write", dev, k.data_ptr(), kt, ks0, ks1, v.data_ptr(), vt, vs0, vs1, tokens, cu.data_ptr(),
          cu.shape[0] - 1, slots.data_ptr(), kc.data_ptr(), ks.data_ptr(), vc.data_ptr(), vs.data_ptr(), pages, page,
          kv, hd)


@functools.lru_cache(maxsize=4096)
def kv_attention_workspace(tokens: int, requests: int, heads: int, kv_heads: int, head_dim: int, max_kv: int) -> int:
    """Bytes of workspace of ``kv_attention`` for these sizes (mlcv_kv_attention_workspace)."""
    n = ctypes.c_size_t()
    N.call("mlcv_kv_attention_workspace", tokens, requests, heads, kv_heads, head_dim, max_kv, ctypes.byref(n))
    return n.value


def kv_attention(q, cu_seqlens, kv_lens, block_table, k_cache, k_scale, v_cache, v_scale, *, causal: bool = True,
                 scale: Optional[float] = None, max_kv: Optional[int] = None, out=None, workspace=None) -> Tensor:
    """Attention of the last tokens of each request, q [tokens, H, hd], over its cached keys and values
    (mlcv_kv_attention).  ``scale``: 1 / sqrt(hd) if not given; ``max_kv``: a bound on kv_lens (default: the
    block table's width; one far above the lengths, as a wide table's, splits the keys badly: up to 3.6 times the
    time); ``out``: rows behind the last request are left as they were, so by default they are not initialized;
    ``workspace``: uint8 tensor of ``kv_attention_workspace`` bytes (default: allocated here)."""
    q, cu, lens, table = _t(q), _t(cu_seqlens), _t(kv_lens), _t(block_table)
    kc, ks, vc, vs = _t(k_cache), _t(k_scale), _t(v_cache), _t(v_scale)
    dev, shape, name = q.get_device(), kc.shape, _NAME.get(q.dtype)
    pages, kv, page, hd = shape if len(shape) == 4 else (-1,) * 4
    tokens, heads, d = q.shape if q.dim() == 3 else (-1,) * 3
    n, wide = table.shape if table.dim() == 2 else (-1, 0)
    if not (name and d == hd and kc.dtype is _F8 and vc.dtype is _F8 and ks.dtype is _F32 and vs.dtype is _F32
            and cu.dtype is _I32 and lens.dtype is _I32 and table.dtype is _I32
            and vc.shape == (pages, kv, hd, page) and ks.shape == (pages, kv) and vs.shape == (pages, kv)
            and cu.shape == (n + 1,) and lens.shape == (n,) and (q.stride(2) == 1 or not tokens * heads)
            and kc.is_contiguous() and vc.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()
            and cu.is_contiguous() and lens.is_contiguous() and table.is_contiguous()
            and dev >= 0 and kc.get_device() == ks.get_device() == vc.get_device() == vs.get_device()
            == cu.get_device() == lens.get_device() == table.get_device() == dev):
        i32, b = (_I32,), table.shape[0] if table.dim() else None
        _refuse("kv_attention", dev, (("q", q, _NAME, (None, None, hd if len(shape) == 4 else None), False),)
                + _cache_wanted(kc, ks, vc, vs)
                + (("block_table", table, i32, (None, None), True), ("kv_lens", lens, i32, (b,), True),
                   ("cu_seqlens", cu, i32, (b + 1 if b is not None else None,), True)))
    o = _like(q) if out is None else _given("kv_attention", out, q, dev)
    most = min(wide * page if max_kv is None else max_kv, 0x7fffffff)
    size = kv_attention_workspace(tokens, n, heads, kv, hd, most)
    at = None
    if size:
        if workspace is None:
            workspace = torch.empty(size, dtype=_U8, device=q.device)
        else:
            workspace = _t(workspace)
            size = workspace.numel()
            if not (workspace.dtype is _U8 and workspace.is_contiguous() and workspace.get_device() == dev):
                _refuse("kv_attention", dev, (("workspace", workspace, (_U8,), (None,), True),))
        at = workspace.data_ptr()
    qt, qh, _ = q.stride()
    ot, oh, _ = o.stride()
    _call("mlcv_kv_attention", dev, q.data_ptr(), _CODE[q.dtype], qt, qh, tokens, cu.data_ptr(), n, lens.data_ptr(),
          table.data_ptr(), wide, kc.data_ptr(), ks.data_ptr(), vc.data_ptr(), vs.data_ptr(), pages, page, heads, kv,
          hd, hd ** -0.5 if scale is None else scale, causal, most, o.data_ptr(), ot, oh, at, size)
    return Tensor(o, name)


def prompt_attention(q, k, v, cu_seqlens, *, causal: bool = True, bidir=None, scale: Optional[float] = None,
                     out=None) -> Tensor:
    """Attention of packed prompts, q [tokens, H, hd], k and v [tokens, KV, hd] in float16 or bfloat16
    (mlcv_prompt_attention).  ``bidir`` [B] int32: the first tokens of each prompt that all see one another.  Rows
    that are not 16-byte aligned, and tokens that share keys or values, are copied first.  ``out``: 8-byte aligned
    rows; those behind the last prompt are left as they were, so by default they are not initialized."""
    q, k, v, cu = _t(q), _t(k), _t(v), _t(cu_seqlens)
    dev, dt, name = q.get_device(), q.dtype, _NAME.get(q.dtype)
    tokens, heads, hd = q.shape if q.dim() == 3 else (-1,) * 3
    kv = k.shape[1] if k.dim() == 3 else -1
    n = cu.shape[0] - 1 if cu.dim() == 1 else -1
    if not (name and k.dtype is dt and v.dtype is dt and cu.dtype is _I32 and k.shape == (tokens, kv, hd)
            and v.shape == k.shape and n >= 0 and cu.is_contiguous()
            and (q.stride(2) == k.stride(2) == v.stride(2) == 1 or not tokens * hd)
            and dev >= 0 and k.get_device() == v.get_device() == cu.get_device() == dev):
        t, d = (tokens, hd) if q.dim() == 3 else (None, None)
        _refuse("prompt_attention", dev, (("q", q, _NAME, (None,) * 3, False), ("k", k, (dt,), (t, None, d), False),
                                          ("v", v, (dt,), tuple(k.shape), False),
                                          ("cu_seqlens", cu, (_I32,), (None,), True)))
    pre = None
    if bidir is not None:
        bidir = _t(bidir)
        if not (bidir.dtype is _I32 and bidir.shape == (n,) and bidir.is_contiguous() and bidir.get_device() == dev):
            _refuse("prompt_attention", dev, (("bidir", bidir, (_I32,), (n,), True),))
        pre = bidir.data_ptr()
    o = _like(q) if out is None else _given("prompt_attention", out, q, dev)
    q, k, v = _aligned(q, 0), _aligned(k, hd), _aligned(v, hd)
    qt, qh, _ = q.stride()
    kt, kh, _ = k.stride()
    vt, vh, _ = v.stride()
    ot, oh, _ = o.stride()
    _call("mlcv_prompt_attention", dev, q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, _CODE[dt],
          tokens, cu.data_ptr(), n, heads, kv, hd, hd ** -0.5 if scale is None else scale, causal, pre, o.data_ptr(),
          ot, oh)
    return Tensor(o, name)


def _pool(fn: str, k, k_scale, v, v_scale):
    """A cache's four tensors, of one layer or (with one more dim in front) several: their addresses, and (device, layers,
    pages, KV, page, hd)."""
    kc, ks, vc, vs = _t(k), _t(k_scale), _t(v), _t(v_scale)
    dev, shape = kc.get_device(), tuple(kc.shape)
    size = (1,) + shape if len(shape) == 4 else shape if len(shape) == 5 else (-1,) * 5
    _, pages, kv, page, hd = size
    top = shape[:-2]
    if not (kc.dtype is _F8 and vc.dtype is _F8 and ks.dtype is _F32 and vs.dtype is _F32 and size[0] >= 0
            and vc.shape == top + (hd, page) and ks.shape == top and vs.shape == top and kc.is_contiguous()
            and vc.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()
            and dev >= 0 and ks.get_device() == vc.get_device() == vs.get_device() == dev):
        _refuse(fn, dev, (("k_cache", kc, (_F8,), shape if len(shape) == 5 else (None,) * 4, True),
                          ("k_scale", ks, (_F32,), top, True), ("v_cache", vc, (_F8,), top + (hd, page), True),
                          ("v_scale", vs, (_F32,), top, True)))
    return (kc.data_ptr(), ks.data_ptr(), vc.data_ptr(), vs.data_ptr()), (dev,) + size


def _rows(fn: str, block_table, kv_lens, dev: Optional[int] = None):
    """(table, lengths, device, rows, entries of a row)"""
    table, lens = _t(block_table), _t(kv_lens)
    if dev is None:
        dev = table.get_device()
    n, wide = table.shape if table.dim() == 2 else (-1, 0)
    if not (table.dtype is _I32 and lens.dtype is _I32 and lens.shape == (n,) and table.is_contiguous()
            and lens.is_contiguous() and dev >= 0 and table.get_device() == lens.get_device() == dev):
        b = table.shape[0] if table.dim() else None
        _refuse(fn, dev, (("block_table", table, (_I32,), (None, None), True), ("kv_lens", lens, (_I32,), (b,), True)))
    return table, lens, dev, n, wide


def _outs(fn: str, dev: int, out, shapes):
    """The tensors of ``out`` (a named tuple) checked for their shapes."""
    ts = tuple(_t(x) for x in out)
    if len(ts) != len(shapes):
        _bad(fn, "out", f"is not {len(shapes)} tensors")
    for name, t, s in zip(out._fields, ts, shapes):
        if not (t.dtype is _I32 and t.shape == s and t.is_contiguous() and t.get_device() == dev):
            _refuse(fn, dev, (("out." + name, t, (_I32,), s, True),))
    return ts


def _pages_workspace(name: str, num_pages: int) -> int:
    n = ctypes.c_size_t()
    N.call(name, num_pages, ctypes.byref(n))
    return n.value


@functools.lru_cache(maxsize=256)
def kv_free_workspace(num_pages: int) -> int:
    """Bytes of workspace of ``kv_free`` (mlcv_kv_free_workspace)."""
    return _pages_workspace("mlcv_kv_free_workspace", num_pages)


@functools.lru_cache(maxsize=256)
def kv_compact_workspace(num_pages: int) -> int:
    """Bytes of workspace of ``kv_compact`` (mlcv_kv_compact_workspace)."""
    return _pages_workspace("mlcv_kv_compact_workspace", num_pages)


def _front(size: int, outs: int) -> int:
    """Ints in front of ``outs`` of them that are a call's outputs, for a workspace of ``size`` bytes in their allocation; 0: it is
    to have its own.  One allocation takes 1.3 us less than two, but lives as long as the outputs do: where the workspace is up to
    64 KB or a quarter of them."""
    return (size + 15) // 16 * 4 if size <= max(1 << 16, outs) else 0


def _space(fn: str, workspace, size: int, dev: int):
    w = _t(workspace)
    if not (w.dtype is _U8 and w.is_contiguous() and w.get_device() == dev):
        _refuse(fn, dev, (("workspace", w, (_U8,), (None,), True),))
    return w, w.numel()


def kv_free(block_table, kv_lens, *, num_pages: int, page_size: int, out: Optional[KVFree] = None,
            workspace=None) -> KVFree:
    """The pages that no row of block_table [B, max_pages] holds, as the free list of the next plan or fork
    (mlcv_kv_free).  A finished request's length is 0; one that a plan refused still has its old length."""
    table, lens, dev, n, wide = _rows("kv_free", block_table, kv_lens)
    if not 0 <= num_pages < 1 << 27:
        _bad("kv_free", "num_pages", "is negative or past 2^27 - 1")
    size = kv_free_workspace(num_pages)
    front = _front(size, num_pages + 1) if out is None and workspace is None else 0
    if out is None:
        both = torch.empty(front + num_pages + 1, dtype=_I32, device=table.device)
        pages, count = both.as_strided((num_pages,), (1,), front), both.as_strided((1,), (1,), front + num_pages)
        out = KVFree(Tensor(pages, "int32"), Tensor(count, "int32"))
    else:
        pages, count = _outs("kv_free", dev, out, ((num_pages,), (1,)))
    if workspace is None:
        ws = both if front else torch.empty(size, dtype=_U8, device=table.device)
    else:
        ws, size = _space("kv_free", workspace, size, dev)
    _call("mlcv_kv_free", dev, table.data_ptr(), n, wide, lens.data_ptr(), num_pages, page_size, pages.data_ptr(),
          count.data_ptr(), ws.data_ptr(), size)
    return out


def kv_copy(src, dst, k_cache, k_scale, v_cache, v_scale, *, into=None) -> None:
    """Copy pages src [n] to pages dst [n] (int32), in all layers, within a cache or ``into`` the four tensors of another
    (mlcv_kv_copy).  Caches of one layer [pages, KV, page, hd] or of all [layers, pages, KV, page, hd]."""
    cache, (dev, layers, pages, kv, page, hd) = _pool("kv_copy", k_cache, k_scale, v_cache, v_scale)
    to, size = (cache, None) if into is None else _pool("kv_copy", *into)
    if size is not None and (size[:2] != (dev, layers) or size[3:] != (kv, page, hd)):
        _bad("kv_copy", "into", "is a cache of other layers, heads or pages")
    s, d = _t(src), _t(dst)
    n = s.shape[0] if s.dim() == 1 else -1
    if not (s.dtype is _I32 and d.dtype is _I32 and d.shape == (n,) and s.is_contiguous() and d.is_contiguous()
            and s.get_device() == d.get_device() == dev):
        _refuse("kv_copy", dev, (("src", s, (_I32,), (None,), True), ("dst", d, (_I32,), (n,), True)))
    _call("mlcv_kv_copy", dev, s.data_ptr(), d.data_ptr(), n, *cache, pages, *to, pages if size is None else size[2],
          layers, page, kv, hd)


def kv_fork(parents, block_table, kv_lens, free_pages, k_cache, k_scale, v_cache, v_scale, *, free_count=None,
            out: Optional[KVFork] = None) -> KVFork:
    """Rows that go on from the requests ``parents`` [N] int32 of block_table [B, max_pages] (mlcv_kv_fork): beams,
    samples of one prompt.  Full pages are shared; of a last page that is not full all rows but the first of its parent get a
    copy, on pages from the front of ``free_pages``, of which ``free_count`` [1] are free (default: all).  The old table
    is done with; a request that stays beside its forks is a row of its own."""
    cache, (dev, layers, pages, kv, page, hd) = _pool("kv_fork", k_cache, k_scale, v_cache, v_scale)
    table, lens, _, b, wide = _rows("kv_fork", block_table, kv_lens, dev)
    p, free = _t(parents), _t(free_pages)
    if not (p.dtype is _I32 and free.dtype is _I32 and p.dim() == 1 and free.dim() == 1 and p.is_contiguous()
            and free.is_contiguous() and p.get_device() == free.get_device() == dev):
        _refuse("kv_fork", dev, (("parents", p, (_I32,), (None,), True), ("free_pages", free, (_I32,), (None,), True)))
    n = p.shape[0]
    if out is None:
        both = torch.empty(n * wide + n + 2, dtype=_I32, device=table.device)
        t, m = both.as_strided((n, wide), (wide, 1)), both.as_strided((n,), (1,), n * wide)
        status = both.as_strided((2,), (1,), n * (wide + 1))
        out = KVFork(Tensor(t, "int32"), Tensor(m, "int32"), Tensor(status, "int32"))
    else:
        t, m, status = _outs("kv_fork", dev, out, ((n, wide), (n,), (2,)))
    _call("mlcv_kv_fork", dev, p.data_ptr(), n, table.data_ptr(), b, wide, lens.data_ptr(), free.data_ptr(),
          free.shape[0], None if free_count is None else _count("kv_fork", free_count, dev), *cache, layers, pages, page, kv,
          hd, t.data_ptr(), m.data_ptr(), status.data_ptr())
    return out


def kv_compact(block_table, kv_lens, k_cache, k_scale, v_cache, v_scale, *, out: Optional[KVCompact] = None,
               workspace=None) -> KVCompact:
    """Move the pages in use to the front of the pool, in all layers (mlcv_kv_compact); ``out``: its block table may be
    the given one."""
    cache, (dev, layers, pages, kv, page, hd) = _pool("kv_compact", k_cache, k_scale, v_cache, v_scale)
    table, lens, _, n, wide = _rows("kv_compact", block_table, kv_lens, dev)
    size = kv_compact_workspace(pages)
    front = _front(size, n * wide + 2) if out is None and workspace is None else 0
    if out is None:
        both = torch.empty(front + n * wide + 2, dtype=_I32, device=table.device)
        t, status = both.as_strided((n, wide), (wide, 1), front), both.as_strided((2,), (1,), front + n * wide)
        out = KVCompact(Tensor(t, "int32"), Tensor(status, "int32"))
    else:
        t, status = _outs("kv_compact", dev, out, ((n, wide), (2,)))
    if workspace is None:
        ws = both if front else torch.empty(size, dtype=_U8, device=table.device)
    else:
        ws, size = _space("kv_compact", workspace, size, dev)
    _call("mlcv_kv_compact", dev, table.data_ptr(), n, wide, lens.data_ptr(), *cache, layers, pages, page, kv, hd,
          t.data_ptr(), status.data_ptr(), ws.data_ptr(), size)
    return out


class PagedKVCache:
    """The pages of every layer of a model: ``num_pages`` pages of ``page_size`` tokens (16, 32, 64 or 128) in
    float8_e4m3fn with their scales.  A block table's page numbers are the same in every layer."""

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, layers: int = 1, dev=None):
        if page_size not in (16, 32, 64, 128) or head_dim not in (64, 128, 256):
            raise ValueError("page_size must be 16, 32, 64 or 128 and head_dim 64, 128 or 256")
        if not 0 <= num_pages * page_size <= 2 ** 31 - 256:
            raise ValueError("more than 2^31 - 256 slots")
        d = (dev or device()).torch
        shape = (layers, num_pages, num_kv_heads)
        self.page_size, self.num_pages, self.layers = page_size, num_pages, layers
        self.k = torch.zeros(shape + (page_size, head_dim), dtype=torch.uint8, device=d).view(_F8)
        self.v = torch.zeros(shape + (head_dim, page_size), dtype=torch.uint8, device=d).view(_F8)
        self.k_scale, self.v_scale = (torch.zeros(shape, dtype=torch.float32, device=d) for _ in range(2))

    def pages(self, layer: int = 0):
        """(k_cache, k_scale, v_cache, v_scale) of one layer."""
        return self.k[layer], self.k_scale[layer], self.v[layer], self.v_scale[layer]

    def all_layers(self):
        """(k_cache, k_scale, v_cache, v_scale) of all layers, each with a dim of layers in front."""
        return self.k, self.k_scale, self.v, self.v_scale

    def plan(self, past_lens, new_lens, block_table, free_pages, tokens: int, out: Optional[KVPlan] = None,
             free_count=None) -> KVPlan:
        return kv_plan(past_lens, new_lens, block_table, free_pages, num_pages=self.num_pages,
                       page_size=self.page_size, tokens=tokens, free_count=free_count, out=out)

    def free(self, block_table, kv_lens, **options) -> KVFree:
        return kv_free(block_table, kv_lens, num_pages=self.num_pages, page_size=self.page_size, **options)

    def fork(self, parents, block_table, kv_lens, free_pages, free_count=None, **options) -> KVFork:
        return kv_fork(parents, block_table, kv_lens, free_pages, *self.all_layers(), free_count=free_count, **options)

    def compact(self, block_table, kv_lens, **options) -> KVCompact:
        return kv_compact(block_table, kv_lens, *self.all_layers(), **options)

    def copy(self, src, dst, into: Optional["PagedKVCache"] = None) -> None:
        kv_copy(src, dst, *self.all_layers(), into=None if into is None else into.all_layers())

    def write(self, k, v, plan: KVPlan, layer: int = 0) -> None:
        kv_write(k, v, plan.cu_seqlens, plan.slot_map, *self.pages(layer))

    def attention(self, q, plan: KVPlan, block_table, layer: int = 0, **options) -> Tensor:
        return kv_attention(q, plan.cu_seqlens, plan.kv_lens, block_table, *self.pages(layer), **options)
