"""Several requests at once: packed prompts and a paged 8-bit key/value cache.

No counterpart in the reference, which serves one request over a dense cache.  Tokens of the
requests are packed one after another, ``cu_seqlens`` [B + 1] int32 says where each begins, and every
length stays on the device: nothing here synchronizes, so a serving step can be captured into a graph.

    plan = kv_plan(past, new, table, free, num_pages=..., page_size=64, tokens=T)   # slots of the new tokens
    out = prompt_attention(q, k, v, plan.cu_seqlens)                                # a prompt's own attention
    cache.write(k, v, plan, layer)                                                  # into the pages
    out = cache.attention(q, plan, table, layer)                                    # later tokens

Every function body is one call into ``libmlcvla_hip.so`` (include/mlcvla.h says what each computes);
tensors are ``runtime.Tensor`` or torch tensors on one HIP device, on whose current stream the work runs.
Keys and values of any strides with contiguous rows are taken in place.
"""

from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple, Optional

import torch

from . import _native as N
from .runtime import Tensor, device

_F16, _BF16, _F32, _I32, _U8 = torch.float16, torch.bfloat16, torch.float32, torch.int32, torch.uint8
_F8 = torch.float8_e4m3fn
_CODE = {_F16: N.MLCV_DTYPE_F16, _F32: N.MLCV_DTYPE_F32, _BF16: N.MLCV_DTYPE_BF16}
_NAME = {_F16: "float16", _BF16: "bfloat16"}


class KVPlan(NamedTuple):
    """What ``kv_plan`` made: see mlcv_kv_plan."""

    cu_seqlens: Tensor  # [B + 1] first token of each request
    kv_lens: Tensor     # [B] cached tokens after the new ones are written; 0: the request was refused
    slot_map: Tensor    # [tokens] slot of each new token, -1: none
    status: Tensor      # [2] pages taken from the front of the free list; requests refused


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
    return torch.empty_like(q) if q.is_contiguous() else torch.empty(q.shape, dtype=q.dtype, device=q.device)


def _given(fn: str, out, q: torch.Tensor, dev: int) -> torch.Tensor:
    o = _t(out)
    if not (o.shape == q.shape and o.dtype is q.dtype and o.get_device() == dev
            and (o.stride(2) == 1 or not o.numel())):
        _refuse(fn, dev, (("out", o, (q.dtype,), q.shape, False),))
    return o


def kv_plan(past_lens, new_lens, block_table, free_pages, *, num_pages: int, page_size: int, tokens: int,
            out: Optional[KVPlan] = None) -> KVPlan:
    """Block tables and slot maps from request lengths (mlcv_kv_plan).

    past_lens, new_lens [B], block_table [B, max_pages] (its new entries are written), free_pages [F], all int32;
    ``tokens``: the packed tokens of the call.  ``out``: a plan of the same sizes to write into; not the one whose
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
    _call("mlcv_kv_plan", dev, past.data_ptr(), new.data_ptr(), n, free.data_ptr(), free.shape[0], num_pages,
          page_size, table.data_ptr(), wide, cu.data_ptr(), lens.data_ptr(), slots.data_ptr(), tokens,
          status.data_ptr())
    return out


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

    def plan(self, past_lens, new_lens, block_table, free_pages, tokens: int, out: Optional[KVPlan] = None) -> KVPlan:
        return kv_plan(past_lens, new_lens, block_table, free_pages, num_pages=self.num_pages,
                       page_size=self.page_size, tokens=tokens, out=out)

    def write(self, k, v, plan: KVPlan, layer: int = 0) -> None:
        kv_write(k, v, plan.cu_seqlens, plan.slot_map, *self.pages(layer))

    def attention(self, q, plan: KVPlan, block_table, layer: int = 0, **options) -> Tensor:
        return kv_attention(q, plan.cu_seqlens, plan.kv_lens, block_table, *self.pages(layer), **options)
