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


# The checks below run on every call of a serving loop, whose kernels take a few microseconds: they read the
# tensors' attributes once and build nothing.
def _t(x) -> torch.Tensor:
    if type(x) is Tensor:
        return x.torch
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"expected a device tensor, got {type(x).__name__}")
    return x


def _bad(fn: str, name: str, what: str):
    raise ValueError(f"{fn}: argument {name} {what}")


def _dense(fn: str, name: str, x, dtype, shape, dev: int) -> torch.Tensor:
    """The torch tensor of argument ``name``, which has to be contiguous, of ``dtype`` and ``shape``, on HIP device
    ``dev`` (None: any)."""
    t = _t(x)
    if t.dtype is not dtype:
        _bad(fn, name, f"has dtype {t.dtype}, not {dtype}")
    if t.shape != shape:
        _bad(fn, name, f"expects shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.get_device() != dev:
        _bad(fn, name, "is not on the HIP device of the other tensors")
    if not t.is_contiguous():
        _bad(fn, name, "must be contiguous")
    return t


def _rows(fn: str, name: str, x, dtypes, dev: Optional[int] = None) -> torch.Tensor:
    """The torch tensor of argument ``name``: [tokens, heads, hd] of one of ``dtypes`` with contiguous rows, on HIP
    device ``dev`` (None: any)."""
    t = _t(x)
    if t.dtype not in dtypes:
        _bad(fn, name, f"has dtype {t.dtype}")
    if t.dim() != 3:
        _bad(fn, name, f"expects shape [tokens, heads, head_dim], got {tuple(t.shape)}")
    i = t.get_device()
    if i < 0 or (dev is not None and i != dev):
        _bad(fn, name, "is not on the HIP device of the other tensors")
    if t.stride(2) != 1 and t.numel() > 0:
        _bad(fn, name, "must have contiguous rows")
    return t


def _ids(fn: str, name: str, x) -> torch.Tensor:
    """A contiguous int32 vector on a HIP device."""
    t = _t(x)
    if t.dtype is not _I32:
        _bad(fn, name, f"has dtype {t.dtype}, not {_I32}")
    if t.dim() != 1 or not t.is_contiguous():
        _bad(fn, name, "must be a contiguous vector")
    if t.get_device() < 0:
        _bad(fn, name, "is not on a HIP device")
    return t


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


def _out(fn: str, out, q: torch.Tensor, dev: int) -> torch.Tensor:
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    o = _rows(fn, "out", out, (q.dtype,), dev)
    if o.shape != q.shape:
        _bad(fn, "out", f"expects shape {tuple(q.shape)}, got {tuple(o.shape)}")
    return o


def kv_plan(past_lens, new_lens, block_table, free_pages, *, num_pages: int, page_size: int, tokens: int,
            out: Optional[KVPlan] = None) -> KVPlan:
    """Block tables and slot maps from request lengths (mlcv_kv_plan).

    past_lens, new_lens [B], block_table [B, max_pages] (its new entries are written), free_pages [F], all int32;
    ``tokens``: the packed tokens of the call.  ``out``: a plan of the same sizes to write into."""
    past, free = _ids("kv_plan", "past_lens", past_lens), _ids("kv_plan", "free_pages", free_pages)
    table = _t(block_table)
    n, dev, tokens = past.shape[0], past.get_device(), int(tokens)
    new = _dense("kv_plan", "new_lens", new_lens, _I32, (n,), dev)
    if table.dim() != 2:
        _bad("kv_plan", "block_table", f"expects shape [requests, max_pages], got {tuple(table.shape)}")
    wide = table.shape[1]
    _dense("kv_plan", "block_table", table, _I32, (n, wide), dev)
    if free.get_device() != dev:
        _bad("kv_plan", "free_pages", "is not on the HIP device of the other tensors")
    if tokens < 0:
        _bad("kv_plan", "tokens", "is negative")
    if out is None:
        cu, lens, slots, status = torch.empty(tokens + 2 * n + 3, dtype=_I32, device=past.device).split(
            (n + 1, n, tokens, 2))
        out = KVPlan(Tensor(cu, "int32"), Tensor(lens, "int32"), Tensor(slots, "int32"), Tensor(status, "int32"))
    else:
        cu, lens, slots, status = (_dense("kv_plan", "out", x, _I32, (s,), dev)
                                   for x, s in zip(out, (n + 1, n, tokens, 2)))
    _call("mlcv_kv_plan", dev, past.data_ptr(), new.data_ptr(), n, free.data_ptr(), free.shape[0], num_pages,
          page_size, table.data_ptr(), wide, cu.data_ptr(), lens.data_ptr(), slots.data_ptr(), tokens,
          status.data_ptr())
    return out


def _cache(fn: str, k_cache, k_scale, v_cache, v_scale, dev: int):
    kc = _t(k_cache)
    if kc.dim() != 4:
        _bad(fn, "k_cache", f"expects shape [pages, heads, page, head_dim], got {tuple(kc.shape)}")
    pages, kv, page, hd = shape = kc.shape
    _dense(fn, "k_cache", kc, _F8, shape, dev)
    return (kc.data_ptr(), _dense(fn, "k_scale", k_scale, _F32, (pages, kv), dev).data_ptr(),
            _dense(fn, "v_cache", v_cache, _F8, (pages, kv, hd, page), dev).data_ptr(),
            _dense(fn, "v_scale", v_scale, _F32, (pages, kv), dev).data_ptr(), pages, page), kv, hd


def kv_write(k, v, cu_seqlens, slot_map, k_cache, k_scale, v_cache, v_scale) -> None:
    """Write new keys and values [tokens, KV, hd] (float16, bfloat16 or float32, any strides with contiguous rows)
    into their slots of the cache (mlcv_kv_write): k_cache [pages, KV, page, hd] and v_cache [pages, KV, hd, page]
    float8_e4m3fn, their scales [pages, KV] float32."""
    k = _rows("kv_write", "k", k, _CODE)
    dev, tokens = k.get_device(), k.shape[0]
    v = _rows("kv_write", "v", v, _CODE, dev)
    cache, kv, hd = _cache("kv_write", k_cache, k_scale, v_cache, v_scale, dev)
    if k.shape != (tokens, kv, hd) or v.shape != k.shape:
        _bad("kv_write", "k or v", f"expects shape {(tokens, kv, hd)}, got {tuple(k.shape)}, {tuple(v.shape)}")
    cu = _ids("kv_write", "cu_seqlens", cu_seqlens)
    if cu.get_device() != dev or cu.shape[0] < 1:
        _bad("kv_write", "cu_seqlens", "expects requests + 1 offsets on the HIP device of the other tensors")
    slots = _dense("kv_write", "slot_map", slot_map, _I32, (tokens,), dev)
    kt, kh, _ = k.stride()
    vt, vh, _ = v.stride()
    _call("mlcv_kv_write", dev, k.data_ptr(), _CODE[k.dtype], kt, kh, v.data_ptr(), _CODE[v.dtype], vt, vh, tokens,
          cu.data_ptr(), cu.shape[0] - 1, slots.data_ptr(), *cache, kv, hd)


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
    block table's width); ``workspace``: uint8 tensor of ``kv_attention_workspace`` bytes (default: allocated here)."""
    q = _rows("kv_attention", "q", q, _NAME)
    dev = q.get_device()
    cache, kv, hd = _cache("kv_attention", k_cache, k_scale, v_cache, v_scale, dev)
    tokens, heads, d = q.shape
    if d != hd:
        _bad("kv_attention", "q", f"expects head_dim {hd}, got {d}")
    table = _t(block_table)
    if table.dim() != 2:
        _bad("kv_attention", "block_table", f"expects shape [requests, max_pages], got {tuple(table.shape)}")
    n, wide = table.shape
    _dense("kv_attention", "block_table", table, _I32, (n, wide), dev)
    lens = _dense("kv_attention", "kv_lens", kv_lens, _I32, (n,), dev)
    cu = _dense("kv_attention", "cu_seqlens", cu_seqlens, _I32, (n + 1,), dev)
    o = _out("kv_attention", out, q, dev)
    most = wide * cache[5] if max_kv is None else max_kv
    size = kv_attention_workspace(tokens, n, heads, kv, hd, most)
    at = None
    if size:
        if workspace is None:
            workspace = torch.empty(size, dtype=_U8, device=q.device)
        else:
            workspace = _t(workspace)
            size = workspace.numel()
            _dense("kv_attention", "workspace", workspace, _U8, (size,), dev)
        at = workspace.data_ptr()
    qt, qh, _ = q.stride()
    ot, oh, _ = o.stride()
    _call("mlcv_kv_attention", dev, q.data_ptr(), _CODE[q.dtype], qt, qh, tokens, cu.data_ptr(), n, lens.data_ptr(),
          table.data_ptr(), wide, *cache, heads, kv, hd, hd ** -0.5 if scale is None else scale, causal, most,
          o.data_ptr(), ot, oh, at, size)
    return Tensor(o, _NAME[q.dtype])


def prompt_attention(q, k, v, cu_seqlens, *, causal: bool = True, bidir=None, scale: Optional[float] = None,
                     out=None) -> Tensor:
    """Attention of packed prompts, q [tokens, H, hd], k and v [tokens, KV, hd] in float16 or bfloat16
    (mlcv_prompt_attention).  ``bidir`` [B] int32: the first tokens of each prompt that all see one another."""
    q = _rows("prompt_attention", "q", q, _NAME)
    dev, dt = q.get_device(), (q.dtype,)
    tokens, heads, hd = q.shape
    k = _rows("prompt_attention", "k", k, dt, dev)
    kv = k.shape[1]
    v = _rows("prompt_attention", "v", v, dt, dev)
    if k.shape != (tokens, kv, hd) or v.shape != k.shape:
        _bad("prompt_attention", "k or v", f"expects shape [{tokens}, KV, {hd}], got {(*k.shape,)}, {(*v.shape,)}")
    cu = _ids("prompt_attention", "cu_seqlens", cu_seqlens)
    n = cu.shape[0] - 1
    if cu.get_device() != dev or n < 0:
        _bad("prompt_attention", "cu_seqlens", "expects requests + 1 offsets on the HIP device of the other tensors")
    pre = None if bidir is None else _dense("prompt_attention", "bidir", bidir, _I32, (n,), dev).data_ptr()
    o = _out("prompt_attention", out, q, dev)
    q, k, v = _aligned(q, 0), _aligned(k, hd), _aligned(v, hd)
    qt, qh, _ = q.stride()
    kt, kh, _ = k.stride()
    vt, vh, _ = v.stride()
    ot, oh, _ = o.stride()
    _call("mlcv_prompt_attention", dev, q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh,
          _CODE[q.dtype], tokens, cu.data_ptr(), n, heads, kv, hd, hd ** -0.5 if scale is None else scale, causal, pre,
          o.data_ptr(), ot, oh)
    return Tensor(o, _NAME[q.dtype])


class PagedKVCache:
    """The pages of every layer of a model: ``num_pages`` pages of ``page_size`` tokens (16, 32, 64 or 128) in
    float8_e4m3fn with their scales.  A block table's page numbers are the same in every layer."""

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, layers: int = 1, dev=None):
        if page_size not in (16, 32, 64, 128) or head_dim not in (64, 128, 256):
            raise ValueError("page_size must be 16, 32, 64 or 128 and head_dim 64, 128 or 256")
        if num_pages * page_size > 2 ** 31 - 1:
            raise ValueError("more than 2^31 - 1 slots")
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
