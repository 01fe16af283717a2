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
from typing import NamedTuple, Optional

import torch

from . import _native as N
from .runtime import Tensor, device

_CODE = {torch.float16: N.MLCV_DTYPE_F16, torch.float32: N.MLCV_DTYPE_F32, torch.bfloat16: N.MLCV_DTYPE_BF16}
_NAME = {torch.float16: "float16", torch.bfloat16: "bfloat16", torch.int32: "int32"}
_HALF = (torch.float16, torch.bfloat16)
_F8 = torch.float8_e4m3fn


class KVPlan(NamedTuple):
    """What ``kv_plan`` made: see mlcv_kv_plan."""

    cu_seqlens: Tensor  # [B + 1] first token of each request
    kv_lens: Tensor     # [B] cached tokens after the new ones are written; 0: the request was refused
    slot_map: Tensor    # [tokens] slot of each new token, -1: none
    status: Tensor      # [2] pages taken from the front of the free list; requests refused


def _t(x) -> torch.Tensor:
    t = x.torch if isinstance(x, Tensor) else x
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"expected a device tensor, got {type(x).__name__}")
    return t


def _arg(fn: str, name: str, x, dtypes, shape, like: Optional[torch.Tensor] = None,
         dense: bool = True) -> torch.Tensor:
    """The torch tensor of argument ``name``: its dtype one of ``dtypes``, its shape ``shape`` (None: any size),
    on the device of ``like``, contiguous (or, with ``dense`` false, with contiguous rows)."""
    t = _t(x)
    if t.dtype not in dtypes:
        raise ValueError(f"{fn}: argument {name} has dtype {t.dtype}")
    if t.dim() != len(shape) or any(w is not None and w != s for w, s in zip(shape, t.shape)):
        raise ValueError(f"{fn}: argument {name} expects shape {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_cuda or (like is not None and t.device != like.device):
        raise ValueError(f"{fn}: argument {name} is not on the HIP device of the other tensors")
    if not (t.is_contiguous() if dense else t.stride(-1) == 1 or t.shape[-1] == 1 or t.numel() == 0):
        raise ValueError(f"{fn}: argument {name} must {'be contiguous' if dense else 'have contiguous rows'}")
    return t


def _call(name: str, t: torch.Tensor, *args) -> None:
    """One native call on the device and the current stream of ``t``."""
    i = t.device.index
    if i == torch.cuda.current_device():
        N.check(getattr(N.load(), name)(*args, torch.cuda.current_stream(i).cuda_stream))
    else:
        with torch.cuda.device(i):
            N.check(getattr(N.load(), name)(*args, torch.cuda.current_stream(i).cuda_stream))


def _rows16(t: torch.Tensor, low: int = 0) -> torch.Tensor:
    """``t`` [tokens, heads, hd] of 16-bit elements with 16-byte aligned rows, its tokens at least ``low`` and less
    than 2^24 elements apart: itself, or a copy."""
    a, b, _ = t.stride()
    return t if t.data_ptr() % 16 == 0 and a % 8 == 0 and b % 8 == 0 and low <= a < 1 << 24 else t.contiguous().clone() \
        if t.is_contiguous() else t.contiguous()


def _out(fn: str, out, q: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    return _arg(fn, "out", out, (q.dtype,), q.shape, q, dense=False)


def _scale(scale: Optional[float], hd: int) -> float:
    return hd ** -0.5 if scale is None else float(scale)


def kv_plan(past_lens, new_lens, block_table, free_pages, *, num_pages: int, page_size: int, tokens: int,
            out: Optional[KVPlan] = None) -> KVPlan:
    """Block tables and slot maps from request lengths (mlcv_kv_plan).

    past_lens, new_lens [B], block_table [B, max_pages] (its new entries are written), free_pages [F], all int32;
    ``tokens``: the packed tokens of the call.  ``out``: a plan of the same sizes to write into."""
    i32 = (torch.int32,)
    past = _arg("kv_plan", "past_lens", past_lens, i32, (None,))
    n = past.shape[0]
    new = _arg("kv_plan", "new_lens", new_lens, i32, (n,), past)
    table = _arg("kv_plan", "block_table", block_table, i32, (n, None), past)
    free = _arg("kv_plan", "free_pages", free_pages, i32, (None,), past)
    tokens = int(tokens)
    if tokens < 0:
        raise ValueError("kv_plan: tokens is negative")
    if out is None:
        out = KVPlan(*(Tensor(torch.empty(s, dtype=torch.int32, device=past.device), "int32")
                       for s in (n + 1, n, tokens, 2)))
    cu, lens, slots, status = (_arg("kv_plan", "out", x, i32, (s,), past)
                               for x, s in zip(out, (n + 1, n, tokens, 2)))
    _call("mlcv_kv_plan", past, past.data_ptr(), new.data_ptr(), n, free.data_ptr(), free.shape[0], int(num_pages),
          int(page_size), table.data_ptr(), table.shape[1], cu.data_ptr(), lens.data_ptr(), slots.data_ptr(), tokens,
          status.data_ptr())
    return out


def _cache_args(fn: str, k_cache, k_scale, v_cache, v_scale, like: torch.Tensor):
    kc = _arg(fn, "k_cache", k_cache, (_F8,), (None,) * 4, like)
    pages, kv, page, hd = kc.shape
    vc = _arg(fn, "v_cache", v_cache, (_F8,), (pages, kv, hd, page), like)
    ks = _arg(fn, "k_scale", k_scale, (torch.float32,), (pages, kv), like)
    vs = _arg(fn, "v_scale", v_scale, (torch.float32,), (pages, kv), like)
    return kc, ks, vc, vs


def kv_write(k, v, cu_seqlens, slot_map, k_cache, k_scale, v_cache, v_scale) -> None:
    """Write new keys and values [tokens, KV, hd] (float16, bfloat16 or float32, any strides with contiguous rows)
    into their slots of the cache (mlcv_kv_write): k_cache [pages, KV, page, hd] and v_cache [pages, KV, hd, page]
    float8_e4m3fn, their scales [pages, KV] float32."""
    k = _arg("kv_write", "k", k, _CODE, (None,) * 3, None, dense=False)
    v = _arg("kv_write", "v", v, _CODE, k.shape, k, dense=False)
    cu = _arg("kv_write", "cu_seqlens", cu_seqlens, (torch.int32,), (None,), k)
    slots = _arg("kv_write", "slot_map", slot_map, (torch.int32,), (k.shape[0],), k)
    kc, ks, vc, vs = _cache_args("kv_write", k_cache, k_scale, v_cache, v_scale, k)
    pages, kv, page, hd = kc.shape
    if k.shape[1:] != (kv, hd):
        raise ValueError(f"kv_write: argument k expects {kv} heads of {hd}, got {tuple(k.shape[1:])}")
    _call("mlcv_kv_write", k, k.data_ptr(), _CODE[k.dtype], k.stride(0), k.stride(1), v.data_ptr(), _CODE[v.dtype],
          v.stride(0), v.stride(1), k.shape[0], cu.data_ptr(), max(0, cu.shape[0] - 1), slots.data_ptr(),
          kc.data_ptr(), ks.data_ptr(), vc.data_ptr(), vs.data_ptr(), pages, page, kv, hd)


def kv_attention_workspace(tokens: int, requests: int, heads: int, kv_heads: int, head_dim: int, max_kv: int) -> int:
    """Bytes of workspace of ``kv_attention`` for these sizes (mlcv_kv_attention_workspace)."""
    n = ctypes.c_size_t()
    N.call("mlcv_kv_attention_workspace", int(tokens), int(requests), int(heads), int(kv_heads), int(head_dim),
           int(max_kv), ctypes.byref(n))
    return n.value


def kv_attention(q, cu_seqlens, kv_lens, block_table, k_cache, k_scale, v_cache, v_scale, *, causal: bool = True,
                 scale: Optional[float] = None, max_kv: Optional[int] = None, out=None, workspace=None) -> Tensor:
    """Attention of the last tokens of each request, q [tokens, H, hd], over its cached keys and values
    (mlcv_kv_attention).  ``scale``: 1 / sqrt(hd) if not given; ``max_kv``: a bound on kv_lens (default: the
    block table's width); ``workspace``: uint8 tensor of ``kv_attention_workspace`` bytes (default: allocated here)."""
    q = _arg("kv_attention", "q", q, _HALF, (None,) * 3, None, dense=False)
    kc, ks, vc, vs = _cache_args("kv_attention", k_cache, k_scale, v_cache, v_scale, q)
    pages, kv, page, hd = kc.shape
    if q.shape[2] != hd:
        raise ValueError(f"kv_attention: argument q expects head_dim {hd}, got {q.shape[2]}")
    i32 = (torch.int32,)
    lens = _arg("kv_attention", "kv_lens", kv_lens, i32, (None,), q)
    n = lens.shape[0]
    cu = _arg("kv_attention", "cu_seqlens", cu_seqlens, i32, (n + 1,), q)
    table = _arg("kv_attention", "block_table", block_table, i32, (n, None), q)
    o = _out("kv_attention", out, q)
    most = table.shape[1] * page if max_kv is None else int(max_kv)
    tokens, heads, _ = q.shape
    need = kv_attention_workspace(tokens, n, heads, kv, hd, most)
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if workspace is None else \
            _arg("kv_attention", "workspace", workspace, (torch.uint8,), (None,), q)
        at, size = ws.data_ptr(), ws.numel()
    else:
        at, size = None, 0
    _call("mlcv_kv_attention", q, q.data_ptr(), _CODE[q.dtype], q.stride(0), q.stride(1), tokens, cu.data_ptr(), n,
          lens.data_ptr(), table.data_ptr(), table.shape[1], kc.data_ptr(), ks.data_ptr(), vc.data_ptr(),
          vs.data_ptr(), pages, page, heads, kv, hd, _scale(scale, hd), int(bool(causal)), most, o.data_ptr(),
          o.stride(0), o.stride(1), at, size)
    return Tensor(o, _NAME[q.dtype])


def prompt_attention(q, k, v, cu_seqlens, *, causal: bool = True, bidir=None, scale: Optional[float] = None,
                     out=None) -> Tensor:
    """Attention of packed prompts, q [tokens, H, hd], k and v [tokens, KV, hd] in float16 or bfloat16
    (mlcv_prompt_attention).  ``bidir`` [B] int32: the first tokens of each prompt that all see one another."""
    q = _arg("prompt_attention", "q", q, _HALF, (None,) * 3, None, dense=False)
    tokens, heads, hd = q.shape
    k = _arg("prompt_attention", "k", k, (q.dtype,), (tokens, None, hd), q, dense=False)
    kv = k.shape[1]
    v = _arg("prompt_attention", "v", v, (q.dtype,), k.shape, q, dense=False)
    i32 = (torch.int32,)
    cu = _arg("prompt_attention", "cu_seqlens", cu_seqlens, i32, (None,), q)
    n = max(0, cu.shape[0] - 1)
    pre = None if bidir is None else _arg("prompt_attention", "bidir", bidir, i32, (n,), q).data_ptr()
    o = _out("prompt_attention", out, q)
    q, k, v = _rows16(q), _rows16(k, hd), _rows16(v, hd)
    _call("mlcv_prompt_attention", q, q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
          v.data_ptr(), v.stride(0), v.stride(1), _CODE[q.dtype], tokens, cu.data_ptr(), n, heads, kv, hd,
          _scale(scale, hd), int(bool(causal)), pre, o.data_ptr(), o.stride(0), o.stride(1))
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
