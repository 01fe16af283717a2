"""What logits say: log probabilities of given tokens, entropy and the best alternatives, for generating text.

No counterpart in the reference.  The function body is one call into ``libmlcvla_hip.so`` (include/mlcvla.h says what
it computes); tensors are ``runtime.Tensor`` or torch tensors on one HIP device, on whose current stream the work runs.
Nothing synchronizes, so a decode step can be captured into a graph.
"""

from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple, Optional

import torch

from . import _native as N
from .kv_cache import _CODE, _F32, _I32, _U8, _bad, _call, _refuse, _t
from .runtime import Tensor


class TokenLogprobs(NamedTuple):
    """What ``token_logprobs`` made: see mlcv_token_logprobs.  All of float32 but the ids, which are int32."""

    logprobs: Optional[Tensor]      # like tokens; None without them
    entropy: Tensor                 # [rows]
    top_ids: Optional[Tensor]       # [rows, top]; None without alternatives
    top_logprobs: Optional[Tensor]  # [rows, top]


@functools.lru_cache(maxsize=4096)
def token_logprobs_workspace(rows: int, vocab: int, top: int) -> int:
    """Bytes of workspace of ``token_logprobs`` for these sizes (mlcv_token_logprobs_workspace)."""
    n = ctypes.c_size_t()
    N.call("mlcv_token_logprobs_workspace", rows, vocab, top, ctypes.byref(n))
    return n.value


def token_logprobs(logits, tokens=None, *, top: int = 0, scale: float = 1.0, out: Optional[TokenLogprobs] = None,
                   workspace=None) -> TokenLogprobs:
    """Log probabilities under softmax(scale * logits), logits [rows, vocab] in float16, bfloat16 or float32 with
    contiguous rows (mlcv_token_logprobs).

    tokens [rows] or [rows, n] int32: the given tokens; one outside [0, vocab) counts 0.  ``top``: how many alternatives, up
    to 64, the likeliest first and equal logits by their index.  ``out``: contiguous tensors of the same sizes to write into,
    which share nothing with the inputs or one another; ``workspace``: uint8 tensor of ``token_logprobs_workspace`` bytes
    (default: allocated here)."""
    x = _t(logits)
    dev, code = x.get_device(), _CODE.get(x.dtype)
    rows, vocab = x.shape if x.dim() == 2 else (-1, -1)
    if not (code and rows >= 0 and dev >= 0 and (x.stride(1) == 1 or vocab == 1 or not rows)):
        _refuse("token_logprobs", dev, (("logits", x, _CODE, (None, None), False),))
    if not isinstance(top, int) or top < 0:
        _bad("token_logprobs", "top", "is not a number of alternatives")
    given, at, shape = 0, None, None
    if tokens is not None:
        t = _t(tokens)
        shape = t.shape
        given = 1 if t.dim() == 1 else shape[-1] if shape else -1
        if not (t.dtype is _I32 and t.dim() in (1, 2) and shape[0] == rows and t.is_contiguous()
                and t.get_device() == dev):
            _refuse("token_logprobs", dev, (("tokens", t, (_I32,), (rows,) if t.dim() < 2 else (rows, None), True),))
        at = t.data_ptr()
    size = token_logprobs_workspace(rows, vocab, top)
    if out is None:
        # one allocation: given tokens, entropy, alternatives' ids and log probabilities
        n = rows * given
        f = torch.empty(n + rows * (1 + 2 * top), dtype=_F32, device=x.device)
        h = f.as_strided((rows,), (1,), n)
        lp = ids = tlp = given_lp = top_ids = top_lp = None
        if at is not None:
            lp = f.as_strided(shape, (1,) if len(shape) == 1 else (given, 1))
            given_lp = Tensor(lp, "float32")
        if top:
            ids = f.view(_I32).as_strided((rows, top), (top, 1), n + rows)
            tlp = f.as_strided((rows, top), (top, 1), n + rows * (1 + top))
            top_ids, top_lp = Tensor(ids, "int32"), Tensor(tlp, "float32")
        out = TokenLogprobs(given_lp, Tensor(h, "float32"), top_ids, top_lp)
    else:
        lp, h, ids, tlp = (None if o is None else _t(o) for o in out)
        for name, o, dt, want in (("logprobs", lp, _F32, shape), ("entropy", h, _F32, (rows,)),
                                  ("top_ids", ids, _I32, (rows, top) if top else None),
                                  ("top_logprobs", tlp, _F32, (rows, top) if top else None)):
            if (o is None) != (want is None):
                _bad("token_logprobs", "out." + name, "is missing" if o is None else "has nothing to hold")
            if o is not None and not (o.dtype is dt and o.shape == want and o.is_contiguous() and o.get_device() == dev):
                _refuse("token_logprobs", dev, (("out." + name, o, (dt,), want, True),))
    ws = None
    if size:
        if workspace is None:
            workspace = torch.empty(size, dtype=_U8, device=x.device)
        else:
            workspace = _t(workspace)
            size = workspace.numel()
            if not (workspace.dtype is _U8 and workspace.is_contiguous() and workspace.get_device() == dev):
                _refuse("token_logprobs", dev, (("workspace", workspace, (_U8,), (None,), True),))
        ws = workspace.data_ptr()
    _call("mlcv_token_logprobs", dev, x.data_ptr(), code, x.stride(0), rows, vocab, scale, at, given,
          lp.data_ptr() if given else None, h.data_ptr(), top, ids.data_ptr() if top else None,
          tlp.data_ptr() if top else None, ws, size)
    return out
