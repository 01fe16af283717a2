"""Plain implementations in 64 bits on the CPU of what a decode step of several requests needs around its attention
(mlc_vla.kv_cache.qk_rope, kv_copy, kv_fork, kv_compact, kv_free; mlc_vla.logits), and the bounds of their results."""

from __future__ import annotations

import numpy as np
import torch

E32 = 2.0 ** -24  # half a step of float32, relative


def places(cu, lens, tokens):
    """Positions of packed tokens, and which tokens belong to a request."""
    pos, there = np.zeros(tokens, np.int64), np.zeros(tokens, bool)
    for b in range(len(lens)):
        for i, t in enumerate(range(cu[b], cu[b + 1])):
            pos[t], there[t] = lens[b] - (cu[b + 1] - cu[b]) + i, True
    return pos, there


def rope(x, pos, rd, theta, norm=False, weight=None, offset=1.0, eps=1e-6):
    """x [tokens, heads, hd] float64 -> (result, size of what each result is a sum of)."""
    y = x
    if norm:
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        if weight is not None:
            y = y * (offset + weight)
    # long double: a float64 angle at position 2^31 is off by 2^-22
    freq = np.array([np.longdouble(theta) ** (np.longdouble(-2 * i) / max(rd, 1)) for i in range(rd // 2)], np.longdouble)
    ang = np.asarray(pos, np.longdouble)[:, None, None] * freq
    c, s = np.cos(ang).astype(np.float64), np.sin(ang).astype(np.float64)
    out, size = y.copy(), np.abs(y)
    a, b = y[..., :rd // 2], y[..., rd // 2:rd]
    out[..., :rd // 2], out[..., rd // 2:rd] = a * c - b * s, b * c + a * s
    size[..., :rd // 2] = size[..., rd // 2:rd] = np.abs(a) + np.abs(b)
    return out, size


def rope_bound(out, size, dtype, hd, pos, norm):
    """How far a result may be.
      output rounding      u(dtype) |out|, and half the smallest subnormal
      angle                the rest of a turn as float32 (2 pi 2^-26), frequencies from five float64 products and powers
                           (8 half steps of 2^-53 of the turns, at most pos / (2 pi), times 2 pi)
      sine and cosine      pi as float32, the polynomials' steps and ends: 6 half steps of float32
      products and sum     3 half steps
      norm                 hd products and sums, mean, eps, root, reciprocal and two products: hd + 8 half steps
    the last four relative to |y_i| + |y_j|."""
    rel = (2 * np.pi * 2.0 ** -26 + 8 * 2.0 ** -53 * np.abs(np.asarray(pos, np.float64))[:, None, None]
           + (9 + (hd + 8 if norm else 0)) * E32)
    f = torch.finfo(dtype)
    return f.eps / 2 * np.abs(out) + rel * size * (1 + f.eps) + f.smallest_normal * f.eps / 2
