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


def logprobs(x, scale, tokens, top):
    """x [rows, vocab] float64 -> (log probabilities of tokens [rows, n] or None, entropy, ids, their log probabilities)."""
    rows, vocab = x.shape
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        z = x * scale
        m = z.max(1, keepdims=True)
        e = np.exp(z - np.where(np.isfinite(m), m, 0.0))
        s = e.sum(1, keepdims=True)
        lp = (z - np.where(np.isfinite(m), m, 0.0)) - np.log(s)  # m + ln s would lose ln s next to logits of 1e38
        p = e / s
        h = -np.where(p > 0, p * lp, 0.0).sum(1)
    lp[lp < -np.finfo(np.float32).max] = -np.inf  # what the results' type cannot hold
    none, bad = (m == -np.inf)[:, 0], np.isnan(x).any(1) | (x == np.inf).any(1)
    lp[none], h[none] = -np.inf, 0.0
    lp[bad], h[bad] = np.nan, np.nan
    got = None
    if tokens is not None:
        there = (tokens >= 0) & (tokens < vocab)
        got = np.where(there, np.take_along_axis(lp, np.where(there, tokens, 0), 1), 0.0)
    # largest first, equal ones by their index, NaN behind -inf
    rank = np.where(np.isnan(x), -np.inf, x)
    ids = np.stack([np.lexsort((np.arange(vocab), np.isnan(r), -q))[:top] for r, q in zip(x, rank)]) \
        if rows else np.zeros((0, top), int)
    return got, h, ids, np.take_along_axis(lp, ids, 1)


def logprobs_bound(x, scale, vocab):
    """(bound of each log probability given its value, bound of the entropy), per row, as functions of what is compared.
    With w the spread of scaled logits that carry weight (those further than 104 below the largest are below the smallest
    float32) and u = 2^-24:
      exponents     scale * log2(e) rounded (1 u of |z|, of every term the same factor but for its distance from the
                    largest: w), one fused product (w), the hardware's exponential 2 u: a weight is off by (2 w + 2) u
      sums          up to vocab terms of one sign, in chains of at most vocab / 256 + 32: that many u
      logarithm     2 u of ln s (at most ln vocab), and of a log probability the subtraction, product and sum: 3 u of it"""
    with np.errstate(invalid="ignore", over="ignore"):
        z = x * scale
        m = np.max(np.where(np.isfinite(z), z, -np.inf), 1, keepdims=True)
        d = np.where(np.isfinite(z), m - z, 0.0)
    w = np.where(d < 104, d, 0.0).max(1)
    chain = vocab / 256 + 32
    rel = (2 * w + 2 + chain + 8) * E32           # of s, and of u
    base = 1.1 * (rel + 2 * E32 * np.log(vocab + 1))
    return (lambda lp: base[:, None] + 4 * E32 * np.abs(lp)), base + 2 * rel * (np.log(vocab) + 1) + 4 * E32 * np.log(vocab + 1)


def used_pages(table, lens, num_pages, page):
    """(pages in use, which entries of the table hold one)."""
    b, wide = table.shape
    held = np.arange(wide)[None, :] < -(-np.clip(lens, 0, wide * page) // page)[:, None]
    held &= (table >= 0) & (table < num_pages)
    return np.unique(table[held]), held


def free(table, lens, num_pages, page):
    used, _ = used_pages(table, lens, num_pages, page)
    rest = np.setdiff1d(np.arange(num_pages), used)
    return np.concatenate([rest, np.full(num_pages - len(rest), -1)]), len(rest)


def fork(parents, table, lens, free_pages, page):
    """What mlcv_kv_fork documents, row by row: (table, lengths, status, pairs of pages copied)."""
    b, wide = table.shape
    out, got = np.full((len(parents), wide), -1), np.zeros(len(parents), int)
    seen, pairs, refused = set(), [], 0
    for i, p in enumerate(parents):
        if not 0 <= p < b:
            continue
        n = int(np.clip(lens[p], 0, wide * page))
        has = -(-n // page)
        if n % page and p in seen:
            if len(pairs) == len(free_pages):
                refused += 1
                continue
            out[i, :has] = table[p, :has]
            out[i, has - 1] = free_pages[len(pairs)]
            pairs.append((table[p, has - 1], free_pages[len(pairs)]))
        else:
            out[i, :has] = table[p, :has]
        seen.add(p)
        got[i] = n
    return out, got, np.array([len(pairs), refused]), pairs


def compact(table, lens, num_pages, page):
    """(table, status, pairs of pages moved)."""
    used, held = used_pages(table, lens, num_pages, page)
    m = len(used)
    src = used[used >= m]
    dst = np.setdiff1d(np.arange(m), used)
    to = dict(zip(src.tolist(), dst.tolist()))
    out = table.copy()
    out[held] = [to.get(int(e), int(e)) for e in table[held]]
    return out, np.array([m, len(src)]), list(zip(src, dst))
