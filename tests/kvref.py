"""Plain implementations of the request entry points (mlc_vla.kv_cache) in 64 bits on the CPU, and the bounds that
a result may differ by."""

from __future__ import annotations

import numpy as np
import torch


def plan(past, new, table, free, num_pages, page, tokens):
    """What mlcv_kv_plan documents, request by request.  `table` is written."""
    b, wide = table.shape
    cu, lens, slots = [0], [], np.full(tokens, -1, np.int64)
    at, end, refused, dry = 0, 0, 0, False
    for i in range(b):
        n = max(int(new[i]), 0)
        start, end = end, end + n
        cu.append(min(end, tokens))
        had, has = -(-int(past[i]) // page), -(-(int(past[i]) + n) // page)
        ok = past[i] >= 0 and new[i] >= 0 and has <= wide and end <= tokens
        need = has - had if ok else 0
        if need and (dry or at + need > len(free)):
            ok, dry = False, True
        if not ok:
            refused += 1
            lens.append(0)
            continue
        table[i, had:has] = free[at:at + need]
        at += need
        lens.append(int(past[i]) + n)
        for t in range(n):
            pos = int(past[i]) + t
            pg = int(table[i, pos // page])
            if 0 <= pg < num_pages:
                slots[start + t] = pg * page + pos % page
    return np.array(cu), np.array(lens, np.int64), slots, np.array([at, refused])


def e4m3(x):
    """float64 -> the nearest e4m3 value (ties to even), saturating at 448; NaN stays."""
    x = np.clip(x, -448.0, 448.0)
    with np.errstate(divide="ignore"):
        step = np.exp2(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6))) - 3)
    return np.round(x / step) * step


def scale_for(amax):
    e = -64
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def write(x, cu, slots, data, scale, page):
    """x [tokens, KV, hd] float64 into data [pages, KV, page, hd] (code values) and scale [pages, KV], in place."""
    pages, kv = scale.shape
    for a, z in zip(cu, cu[1:]):
        t = a
        while t < z:
            o = int(slots[t]) % page
            # the tokens that the request's own offset puts on one page
            first = int(slots[a]) % page
            stop = a + page - first if t == a else t + page
            stop = min(stop, z)
            n = 0
            while t + n < stop and slots[t] >= 0 and slots[t + n] == slots[t] + n and o + n < page:
                n += 1
            pg = int(slots[t]) // page
            if slots[t] >= 0 and pg < pages and n and (t == a or o == 0):
                part = x[t:t + n].transpose(1, 0, 2)
                for h in range(kv):
                    fin = np.abs(part[h][np.isfinite(part[h])])
                    want = scale_for(fin.max() if fin.size else 0.0)
                    now = max(want, scale[pg, h]) if o else want
                    if o:
                        data[pg, h, :o] = e4m3(data[pg, h, :o] * (scale[pg, h] / now))
                    data[pg, h, o:o + n] = e4m3(part[h] / now)
                    scale[pg, h] = now
            t = stop
    return data, scale


def attend(q, k, v, limit, scale):
    """q [n, H, d], k, v [L, KV, d] float64, limit [n]: (outputs, softmax @ |v|, largest scale * sum|q||k|) of
    each row over the keys that it sees; a row that sees none is zero."""
    n, h, d = q.shape
    out, mass, big = np.zeros((n, h, d)), np.zeros((n, h, d)), np.zeros((n, h, 1))
    grp = h // k.shape[1]
    for i in range(n):
        m = int(limit[i])
        if m <= 0:
            continue
        for j in range(h):
            kk, vv = k[:m, j // grp], v[:m, j // grp]
            x = kk @ q[i, j] * scale
            with np.errstate(invalid="ignore", over="ignore"):
                p = np.exp(x - x.max())
                p /= p.sum()
                out[i, j] = (p[:, None] * vv).sum(0)
                mass[i, j] = (p[:, None] * np.abs(vv)).sum(0)
                big[i, j] = (np.abs(kk) @ np.abs(q[i, j]) * scale).max()
    return out, mass, big


def bound(out, mass, big, dtype, keys, hd, weights, tiny):
    """How far a float32 computation with weights rounded to `weights` and results rounded to `dtype` may be from
    the 64-bit values.  With u = half a step of a type:
      output rounding              u(dtype) |o|
      each weight's rounding       u(weights) sum p |v|, and `keys` times `tiny`, what the absolute step of a
                                   weight below fp16's normal range is worth (0 for bfloat16 weights)
      logits: hd products summed in float32 and two more roundings, each 2^-24 relative to sum |q||k|, in units
      of log2 (1.45), and the hardware's exponential (2 steps of float32): a relative change of every weight, in
      numerator and sum
      sums over the keys           keys 2^-24 sum p |v|, and as much for the sum of the weights
    """
    u, w = torch.finfo(dtype).eps / 2, torch.finfo(weights).eps / 2
    logits = (2.0 ** -24) * (hd + 4) * big * 1.45 + 2.0 ** -22
    rel = w + 2 * logits + 2 * keys * 2.0 ** -24
    return u * np.abs(out) + (rel * mass + keys * tiny) * (1 + u) + torch.finfo(dtype).smallest_normal * u
