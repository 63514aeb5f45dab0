"""Oracle of prompt attention and of 8-bit caches, in float64 numpy, from their
definitions: what each query sees is written out key by key, caches are written
token run by token run.

  oracle_prefill   packed causal attention, with the bound terms of a test
  oracle_append    8-bit cache write (elements as the numbers they hold)
  oracle_decode    one query per sequence over cached values
"""
from __future__ import annotations

import numpy as np

TOP = {"e4m3": 448.0, "int8": 127.0}


def attend(q, k, v, scale):
    """q [D], k and v [n, D]: out, sum of weight |v|, largest sum of |q k| scale, weights."""
    s = (k @ q) * scale
    w = np.exp(s - s.max())
    w /= w.sum()
    return w @ v, w @ np.abs(v), (np.abs(k) @ np.abs(q)).max() * scale, w


def oracle_prefill(q, key, value, cu, cu_k, window, sinks, scale):
    """q [Tq, Hq, D], key and value [Tk, Hkv, D] float64.  Returns out, and per row
    the sum of weight times |value| and the largest sum of |q k| scale."""
    Tq, Hq, D = q.shape
    group = Hq // key.shape[1]
    out, spread, size = np.zeros_like(q), np.zeros_like(q), np.zeros((Tq, Hq))
    cu_k = cu if cu_k is None else cu_k
    for b in range(len(cu) - 1):
        nq, nk = cu[b + 1] - cu[b], cu_k[b + 1] - cu_k[b]
        k, v = key[cu_k[b]:cu_k[b + 1]], value[cu_k[b]:cu_k[b + 1]]
        for i in range(nq):
            at = nk - nq + i
            seen = [j for j in range(nk) if j <= at and (window == 0 or j > at - window or j < sinks)]
            if not seen:
                continue
            for h in range(Hq):
                t = cu[b] + i
                out[t, h], spread[t, h], size[t, h], _ = attend(q[t, h], k[seen, h // group], v[seen, h // group], scale)
    return out, spread, size


def round_to(x, kind):
    """x on the grid of the type, ties to even; |x| at most the type's largest value."""
    x = np.asarray(x, dtype=np.float64)
    if kind == "int8":
        return np.rint(x)
    _, e = np.frexp(np.abs(x))          # |x| = m 2^e, m in [0.5, 1)
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.rint(x / step) * step


def power_scale(most, kind):
    """The smallest power of two s >= 2^-100 with most <= s * TOP; NaN where most is not finite or s passes 2^100."""
    if not np.isfinite(most):
        return np.nan
    e = -100
    while most > np.ldexp(TOP[kind], e):
        e += 1
    return np.ldexp(1.0, e) if e <= 100 else np.nan


def oracle_append(key, value, k_cache, v_cache, k_scales, v_scales, table, positions, cu, kind):
    """Float64 arrays, caches hold elements; cu None: a token per sequence.  Returns the four as new arrays."""
    found = []
    N, P = k_cache.shape[:2]
    for rows, cache, scales in ((key, k_cache, k_scales), (value, v_cache, v_scales)):
        cache, scales = cache.copy(), scales.copy()
        for b in range(len(positions)):
            lo, hi = (b, b + 1) if cu is None else (cu[b], cu[b + 1])
            at, end = int(positions[b]), int(positions[b]) + hi - lo
            if at < 0:
                continue
            first = at
            while at < end:
                stop = min(end, (at // P + 1) * P)
                page = at // P
                phys = int(table[b, page]) if page < table.shape[1] else -1
                if 0 <= phys < N:
                    new = rows[lo + at - first:lo + stop - first]
                    for h in range(cache.shape[2]):
                        with np.errstate(invalid="ignore"):
                            scale = power_scale(np.max(np.abs(new[:, h])), kind)
                        if at % P:
                            old = scales[phys, h]
                            scale = np.nan if np.isnan(old) or np.isnan(scale) else old if abs(old) >= scale else scale
                            if scale != old:
                                cache[phys, :at % P, h] = round_to(cache[phys, :at % P, h] * (old / scale), kind)
                        with np.errstate(invalid="ignore"):
                            cache[phys, at % P:at % P + stop - at, h] = round_to(new[:, h] / scale, kind)
                        scales[phys, h] = scale
                at = stop
        found += [cache, scales]
    return found[0], found[2], found[1], found[3]


def cached_rows(cache, scales, table_row, n):
    """Values of tokens 0 .. n - 1 of a sequence [n, Hkv, D] and the scales of their pages [n, Hkv]."""
    N, P = cache.shape[:2]
    tok = np.arange(n)
    phys = np.clip(table_row[tok // P].astype(np.int64), 0, N - 1)
    return cache[phys, tok % P] * scales[phys][:, :, None], scales[phys]


def oracle_decode(q, k_cache, v_cache, k_scales, v_scales, table, lens, scale):
    """q [B, Hq, D].  Returns out, spread and size as oracle_prefill, and per row the largest weight times the
    scale of its values' page."""
    B, Hq, D = q.shape
    P, Hkv = k_cache.shape[1:3]
    out, spread, size, top = np.zeros_like(q), np.zeros_like(q), np.zeros((B, Hq)), np.zeros((B, Hq))
    for b in range(B):
        n = min(max(int(lens[b]), 0), table.shape[1] * P)
        if n == 0:
            continue
        k, _ = cached_rows(k_cache, k_scales, table[b], n)
        v, vs = cached_rows(v_cache, v_scales, table[b], n)
        for h in range(Hq):
            g = h // (Hq // Hkv)
            out[b, h], spread[b, h], size[b, h], w = attend(q[b, h], k[:, g], v[:, g], scale)
            top[b, h] = np.max(w * np.abs(vs[:, g]))
    return out, spread, size, top
