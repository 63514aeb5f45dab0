"""Oracle of the operators around decoding with drafted tokens, in float64
numpy, from their definitions: what each query sees is written out token by
token, nothing is skipped or tiled.

  oracle_tree     windowed and tree attention (mask None: one query, the last
                  token of its sequence), with the bound terms of a test
  oracle_write    per-head RMS norm, rotation, cache write
  oracle_compact  rows of accepted drafted tokens moved next to the context
"""
from __future__ import annotations

import numpy as np


def visible(length, masks, count, capacity, window, sinks):
    """bool [queries, length + count]: which context and drafted tokens each
    query sees.  ``masks`` None: one query at position length - 1."""
    length = min(max(length, 0), capacity)
    if masks is None:
        own = [length - 1]
        place = list(range(length))
        drafted = [None] * length
    else:
        masks = [m & ((1 << count) - 1) for m in masks]
        depth = [bin(m).count("1") - 1 for m in masks]
        own = [length + d for d in depth]
        place = list(range(length)) + own
        drafted = [None] * length + list(range(count))
    sees = np.zeros((len(own), len(place)), dtype=bool)
    for t in range(len(own)):
        if masks is not None and masks[t] == 0:
            continue
        for i, (at, j) in enumerate(zip(place, drafted)):
            if j is not None and (not masks[t] >> j & 1 or length + j >= capacity):
                continue
            sees[t, i] = window == 0 or at > own[t] - window or at < sinks
    return sees


def oracle_tree(q, k_cache, v_cache, table, lens, masks, window, sinks, scale):
    """q [B, T, Hq, D] float64 (T = 1 without masks); caches float64; masks int
    [B][T] or None.  Returns out [B, T, Hq, D], and per row the sum of weight
    times |value| [B, T, Hq, D] and the largest sum of |q k| scale [B, T, Hq]."""
    B, T, Hq, D = q.shape
    N, P, Hkv, _ = k_cache.shape
    cap = table.shape[1] * P
    out, spread, size = np.zeros_like(q), np.zeros_like(q), np.zeros((B, T, Hq))
    for b in range(B):
        n = min(max(int(lens[b]), 0), cap)
        sees = visible(int(lens[b]), None if masks is None else masks[b], T, cap, window, sinks)
        for t in range(T):
            toks = np.nonzero(sees[t])[0]
            if not len(toks):
                continue
            phys = np.clip(table[b, toks // P].astype(np.int64), 0, N - 1)
            k, v = k_cache[phys, toks % P], v_cache[phys, toks % P]
            for hq in range(Hq):
                h = hq // (Hq // Hkv)
                s = (k[:, h] @ q[b, t, hq]) * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                out[b, t, hq] = w @ v[:, h]
                spread[b, t, hq] = w @ np.abs(v[:, h])
                size[b, t, hq] = (np.abs(k[:, h]) @ np.abs(q[b, t, hq])).max() * scale
    return out, spread, size


def oracle_write(q, key, value, cos_sin, positions, k_cache, v_cache, slots, q_weight, k_weight, eps, interleaved):
    """Float64 arrays; returns (q_out, k_cache, v_cache) as new arrays."""
    k_cache, v_cache, q_out = k_cache.copy(), v_cache.copy(), np.zeros_like(q)
    flat_k, flat_v = (c.reshape(-1, *c.shape[2:]) for c in (k_cache, v_cache))
    rot = cos_sin.shape[1]

    def turn(x, weight, at):
        if weight is not None:
            x = x / np.sqrt((x ** 2).mean() + eps) * weight
        y = x.copy()
        for i in range(rot // 2):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
            c, s = cos_sin[at, i], cos_sin[at, rot // 2 + i]
            y[a], y[b] = x[a] * c - x[b] * s, x[b] * c + x[a] * s
        return y

    for n in range(q.shape[0]):
        at, slot = int(positions[n]), int(slots[n])
        if not 0 <= at < cos_sin.shape[0]:
            continue
        for h in range(q.shape[1]):
            q_out[n, h] = turn(q[n, h], q_weight, at)
        if 0 <= slot < flat_k.shape[0]:
            for h in range(key.shape[1]):
                flat_k[slot, h] = turn(key[n, h], k_weight, at)
            flat_v[slot] = value[n]
    return q_out, k_cache, v_cache


def oracle_compact(cache, table, lens, accepted):
    """Returns the compacted copy of one cache [N, P, ...]."""
    N, P = cache.shape[:2]
    after = cache.copy()

    def place(b, tok):
        if tok < 0 or tok >= table.shape[1] * P or not 0 <= table[b, tok // P] < N:
            return None
        return int(table[b, tok // P]), tok % P

    for b in range(accepted.shape[0]):
        for i, a in enumerate(accepted[b].tolist()):
            if a < 0 or lens[b] < 0:
                continue
            src, dst = place(b, int(lens[b]) + a), place(b, int(lens[b]) + i)
            if src is not None and dst is not None:
                after[dst] = cache[src]
    return after
