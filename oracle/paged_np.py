"""Plain 64-bit restatements of the paged-cache and logits operators (test infrastructure).

Written row by row from the definitions in include/aria_q4.h; no attempt at speed.
Caches are given as lists of rows per sequence, so that paging stays out of it.
"""
from __future__ import annotations

import numpy as np


def attend(q, keys, vals, scale, present=None):
    """q [Hq][dh]; keys, vals [n][Hkv][dh]; present: bool [n] (absent slots take no part).
    Returns out [Hq][dh], lse [Hq], p [Hq][n] in float64."""
    q, keys, vals = (np.asarray(x, dtype=np.float64) for x in (q, keys, vals))
    Hq, dh = q.shape
    n, Hkv = keys.shape[0], keys.shape[1]
    G = Hq // Hkv
    on = np.ones(n, dtype=bool) if present is None else np.asarray(present)
    out, lse, p = np.zeros((Hq, dh)), np.full(Hq, -np.inf), np.zeros((Hq, n))
    if not on.any():
        return out, lse, p
    idx = np.flatnonzero(on)
    for h in range(Hq):
        s = scale * (keys[idx, h // G] @ q[h])
        m = s.max()
        lse[h] = m + np.log(np.exp(s - m).sum())
        p[h, idx] = np.exp(s - lse[h])
        out[h] = p[h, idx] @ vals[idx, h // G]
    return out, lse, p


def prompt_weights(q, k, scale, first=0, lse=None):
    """q [T][Hq][dh], k [T][Hkv][dh] -> (weights [Hkv][T], lse [Hq][T]) of causal attention;
    lse given: used as is (-inf rows give nothing)."""
    q, k = np.asarray(q, dtype=np.float64), np.asarray(k, dtype=np.float64)
    T, Hq, _ = q.shape
    Hkv = k.shape[1]
    G = Hq // Hkv
    w, rows = np.zeros((Hkv, T)), np.zeros((Hq, T))
    for h in range(Hq):
        for t in range(T):
            if lse is not None and t < first:
                continue
            s = scale * (k[:t + 1, h // G] @ q[t, h])
            m = s.max()
            rows[h, t] = m + np.log(np.exp(s - m).sum()) if lse is None else lse[h, t]
            if t >= first and rows[h, t] != -np.inf:
                w[h // G, :t + 1] += np.exp(s - rows[h, t])
    return w, rows


def evict_row(w, pos, next_pos, keep, recent, sinks):
    """One row of n slots -> (moves [(from, to)], new weights, new positions)."""
    n = len(w)
    w, pos = np.array(w, dtype=np.float32), np.array(pos)
    if n <= keep:
        return [], w, pos
    safe = (pos >= next_pos - recent) | (pos < sinks)

    def rank(i):  # kept positions first, then the largest weights, NaN last, ties by slot
        if safe[i]:
            return (0, 0.0, i)
        return (2, 0.0, i) if np.isnan(w[i]) else (1, -float(w[i]), i)

    kept = set(sorted(range(n), key=rank)[:keep])
    to = [i for i in range(keep) if i not in kept]
    frm = sorted(i for i in kept if i >= keep)
    nw, npos = w.copy(), pos.copy()
    for f, t in zip(frm, to):
        nw[t], npos[t] = w[f], pos[f]
    nw[keep:], npos[keep:] = 0.0, -1
    return list(zip(frm, to)), nw, npos


def adjust_row(x, history=(), prompt_len=0, repetition=1.0, frequency=0.0, presence=0.0, biases=(), allowed=None):
    """x [V] -> (adjusted [V] float64, index of the largest or -1)."""
    x = np.array(x, dtype=np.float64)
    V = len(x)
    hist = [(i, t) for i, t in enumerate(history) if 0 <= t < V]
    for t in {t for _, t in hist}:
        x[t] = x[t] / repetition if x[t] > 0 else x[t] * repetition
    said = [t for i, t in hist if i >= prompt_len]
    for t in set(said):
        x[t] = x[t] - frequency * said.count(t) - presence
    for t, b in biases:
        if 0 <= t < V:
            x[t] += b
    if allowed is not None:
        x[~np.asarray(allowed)] = -np.inf
    y = np.where(np.isnan(x), -np.inf, x)
    best = int(np.argmax(y))
    return x, (best if y[best] > -np.inf else -1)
