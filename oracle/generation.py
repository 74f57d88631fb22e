"""Text generation over a cache of keys and values (test infrastructure): the cache's
quantisation in float32 operation by operation, attention of a run or a tree of new
tokens in float64, and the walk that verifies drafted tokens in float64.
"""
from __future__ import annotations

import numpy as np


def round_e4m3(y):
    """float32 values rounded to 8-bit floats of 4 exponent and 3 mantissa bits, ties to even."""
    y = np.asarray(y, np.float32).astype(np.float64)
    e = np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -30)))
    step = 2.0 ** (np.maximum(e, -6) - 3)
    return np.clip(np.rint(y / step) * step, -448.0, 448.0).astype(np.float32)


def quantise(x, kind):
    """(codes as float32 numbers, scales or None) of x (..., D), kind "bf16", "int8" or "fp8"."""
    x = np.asarray(x, np.float32)
    if kind == "bf16":
        u = x.view(np.uint32).astype(np.uint64)
        r = ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)
        return np.where(np.isnan(x), np.float32(np.nan), r), None
    top = np.float32(127.0 if kind == "int8" else 448.0)
    a = np.abs(x).max(-1, keepdims=True)  # (a NaN is the largest)
    small = a < np.float32(2.0 ** -100)
    good = np.isfinite(a)
    safe = np.where(good & ~small, a, np.float32(1.0))
    y = np.where(good & ~small, np.where(good, x, 0) * (top / safe), np.float32(0.0))
    codes = np.rint(y) if kind == "int8" else round_e4m3(y)
    scale = np.where(good, np.where(small, np.float32(0.0), safe / top), np.float32(np.nan))
    return codes.astype(np.float32), scale[..., 0].astype(np.float32)


def held(x, kind):
    """x as the cache gives it back (float32)."""
    codes, scale = quantise(x, kind)
    return codes if scale is None else codes * scale[..., None]


def lineage(parents, N):
    """For each node its ancestors and itself, root first; None where the parents are no tree's."""
    up = list(range(-1, N - 1)) if parents is None else [int(p) for p in parents]
    lines = []
    for i in range(N):
        line, at = [i], i
        while line is not None and up[at] != -1:
            if not 0 <= up[at] < at:
                line = None
                break
            at = up[at]
            line.insert(0, at)
        lines.append(line)
    return lines


def attend(Q, K, V, length, count, left=-1, parents=None, softcap=0.0, slopes=None):
    """O (N, H, D) of one sequence: Q (N, H, D), K and V (length + count, Hkv, D), the nodes'
    last.  Zeros from node `count` on, NaN for a node that is in no tree."""
    Q, K, V = (np.asarray(a, np.float64) for a in (Q, K, V))
    N, H, D = Q.shape
    O = np.zeros(Q.shape)
    lines = lineage(None if parents is None else parents[:N], N)
    for i in range(count):
        if lines[i] is None:
            O[i] = np.nan
            continue
        depth = len(lines[i]) - 1
        keys = list(range(length)) + [length + j for j in lines[i]]
        far = np.array([length + depth - t for t in range(length)] + [depth - n for n in range(depth + 1)])
        if left >= 0:
            keys, far = [k for k, f in zip(keys, far) if f <= left], far[far <= left]
        for h in range(H):
            k, v = K[keys, h // (H // K.shape[1])], V[keys, h // (H // K.shape[1])]
            s = k @ Q[i, h] / np.sqrt(D)
            if softcap > 0:
                s = softcap * np.tanh(s / softcap)
            if slopes is not None:
                s = s - float(slopes[h]) * far
            e = np.exp(s - s.max())
            O[i, h] = (e / e.sum()) @ v
    return O


def softmax(x, temperature):
    x = np.asarray(x, np.float64)
    with np.errstate(invalid="ignore"):
        e = np.exp((x - x.max(-1, keepdims=True)) / temperature)
        return e / e.sum(-1, keepdims=True)


def draw(w, u):
    """The first index whose cumulative weight is above u of the whole."""
    c = np.cumsum(w)
    return int(np.nonzero(c > u * c[-1])[0][0])


def verify(logits, tokens, u, draft_logits=None, parents=None, count=None, temperature=1.0):
    """(path, token) of one sequence: logits (N, V), tokens and u (N,), draft_logits (N - 1, V)."""
    N, V = logits.shape
    count = N if count is None else count
    if count == 0:
        return [], -1
    up = list(range(-1, N - 1)) if parents is None else [int(p) for p in parents]
    path = [0]
    while True:
        at = path[-1]
        row = np.asarray(logits[at], np.float64)
        if np.isnan(row).any() or row.max() == np.inf or row.max() == -np.inf:
            return path, -1
        children = [i for i in range(1, count) if up[i] == at]
        if temperature == 0:
            best = int(np.argmax(row))
            taken = [i for i in children if tokens[i] == best]
            if not taken:
                return path, best
            path.append(taken[0])
            continue
        p = softmax(row, temperature)
        left, tried, taken = 1.0, [], None
        for i in children:
            x = int(tokens[i])
            if not 0 <= x < V:
                continue
            if draft_logits is not None:
                q = softmax(draft_logits[i - 1], temperature)
                if u[i] * q[x] < p[x]:
                    taken = i
                else:
                    rest = np.maximum(p - q, 0.0)
                    return path, draw(rest if rest.sum() > 2.0 ** -40 else p, float(u[0]))  # (less is roundings)
            elif x not in tried:
                if u[i] * left < p[x]:
                    taken = i
                else:
                    left -= p[x]
                    tried.append(x)
            if taken is not None:
                break
        if taken is None:
            w = p.copy()
            w[tried] = 0.0
            return path, draw(w if w.sum() > 0 else p, float(u[0]))
        path.append(taken)
