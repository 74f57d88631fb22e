"""Dense float64 attention with capped, biased and prefix-masked scores, forward
and backward (test infrastructure).

Q, dO (B, T, H, D), K, V (B, T, Hkv, D); window (left, right) with (-1, 0) causal;
positions (B, T) or None; prefix (B,) or (B, T) or None; slopes (H,) or None.
"""
from __future__ import annotations

import numpy as np


def bounds(T, window, positions, prefix):
    """(lb, ub), each (B or 1, T): the first and last visible key of each query."""
    left, right = window
    if (left, right) == (-1, 0):
        left = T
    q = np.arange(T, dtype=np.int64)[None, :]
    start = np.zeros((1, T), np.int64) if positions is None else np.maximum(q - np.asarray(positions, np.int64), 0)
    lb = np.maximum(start, q - left)
    ub = q + right
    if prefix is not None:
        n = np.asarray(prefix, np.int64)
        n = np.clip(n[:, None] if n.ndim == 1 else n, 0, T)
        ub = np.maximum(ub, start + n - 1)
    return np.broadcast_arrays(lb, np.minimum(ub, T - 1))


def visible(T, window, positions, prefix):
    lb, ub = bounds(T, window, positions, prefix)
    k = np.arange(T)
    return (k >= lb[..., None]) & (k <= ub[..., None])


def _head(q, k, seen, softcap, slope):
    """(x, finished scores) of one head."""
    T = q.shape[0]
    x = q @ k.T / np.sqrt(q.shape[1])
    s = softcap * np.tanh(x / softcap) if softcap > 0 else x
    if slope is not None:
        i = np.arange(T)
        s = s - float(slope) * np.abs(i[:, None] - i[None, :])
    return x, np.where(seen, s, -np.inf)


def forward(Q, K, V, window, positions=None, softcap=0.0, slopes=None, prefix=None):
    """(O, l, m): O float64, l and m (B, H, T); a row without keys has O = 0, l = 0, m = -FLT_MAX."""
    Q, K, V = (np.asarray(a, np.float64) for a in (Q, K, V))
    B, T, H, _ = Q.shape
    group = H // K.shape[2]
    O, l, m = np.zeros(Q.shape), np.zeros((B, H, T)), np.full((B, H, T), float(np.finfo(np.float32).min))
    seen = np.broadcast_to(visible(T, window, positions, prefix), (B, T, T))
    for b in range(B):
        for h in range(H):
            _, s = _head(Q[b, :, h], K[b, :, h // group], seen[b], softcap, None if slopes is None else slopes[h])
            any_ = seen[b].any(-1)
            top = np.where(any_, s.max(-1), 0.0)
            e = np.exp(s - top[:, None])
            l[b, h] = e.sum(-1)
            m[b, h] = np.where(any_, top, m[b, h])
            O[b, :, h] = e @ V[b, :, h // group] / np.where(any_, l[b, h], 1.0)[:, None]
    return O, l, m


def backward(dO, Q, K, V, window, positions=None, softcap=0.0, slopes=None, prefix=None):
    """(dQ, dK, dV); rows with a single visible key have dS = 0."""
    dO, Q, K, V = (np.asarray(a, np.float64) for a in (dO, Q, K, V))
    B, T, H, D = Q.shape
    group = H // K.shape[2]
    dQ, dK, dV = np.zeros(Q.shape), np.zeros(K.shape), np.zeros(V.shape)
    seen = np.broadcast_to(visible(T, window, positions, prefix), (B, T, T))
    for b in range(B):
        many = (seen[b].sum(-1) > 1)[:, None]
        for h in range(H):
            k, v = K[b, :, h // group], V[b, :, h // group]
            x, s = _head(Q[b, :, h], k, seen[b], softcap, None if slopes is None else slopes[h])
            top = np.where(seen[b].any(-1), s.max(-1), 0.0)
            e = np.exp(s - top[:, None])
            p = e / np.maximum(e.sum(-1, keepdims=True), 1e-300)
            dp = dO[b, :, h] @ v.T
            ds = np.where(many, p * (dp - (p * dp).sum(-1, keepdims=True)), 0.0)
            if softcap > 0:
                ds = ds * (1.0 - np.tanh(x / softcap) ** 2)
            dQ[b, :, h] = ds @ k / np.sqrt(D)
            dK[b, :, h // group] += ds.T @ Q[b, :, h] / np.sqrt(D)
            dV[b, :, h // group] += p.T @ dO[b, :, h]
    return dQ, dK, dV
