"""The policy and preference losses over answers in float64 (test infrastructure).

logits (answers, T, V), tokens (answers, T) zero-based; tokens equal to ``ignore``
have no loss and no gradient.  Each function returns the losses and the gradient
of sum(dy * losses), dy broadcast over them.
"""
from __future__ import annotations

import numpy as np


def log_probs(logits, tokens, ignore=-1):
    """(lp, softmax), both 0 where ignored."""
    x = np.asarray(logits, np.float64)
    on = np.asarray(tokens) != ignore
    m = x.max(-1, keepdims=True)
    e = np.exp(x - m)
    s = e.sum(-1, keepdims=True)
    y = np.where(on, tokens, 0)[..., None]
    lp = (np.take_along_axis(x, y, -1) - m - np.log(s))[..., 0]
    return np.where(on, lp, 0.0), np.where(on[..., None], e / s, 0.0)


def _spread(w, p, tokens, ignore):
    """w (onehot - softmax) of every token."""
    g = -w[..., None] * p
    on = np.asarray(tokens) != ignore
    y = np.where(on, tokens, 0)[..., None]
    np.put_along_axis(g, y, np.take_along_axis(g, y, -1) + np.where(on, w, 0.0)[..., None], -1)
    return g


def policy(logits, tokens, old, advantages, ref=None, clip=(0.2, 0.2), kl=0.0, ignore=-1, dy=1.0):
    lp, p = log_probs(logits, tokens, ignore)
    on = np.asarray(tokens) != ignore
    A = np.asarray(advantages, np.float64)
    A = np.broadcast_to(A[:, None] if A.ndim == 1 else A, lp.shape)
    r = np.exp(lp - np.asarray(old, np.float64))
    free, cut = r * A, np.clip(r, 1.0 - clip[0], 1.0 + clip[1]) * A
    loss, w = -np.minimum(free, cut), np.where(free <= cut, -free, 0.0)
    if kl > 0:
        d = np.asarray(ref, np.float64) - lp
        loss, w = loss + kl * (np.exp(d) - d - 1.0), w + kl * (1.0 - np.exp(d))
    loss, w = np.where(on, loss, 0.0), np.where(on, w, 0.0)
    return loss, _spread(w * dy, p, tokens, ignore), w


def preference(logits, tokens, ref, beta=0.1, smoothing=0.0, ignore=-1, dy=1.0):
    lp, p = log_probs(logits, tokens, ignore)
    P = lp.shape[0] // 2
    rewards = beta * (lp.sum(-1) - np.asarray(ref, np.float64))
    h = rewards[:P] - rewards[P:]
    loss = (1.0 - smoothing) * np.logaddexp(0.0, -h) + smoothing * np.logaddexp(0.0, h)
    sig = np.exp(-np.logaddexp(0.0, -h))
    dh = beta * (smoothing * sig - (1.0 - smoothing) * np.exp(-np.logaddexp(0.0, h)))
    w = np.concatenate([dh, -dh])
    dyw = np.broadcast_to(np.asarray(dy, np.float64), (P,))
    full = np.broadcast_to((w * np.concatenate([dyw, dyw]))[:, None], lp.shape)
    return loss, rewards, _spread(full, p, tokens, ignore), w
