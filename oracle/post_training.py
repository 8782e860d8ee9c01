"""Float64 oracle of the post-training losses: log-probabilities and entropies of soft-capped
logits, the clipped policy loss and the preference loss, with their gradients by the logits.

Written from the definitions, row by row where that is plainer; checked against autograd and
differences in tests/test_token_loss_cpu.py.  The reference has no counterparts.
"""

from __future__ import annotations

import numpy as np


def rows(logits, targets, vocab, cap, ignore=-1):
    """(log-probabilities, entropies, z, p) of [rows, columns] logits; zeros in rows without a
    target, NaN log-probabilities where the target is none of the vocabulary."""
    z = cap * np.tanh(np.asarray(logits, np.float64)[:, :vocab] / cap)
    top = z.max(axis=1, keepdims=True)
    lse = top + np.log(np.exp(z - top).sum(axis=1, keepdims=True))
    p = np.exp(z - lse)
    ent = (lse - (p * z).sum(axis=1, keepdims=True))[:, 0]
    logp = np.zeros(len(z))
    for r, t in enumerate(targets):
        if t == ignore:
            ent[r] = 0.0
        else:
            logp[r] = z[r, t] - lse[r, 0] if 0 <= t < vocab else np.nan
    return logp, ent, z, p


def logit_grad(logits, targets, vocab, cap, g, h=None, ignore=-1):
    """Gradient [rows, columns] for upstream gradients g of the log-probabilities, h of the
    entropies: d z_j = g ([j = t] - p_j) - h p_j (log p_j + H), times dz/dl = 1 - (z / cap)^2."""
    _, ent, z, p = rows(logits, targets, vocab, cap, ignore)
    out = np.zeros(np.shape(logits))
    for r, t in enumerate(targets):
        if t == ignore:
            continue
        d = -g[r] * p[r]
        d[t] += g[r]
        if h is not None:
            d = d - h[r] * p[r] * (np.log(p[r]) + ent[r])
        out[r, :vocab] = d * (1 - (z[r] / cap) ** 2)
    return out


def policy(logp, targets, old, adv, ref, weights, lo, hi, kl_coef, ignore=-1):
    """(loss, KL, weight of the clipped rows, d loss / d logp)."""
    on = np.asarray(targets) != ignore
    w = on / on.sum() if weights is None else np.where(on, weights, 0.0)
    loss = kl = share = 0.0
    slope = np.zeros(len(logp))
    for r in np.flatnonzero(w):
        q = np.exp(logp[r] - old[r])
        surrogate = min(q * adv[r], min(max(q, lo), hi) * adv[r])
        clipped = surrogate < q * adv[r]
        d = 0.0 if ref is None else ref[r] - logp[r]
        k = np.expm1(d) - d
        loss += w[r] * (-surrogate + kl_coef * k)
        kl += w[r] * k
        share += w[r] * clipped
        slope[r] = w[r] * ((0.0 if clipped else -q * adv[r]) - kl_coef * np.expm1(d))
    return loss, kl, share, slope


def preference(logp, targets, starts, ref, beta, smoothing, average, ignore=-1):
    """(loss, sequence log-probabilities, margins, d loss / d logp of every row)."""
    pairs = (len(starts) - 1) // 2
    spans = [range(a, b) for a, b in zip(starts, starts[1:])]
    count = [max(1, sum(targets[r] != ignore for r in s)) if average else 1 for s in spans]
    seq = np.array([sum(logp[r] for r in s) / n for s, n in zip(spans, count)])
    gain = seq - (0.0 if ref is None else ref)
    m = beta * (gain[:pairs] - gain[pairs:])
    loss = np.mean((1 - smoothing) * np.logaddexp(0, -m) + smoothing * np.logaddexp(0, m))
    up, down = np.exp(-np.logaddexp(0, -m)), np.exp(-np.logaddexp(0, m))  # sigmoid(m), sigmoid(-m)
    dm = (smoothing * up - (1 - smoothing) * down) * beta / pairs
    slope = np.zeros(len(logp))
    for i, (s, n) in enumerate(zip(spans, count)):
        for r in s:
            slope[r] = (dm[i] if i < pairs else -dm[i - pairs]) / n
    return loss, seq, m, slope


def lora(x, w, a, b, ids, scale, dy=None):
    """y = x W^T + s (x A^T) B^T of rows [M, K] with row ids, and for dy (dx, dW, dA, dB)."""
    y = x @ w.T
    for m, i in enumerate(ids):
        if 0 <= i < len(a):
            y[m] += scale[i] * (b[i] @ (a[i] @ x[m]))
    if dy is None:
        return y
    dx, da, db = dy @ w, np.zeros_like(a), np.zeros_like(b)
    for m, i in enumerate(ids):
        if 0 <= i < len(a):
            t = scale[i] * (dy[m] @ b[i])
            dx[m] += t @ a[i]
            da[i] += np.outer(t, x[m])
            db[i] += scale[i] * np.outer(dy[m], a[i] @ x[m])
    return y, dx, dy.T @ x, da, db
