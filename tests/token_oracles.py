"""Plain implementations of the token operators in 64 bits, on the CPU, row by row."""
import math

import numpy as np


def embed(table, ids, scale):
    """table float64 [v, d]; ids [n]."""
    out = np.zeros((len(ids), table.shape[1]))
    for i, t in enumerate(ids):
        if t >= len(table):
            out[i] = np.nan
        elif t >= 0:
            out[i] = scale * table[t]
    return out


def embed_grad(grad, ids, num_rows, scale):
    """The sums, and those of the magnitudes (what rounding errors go by)."""
    out, size, count = np.zeros((num_rows, grad.shape[1])), np.zeros((num_rows, grad.shape[1])), np.zeros(num_rows)
    for i, t in enumerate(ids):
        if 0 <= t < num_rows:
            out[t] += scale * grad[i]
            size[t] += abs(scale) * np.abs(grad[i])
            count[t] += 1
    return out, size, count


def log_softmax(z, temperature):
    """log p of one row; all -inf for a row of nothing but -inf, NaN with NaN or +inf in it."""
    if np.isnan(z).any() or (z == np.inf).any():
        return np.full(z.shape, np.nan)
    if (z == -np.inf).all():
        return np.full(z.shape, -np.inf)
    x = (z - z.max()) / temperature
    return x - math.log(np.exp(x).sum())


def _plogp(logp):
    p = np.exp(logp)
    return p, np.where(p > 0, p * np.where(p > 0, logp, 0.0), 0.0) if not np.isnan(logp).any() else logp


def token_logprobs(z, targets, top, temperature):
    """(log p, entropy, ids, log p of the ids) of rows z float64 [n, v]."""
    n, v = z.shape
    lp, entropy = np.zeros(n), np.zeros(n)
    ids, lps = np.zeros((n, top), np.int64), np.zeros((n, top))
    for i in range(n):
        logp = log_softmax(z[i], temperature)
        entropy[i] = -_plogp(logp)[1].sum()
        if targets[i] >= v:
            lp[i] = np.nan
        elif targets[i] >= 0:
            lp[i] = logp[targets[i]]
        # descending, ties by index, what is no number or ruled out last by index
        rank = np.where(np.isnan(z[i]), -np.inf, z[i])
        order = np.argsort(-rank, kind="stable")[:top]
        ids[i], lps[i] = order, logp[order]
    return lp, entropy, ids, lps


def token_logprobs_grad(z, targets, temperature, g, h):
    """(gradient, the size of its terms)"""
    out, size = np.zeros(z.shape), np.zeros(z.shape)
    for i in range(len(z)):
        gi = g[i] if targets[i] >= 0 else 0.0
        if (gi == 0 and h[i] == 0) or (z[i] == -np.inf).all():
            continue
        logp = log_softmax(z[i], temperature)
        if np.isnan(logp).any() or (targets[i] >= z.shape[1] and gi):
            out[i] = np.nan
            continue
        p, plogp = _plogp(logp)
        entropy = -plogp.sum()
        out[i] = -gi * p - h[i] * (plogp + p * entropy)
        size[i] = abs(gi) * p + abs(h[i]) * (np.abs(plogp) + p * entropy)
        if targets[i] >= 0:
            out[i, targets[i]] += gi
            size[i, targets[i]] += abs(gi)
    return out / temperature, size / temperature


def distill(z, ids, teacher, temperature, weights):
    """(losses, gradient, the size of its terms)"""
    n, v = z.shape
    losses, grad, size = np.zeros(n), np.zeros(z.shape), np.zeros(z.shape)
    for i in range(n):
        slots = [j for j in range(ids.shape[1]) if ids[i, j] >= 0 and teacher[i, j] != -np.inf]
        if not slots:
            continue
        logp = log_softmax(z[i], temperature)
        logq = log_softmax(teacher[i, slots], temperature)
        if max(ids[i, slots]) >= v or np.isnan(logq).any() or np.isnan(logp).any():
            losses[i] = np.nan
            if weights[i] and not (z[i] == -np.inf).all():
                grad[i] = np.nan
            continue
        q = np.exp(logq)
        for j, lq, qj in zip(slots, logq, q):
            if qj > 0:
                losses[i] += qj * (lq - logp[ids[i, j]])
        if weights[i] == 0 or (z[i] == -np.inf).all():
            continue
        grad[i], size[i] = np.exp(logp), np.exp(logp)
        for j, qj in zip(slots, q):
            grad[i, ids[i, j]] -= qj
            size[i, ids[i, j]] += qj
        grad[i] *= weights[i] / temperature
        size[i] *= abs(weights[i]) / temperature
    return losses, grad, size
