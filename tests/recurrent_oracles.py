"""Plain implementations in 64 bits, on the CPU, of the recurrence, the clipping of gradients and the verification of drafts."""
import math

import numpy as np

STEP = 2.0 ** -24       # half a step of 32 bits


def sequences_of(rows, length, lengths=None, offsets=None):
    """[(row, first token, one behind the last)] of each sequence."""
    if offsets is not None:
        cut = [min(max(int(o), 0), length) for o in offsets]
        return [(0, a, max(a, b)) for a, b in zip(cut[:-1], cut[1:])]
    return [(b, 0, length if lengths is None else min(max(int(lengths[b]), 0), length)) for b in range(rows)]


def gated_scan(x, gates, state, sequences, decay):
    """(h, last, what stands before each token, error of h, error of last): x, gates [rows, length, dim] float64.

    The errors are how far 32 bits may be off, in units of STEP.  A token adds to what it takes over (times a) up to: 6 for
    the gate (an exponential, a reciprocal and their argument's rounding, on the smaller of a and 1 - a), 3 for the difference,
    the product and the sum, 3 for its share of the maps by which groups of 4 to 8 tokens and tiles are joined (products of that many
    factors of 2 roundings each): 12 of the sum of the magnitudes; 16 are allowed."""
    a = gates if decay else 1.0 / (1.0 + np.exp(-gates))
    b = x if decay else x / (1.0 + np.exp(gates))
    h, before, err = (np.zeros_like(x) for _ in range(3))
    last, last_err = state.copy(), np.zeros_like(state)
    for i, (row, lo, hi) in enumerate(sequences):
        now, size, off = state[i].copy(), np.abs(state[i]), np.zeros_like(state[i])
        for t in range(lo, hi):
            before[row, t] = now
            now = a[row, t] * now + b[row, t]
            size = np.abs(a[row, t]) * size + np.abs(b[row, t])
            off = np.abs(a[row, t]) * off + 16.0 * size
            h[row, t], err[row, t] = now, off
        last[i], last_err[i] = now, off
    return h, last, before, err, last_err


def gated_scan_grad(x, gates, state, sequences, decay, dh, dlast):
    """(dx, dgates, dstate) and their errors, in units of STEP, by the same count."""
    a = gates if decay else 1.0 / (1.0 + np.exp(-gates))
    keep = np.ones_like(a) if decay else 1.0 / (1.0 + np.exp(gates))
    _, _, before, err, _ = gated_scan(x, gates, state, sequences, decay)
    dx, dg, ex, eg = (np.zeros_like(x) for _ in range(4))
    dstate, es = dlast.copy(), np.zeros_like(dlast)
    for i, (row, lo, hi) in enumerate(sequences):
        m, size, off = dlast[i].copy(), np.abs(dlast[i]), np.zeros_like(dlast[i])
        for t in range(hi - 1, lo - 1, -1):
            l, size = dh[row, t] + m, np.abs(dh[row, t]) + size
            off = off + 16.0 * size
            A, K, p, xt = a[row, t], keep[row, t], before[row, t], x[row, t]
            p_err = err[row, t - 1] if t > lo else 0.0
            dx[row, t], ex[row, t] = K * l, np.abs(K) * (off + 8.0 * np.abs(l))
            if decay:
                dg[row, t], eg[row, t] = l * p, off * np.abs(p) + np.abs(l) * (p_err + 4.0 * np.abs(p))
            else:
                dg[row, t] = A * K * l * (p - xt)
                eg[row, t] = A * K * ((off + 16.0 * np.abs(l)) * (np.abs(p) + np.abs(xt)) + np.abs(l) * p_err)
            m, size, off = A * l, np.abs(A) * size, np.abs(A) * off
        if hi > lo:
            dstate[i], es[i] = m, off + 8.0 * size
    return dx, dg, dstate, ex, eg, es


def norm(grads, scale):
    return abs(scale) * math.sqrt(math.fsum(float((np.asarray(g, np.float64) ** 2).sum()) for g in grads))


def clip(grads, max_norm, scale):
    with np.errstate(over="ignore"):
        n = norm(grads, scale)
        n = n if np.float32(n) < np.inf else math.inf          # as it is returned
    factor = scale * (max_norm / n if max_norm < n < math.inf else 1.0)
    return n, [np.asarray(g, np.float64) * factor for g in grads]


def softmax(z, temperature=1.0):
    """None where there are no probabilities."""
    if not len(z) or np.isnan(z).any() or (z == np.inf).any() or (z == -np.inf).all():
        return None
    e = np.exp((z - z.max()) / temperature)
    return e / e.sum()


def verify(z, drafts, uniforms, ids, teacher, temperature):
    """(tokens, accepted, logprobs) of logits [n, k + 1, v]; and how near a decision came to a border."""
    n, rows, v = z.shape
    k = rows - 1
    tokens, accepted, logps, near = np.full((n, rows), -1), np.zeros(n, int), np.zeros((n, rows)), 1.0
    for b in range(n):
        for i in range(rows):
            p = softmax(z[b, i], temperature)
            t = drafts[b, i] if i < k else -1
            w = p
            if t >= 0:
                q = np.zeros(v)
                its = 1.0
                if ids is not None:
                    filled = [j for j in range(ids.shape[2]) if ids[b, i, j] >= 0 and teacher[b, i, j] != -np.inf]
                    share = softmax(teacher[b, i, filled]) if filled else np.zeros(0)
                    if share is None:
                        w, its = None, 0.0
                    else:
                        its = sum(s for s, j in zip(share, filled) if ids[b, i, j] == t)
                        for s, j in zip(share, filled):
                            if ids[b, i, j] < v:
                                q[ids[b, i, j]] += s
                elif t < v:
                    q[t] = 1.0
                u = uniforms[b, i]
                pt = p[t] if p is not None and t < v else 0.0
                if w is not None and pt > 0:
                    near = min(near, abs(u * its - pt) / pt)
                    if u * its < pt:
                        tokens[b, i], logps[b, i] = t, math.log(pt)
                        accepted[b] += 1
                        continue
                if w is not None:
                    w = np.maximum(p - q, 0.0)
                    w = p if w.sum() == 0 else w
            u = uniforms[b, k]
            if w is None or np.isnan(u):
                logps[b, i] = np.nan
                break
            sums = np.cumsum(w)
            target = min(max(u, 0.0), 1.0) * sums[-1]
            above = np.flatnonzero((sums > target) & (w > 0))
            t = above[0] if len(above) else np.flatnonzero(w > 0)[-1]
            if 0 < u < 1:
                near = min(near, np.abs(sums[w > 0] - target).min() / sums[-1])
            tokens[b, i], logps[b, i] = t, math.log(p[t])
            break
    return tokens, accepted, logps, near
