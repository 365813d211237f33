"""The row operations over the vocabulary in 64 bits, one row (or sequence) at a time, written from their formulas (test infrastructure only)."""
import numpy as np


def log_softmax(z, temperature):
    """s of one row: -inf where there is nothing, NaN everywhere in a row with a NaN or +inf."""
    z = np.asarray(z, np.float64)
    m = z.max()
    if np.isnan(m) or m == np.inf:
        return np.full_like(z, np.nan)
    if m == -np.inf:
        return np.full_like(z, -np.inf)
    x = (z - m) / temperature
    return x - np.log(np.exp(x).sum())


def lse(z, temperature):
    z = np.asarray(z, np.float64)
    m = z.max()
    if np.isnan(m) or m == np.inf:
        return np.nan
    return -np.inf if m == -np.inf else m / temperature + np.log(np.exp((z - m) / temperature).sum())


def top(z, k, temperature):
    """(index, s, lse): NaN first, then the values downwards, the lowest index first among equals."""
    z = np.asarray(z, np.float64) + 0.0
    order = sorted(range(z.size), key=lambda i: (not np.isnan(z[i]), 0.0 if np.isnan(z[i]) else -z[i], i))[:k] if np.isnan(z).any() else \
        np.argsort(-z, kind="stable")[:k]
    index = np.asarray(order, np.int32)
    return index, log_softmax(z, temperature)[index], lse(z, temperature)


def distill(z, index, t, temperature, mode, w=1.0):
    """(loss, gradient without the factor w / T, parts the tolerances need) of one row."""
    z, t = np.asarray(z, np.float64), np.asarray(t, np.float64)
    index = np.asarray(index)
    v, t = index[index >= 0], t[index >= 0]
    n = z.size
    q_at = np.exp(t)
    mass = q_at.sum()
    if w == 0 or (mode == "renorm" and mass == 0):
        return 0.0, np.zeros(n), None
    if mode == "renorm":
        q_at, t = q_at / mass, t - np.log(mass)
    s = log_softmax(z, temperature)
    p = np.exp(s)
    q = np.zeros(n)
    np.add.at(q, v, q_at)
    with np.errstate(divide="ignore", invalid="ignore"):
        loss = float(sum(qi * (ti - si) for qi, ti, si in zip(q_at, t, s[v]) if not qi == 0))
        if np.isnan(s).any():
            return np.nan, np.full(n, np.nan), None
        grad = p - q
        if mode == "tail":
            listed = np.zeros(n, bool)
            listed[v] = True
            r = np.maximum(0.0, 1.0 - mass)  # a NaN stays
            zo = z[~listed]
            mo = zo.max() if zo.size else -np.inf
            if mo > -np.inf:
                e = np.exp((zo - mo) / temperature)
                log_rest = s[~listed][np.argmax(zo)] + np.log(e.sum())
                grad[~listed] = p[~listed] - r * e / e.sum()
            else:
                log_rest = -np.inf
                grad[~listed] = 0.0
            if r > 0:
                loss += r * (np.log(r) - log_rest)
    return w * loss, grad, (p, q)


def verify(p_rows, q_rows, tok, u_accept, u_sample):
    """(accepted, token) of one sequence: p_rows has one row more than there are drafts; q_rows None: certain drafts."""
    def mass(x):
        return np.where((x > 0) & (x < np.inf), x, 0.0)

    p_rows = np.asarray(p_rows, np.float64)
    for i, d in enumerate(tok):
        q = 1.0 if q_rows is None else float(q_rows[i][d])
        if float(u_accept[i]) * q < p_rows[i][d]:
            continue
        if q_rows is None:
            left = mass(p_rows[i])
            left[d] = 0.0
        else:
            left = mass(p_rows[i] - np.asarray(q_rows[i], np.float64))
        if left.sum() == 0:
            left = mass(p_rows[i])
        n = i
        break
    else:
        left, n = mass(p_rows[-1]), len(tok)
    if left.sum() == 0:
        return n, -1
    run = np.cumsum(left)
    over = np.nonzero((run > max(float(u_sample), 0.0) * run[-1]) & (left > 0))[0]
    return n, int(over[0]) if over.size else int(np.nonzero(left)[0][-1])
