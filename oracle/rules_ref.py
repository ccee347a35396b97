"""Token rules and gradient clipping in 64 bits, row by row (numpy): what the kernels' tests compare with."""
import math

import numpy as np

LN2 = math.log(2.0)


def counts(history, n, vocab):
    c = np.zeros(vocab, dtype=np.int64)
    if history is not None:
        for t in history[:max(0, n)]:
            if 0 <= t < vocab:
                c[t] += 1
    return c


def ruled_row(x, c, rho=1.0, freq=0.0, pres=0.0, bias=None, allowed=None):
    """-> (x4, slope) of one row: x float64 [V], c counts [V]."""
    x = np.asarray(x, dtype=np.float64)
    seen = c > 0
    y = x.copy()
    slope = np.ones_like(x)
    with np.errstate(all="ignore"):
        pos = x > 0
        y[seen & pos] = x[seen & pos] / rho
        y[seen & ~pos] = x[seen & ~pos] * rho
        slope[seen & pos] = 1.0 / rho
        slope[seen & ~pos] = rho
        y[seen] = y[seen] - freq * c[seen] - pres
        if bias is not None:
            y = y + np.asarray(bias, dtype=np.float64)
    if allowed is not None:
        y = np.where(allowed, y, -np.inf)
    return y, slope


def log_softmax(y, temperature):
    """-> (log p, top, Z of exp((y - top) / T)); top nan for a NaN or +inf value, -inf when nothing is left."""
    top = -np.inf if len(y) == 0 else (np.nan if np.isnan(y).any() else y.max())
    if not np.isfinite(top) or not (temperature > 0 and math.isfinite(temperature)):
        bad = np.full_like(y, -np.inf if top == -np.inf else np.nan)
        return bad, (top if top == -np.inf else np.nan), 0.0
    with np.errstate(all="ignore"):
        e = np.exp((y - top) / temperature)
    z = math.fsum(e)
    return (y - top) / temperature - math.log(z), top, z


def choose_row(y, temperature, u=None):
    """-> (token, log p)"""
    lp, top, z = log_softmax(y, temperature)
    if not np.isfinite(top):
        return -1, (-np.inf if top == -np.inf else np.nan)
    if u is None:
        t = int(np.argmax(y))           # the first of equal ones
        return t, lp[t]
    if math.isnan(u):
        return -1, np.nan
    with np.errstate(all="ignore"):
        w = np.exp((y - top) / temperature)
    run = np.cumsum(w.astype(np.longdouble))
    hit = np.nonzero(run > np.longdouble(max(u, 0.0)) * run[-1])[0]
    t = int(hit[0]) if len(hit) else int(np.nonzero(w)[0][-1])
    return t, lp[t]


def logprob_row(y, slope, token, temperature, g, allowed=None):
    """-> (log p of the token, d logits, d values) for the gradient g of log p."""
    n = len(y)
    zero = np.zeros(n)
    if not 0 <= token < n:
        return 0.0, zero, zero
    lp, top, _ = log_softmax(y, temperature)
    if top == -np.inf:
        return -np.inf, zero, zero
    with np.errstate(all="ignore"):
        d = -np.exp(lp)
        d[token] += 1.0
        d = d * (g / temperature)
    if allowed is not None:
        d = np.where(allowed, d, 0.0)
    return lp[token], d * slope, d


def clip(grads, max_norm):
    """-> (norm, coef) of a list of arrays."""
    s = math.fsum(float(v) for a in grads for v in [np.sum(np.square(np.asarray(a, dtype=np.float64)))])
    norm = math.sqrt(s) if s == s and s != math.inf else s
    return norm, (min(1.0, max_norm / (norm + 1e-6)) if norm == norm else norm)
