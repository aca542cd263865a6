"""Oracle of the operators on rows of logits, in 64 bits (numpy): drawing a token, the largest
logits of a row, the distillation loss and its gradient.  Written from the definitions."""
import numpy as np

LOG2E = 1.4426950408889634


def plain(x):
    x = np.asarray(x, dtype=np.float64).copy()
    x[np.isnan(x)] = -np.inf
    return x


def order(x):
    """Indices by falling logit, equal ones by index."""
    return np.lexsort((np.arange(len(x)), -x))


def draw(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, margin): margin is the least distance of a weight sum or weight from a limit it was
    compared with, as a share of the largest weight sum; a draw with a margin well above the
    rounding errors has the same token in any precision."""
    x = plain(x)
    m = x.max()
    if m == -np.inf:
        return -1, np.inf
    if not temperature > 0:
        return int(np.argmax(x)), np.inf
    with np.errstate(invalid='ignore', over='ignore'):
        y = np.where(x == m, 1.0, np.exp2((x - m) * (LOG2E / temperature)))
    by = order(x)
    w = y[by]
    rank = np.arange(len(x))
    if top_k > 0:
        w = np.where(rank < top_k, w, 0.0)
    total = w.sum()
    margin = np.inf
    before = np.cumsum(w) - w
    keep = np.ones(len(x), dtype=bool)
    if top_p < 1.0:
        keep = (before < float(top_p) * total) | (rank == 0)
        near = np.abs(before - float(top_p) * total)[1:][w[1:] > 0]
        if near.size:
            margin = min(margin, near.min() / total)
    if min_p > 0:
        keep &= (y[by] >= min(min_p, 1.0)) | (rank == 0)
        near = np.abs(y[by][1:] / min(min_p, 1.0) - 1.0)
        if near.size:
            margin = min(margin, near.min())
    kept = np.zeros(len(x))
    kept[by] = np.where(keep, w, 0.0)
    prefix = np.cumsum(kept)
    target = float(u) * prefix[-1]
    token = int(np.searchsorted(prefix, target, side='right'))
    token = min(token, int(np.flatnonzero(kept)[-1]))
    inside = prefix[:-1][(prefix[:-1] > 0) & (prefix[:-1] < prefix[-1])]
    if inside.size:
        margin = min(margin, np.abs(inside - target).min() / prefix[-1])
    return token, margin


def top(x, k):
    x = plain(x)
    by = order(x)[:k]
    values = x[by]
    return values, np.where(values == -np.inf, -1, by)


def distill(s, values, indices, temperature=1.0, weight=1.0):
    """(loss, gradient, p, q over the vocabulary) of one row."""
    s, values, indices = np.asarray(s, np.float64), np.asarray(values, np.float64), np.asarray(indices, np.int64)
    used = (indices >= 0) & (indices < len(s)) & (values > -np.inf)
    zero = np.zeros(len(s))
    if not used.any():
        return 0.0, zero, zero, zero
    v, at = values[used] / temperature, indices[used]
    logq = v - v.max() - np.log(np.exp(v - v.max()).sum())
    z = s / temperature
    with np.errstate(invalid='ignore', divide='ignore'):
        logp = z - z.max() - np.log(np.exp(z - z.max()).sum())
    q = np.exp(logq)
    loss = temperature ** 2 * (q * (logq - logp[at])).sum()
    qv = zero.copy()
    np.add.at(qv, at, q)
    p = np.exp(logp)
    return loss, weight * temperature * (p - qv), p, qv
