"""The operators around a language model's logits, from their definitions in float64 (numpy)."""
import numpy as np


def score(z, token, k):
    """One row z (float64): (logprob, rank, entropy, top log probabilities, top ids)."""
    order = np.lexsort((np.arange(z.size), -z))      # by value, equal ones by index
    m = z.max()
    p = np.exp(z - m)
    s = p.sum()
    logq = (z - m) - np.log(s)
    with np.errstate(invalid="ignore"):
        entropy = -np.sum(np.where(p > 0, (p / s) * logq, 0.0))
    scored = 0 <= token < z.size
    rank = int(np.sum(z > z[token]) + np.sum(z[:token] == z[token])) if scored else -1
    return (logq[token] if scored else 0.0), rank, entropy, logq[order[:k]], order[:k]


def distill(z, ids, t, temperature, tail, weight=1.0):
    """One row: (weighted loss, its gradient), both float64."""
    V, T = z.size, temperature
    if weight == 0:
        return 0.0, np.zeros(V)
    x = z / T
    m = x.max()
    e = np.exp(x - m)
    logq = x - m - np.log(e.sum())
    q = np.exp(logq)
    there = (ids >= 0) & (ids < V)
    ids, t = ids[there], t[there]
    p_of = np.zeros(V)
    listed = np.zeros(V, bool)
    listed[ids] = True
    loss, grad = 0.0, np.zeros(V)
    if tail:
        logp = t
        p = np.exp(logp)
        rest = max(0.0, 1.0 - p.sum()) if not listed.all() else 0.0
    else:
        if ids.size == 0 or t.max() == -np.inf:
            return 0.0, np.zeros(V)
        t = t / T
        logp = t - t.max() - np.log(np.exp(t - t.max()).sum())
        p = np.exp(logp)
        rest = 0.0
    np.add.at(p_of, ids, p)
    on = p > 0
    loss = np.sum(p[on] * (logp[on] - logq[ids[on]]))
    grad = q - p_of
    if tail and not listed.all():
        top = logq[~listed].max()
        out = np.exp(logq[~listed] - top)            # against its own largest: top + log(sum) has no digits left where top is 1e38
        if rest > 0:
            loss += rest * (np.log(rest) - top - np.log(out.sum()))
        grad[~listed] = q[~listed] - rest * out / out.sum()
    return weight * T * T * loss, weight * T * grad
