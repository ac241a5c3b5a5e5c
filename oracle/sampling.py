"""Truncated sampling restated in float64 (test infrastructure): entries ordered by (logit descending, index ascending),
top-k, then top-p over what top-k keeps, then min-p, then inversion of the uniform u."""
import numpy as np


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row -> (token, probability among the kept entries, number kept)."""
    l = np.asarray(logits, dtype=np.float64)
    l = np.where(np.isnan(l), -np.inf, l)
    order = np.argsort(-l, kind="stable")
    v = l[order]
    v = v[v > -np.inf]
    if v.size == 0:
        return 0, 0.0, 0
    m = v[0]
    if temperature == 0:
        return int(order[0]), 1.0, 1
    with np.errstate(invalid="ignore"):
        below = np.where(v == m, 0.0, v - m)          # (m may be infinite)
    w = np.exp(below / temperature)
    mass = np.cumsum(w)
    n = v.size if top_k <= 0 else min(top_k, v.size)
    if top_p < 1.0:
        n = min(n, int((mass < top_p * mass[n - 1]).sum()) + 1)
    if min_p > 0.0:
        n = max(1, min(n, int((below >= temperature * np.log(min_p)).sum())))      # w >= min_p, free of exp's rounding
    i = min(int((mass <= u * mass[n - 1]).sum()), n - 1)
    return int(order[i]), float(w[i] / mass[n - 1]), n


def confidence(logits, token, rule, excluded=-1):
    """generate.py:103-123 for a candidate `token` on the row's temperature-1 softmax without the entry `excluded`, float64."""
    l = np.asarray(logits, dtype=np.float64).copy()
    l = np.where(np.isnan(l), -np.inf, l)
    if excluded >= 0:
        l[excluded] = -np.inf
    p = np.exp(l - l.max())
    p /= p.sum()
    if rule == "low_confidence":
        return p[token]
    if rule == "high_confidence":
        return 1.0 - p[token]
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.where(p > 0, p * np.log(p), 0.0).sum()
    return -e if rule == "low_entropy" else e
