"""Plain 64-bit forms of the class-logit operators for the tests (numpy, one row at a time)."""
import math
from fractions import Fraction

import numpy as np


def order_of(row):
    """Classes by logit, larger first, equal ones by lower index, NaN last."""
    key = np.where(np.isnan(row), -np.inf, row)
    return sorted(range(len(row)), key=lambda i: (np.isnan(row[i]), -key[i], i))


def logsumexp(v):
    v = np.asarray(v, dtype=np.float64)
    if np.isnan(v).any():
        return np.nan
    m = v.max() if v.size else -np.inf
    return m if np.isinf(m) and m < 0 else m + np.log(np.exp(v - m).sum())


def log_softmax(v):
    d = v - v.max()  # subtracted first: rows of the type's lowest value have no room for a logarithm
    return d - np.log(np.exp(d).sum())


def top(row, k, temperature):
    o = order_of(row)
    rest = np.nan if np.isnan(row).any() else logsumexp(row[o[k:]] / temperature)
    return np.array(o[:k]), row[o[:k]], rest


def distill(row, index, value, tail, weight, temperature):
    """(loss, der1, p, q) of one row; tail -inf for none."""
    V, T = len(row), temperature
    zero = np.zeros(V)
    if weight == 0:
        return 0.0, zero, zero, zero
    entry = {}
    for i, z in zip(index, value):
        if 0 <= i < V and int(i) not in entry:
            entry[int(i)] = z
    S = sorted(entry)
    z = np.array([entry[i] for i in S] + [0.0])[:-1] / T
    buckets = np.concatenate([z, [tail]])
    if np.isnan(row).any() or np.isnan(buckets).any() or (row == np.inf).any() or (buckets == np.inf).any():
        if not ((row == -np.inf).all() or (buckets == -np.inf).all()):
            return np.nan, np.full(V, np.nan), zero, zero
    if (row == -np.inf).all() or (buckets == -np.inf).all():
        return 0.0, zero, zero, zero
    log_p = log_softmax(row / T)
    p = np.exp(log_p)
    log_q = log_softmax(buckets)
    q = np.exp(log_q)
    rest = np.ones(V, dtype=bool)
    rest[S] = False
    loss = sum(q[j] * (log_q[j] - log_p[i]) for j, i in enumerate(S) if q[j] > 0)
    target = np.zeros(V)
    target[S] = q[:-1]
    if q[-1] > 0:
        log_rest = logsumexp(log_p[rest]) if rest.any() else -np.inf
        loss += q[-1] * (log_q[-1] - log_rest)
        if log_rest > -np.inf:
            # from the logits: log_p of a class 20000 below the others is rounded to 2e-12
            target[rest] = q[-1] * np.exp(log_softmax(row[rest] / T))
    return weight * T * T * loss, weight * T * (target - p), p, target


def sample(row, u, temperature, top_k, top_p, min_p):
    """The drawn class.  Sums are exact (integers of 2^-120), as is u times the mass; p times the
    mass is rounded to a double."""
    if np.isnan(row).any() or (row == -np.inf).all():
        return -1
    o = order_of(row)
    if not temperature > 0:
        return o[0]
    m = row[o[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        e = np.where(row == m, 1.0, np.exp((row - m) / temperature))
    w = [int(math.ldexp(v, 120)) for v in e]
    kept = o[:top_k] if 0 < top_k < len(row) else o
    if top_p < 1:
        part, before, n = top_p * float(sum(w[i] for i in kept)), 0, 0
        for i in kept:
            if n and not before < part:
                break
            before += w[i]
            n += 1
        kept = kept[:n]
    if min_p > 0:
        kept = [i for i in kept if e[i] >= min(min_p, 1.0)]
    kept = sorted(i for i in kept if w[i])
    target = Fraction(float(u)) * sum(w[i] for i in kept)
    upto = 0
    for i in kept:
        upto += w[i]
        if upto > target:
            return i
    return kept[-1]
