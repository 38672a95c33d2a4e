"""Float64 oracle of the scores of tokens (fn_logprobs): a row at a time, from the definitions."""

import numpy as np


def before(x, i, j):
    """Whether entry i stands before entry j: the larger value, of equal ones (-0 equals +0) the lower index."""
    return x[i] > x[j] or (x[i] == x[j] and i < j)


def row(x, token, top):
    """(logprob, rank, entropy, top_ids [top], top_logprobs [top]) of one row."""
    x = np.asarray(x, np.float64)
    ids, logs = np.full(top, -1, np.int64), np.full(top, -np.inf)
    sick = np.isnan(x).any() or (x == np.inf).any()
    live = np.flatnonzero(x > -np.inf)  # NaN is none of them
    order = live[np.lexsort((live, -x[live]))]
    if sick:
        lse, entropy = np.nan, np.nan
    elif len(live) == 0:
        lse, entropy = np.inf, 0.0
    else:
        m = x[live].max()
        e = np.exp(x[live] - m)
        lse = m + np.log(e.sum())
        p = e / e.sum()
        entropy = -(p[p > 0] * np.log(p[p > 0])).sum()
    n = min(top, len(order))
    ids[:n] = order[:n]
    logs[:n] = x[order[:n]] - lse
    if token < 0:
        return 0.0, -1, entropy, ids, logs
    if token >= len(x):
        return np.nan, -1, entropy, ids, logs
    with np.errstate(invalid="ignore"):
        logprob = x[token] - lse if not sick and len(live) else (np.nan if sick else -np.inf)
        rank = -1 if np.isnan(x[token]) else int(((x > x[token]) | ((x == x[token]) & (np.arange(len(x)) < token))).sum())
    return logprob, rank, entropy, ids, logs


def rows(x, tokens, top):
    got = [row(r, int(t), top) for r, t in zip(x, tokens)]
    return {k: np.array([g[i] for g in got]) for i, k in enumerate(("logprob", "rank", "entropy", "top_ids", "top_logprobs"))}
