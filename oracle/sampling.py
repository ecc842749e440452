"""Sampling in 64 bits, row by row: the definition in include/ornith_sample.h."""
import numpy as np


def order(row):
    """Columns that take part, by value descending, then column ascending."""
    live = np.flatnonzero(row > -np.inf)
    return live[np.argsort(-row[live], kind='stable')]


def masses(row, ids, T):
    with np.errstate(invalid='ignore'):
        d = (row[ids] - row[ids[0]]) / T
    return np.where(row[ids] == row[ids[0]], 1.0, np.exp(d))


def kept(row, T, k=0, p=1.0, q=0.0):
    """(columns kept, in ascending order; their masses)."""
    ids = order(row)
    e = masses(row, ids, T)
    n = len(ids) if k <= 0 else min(k, len(ids))
    n_k = n
    if p < 1:
        run = np.cumsum(e[:n_k])
        n = min(n, int(np.searchsorted(run, p * run[-1])) + 1)
    n = min(n, int((e >= q).sum()))
    at = np.argsort(ids[:n])
    return ids[:n][at], e[:n][at]


def sample(row, T, k=0, p=1.0, q=0.0, u=0.0):
    """(token, logprob) of one row in float64; (-1, nan) for a row with nothing."""
    row = np.asarray(row, np.float64)
    ids = order(row)
    if not len(ids):
        return -1, np.nan
    if T == 0:
        return int(ids[0]), 0.0
    cols, e = kept(row, T, k, p, q)
    run = np.cumsum(e)
    i = min(int(np.searchsorted(run, u * run[-1], side='right')), len(cols) - 1)
    return int(cols[i]), float(np.log(e[i] / run[-1]))


def uniform_for(row, T, k, p, q, column):
    """The middle of the numbers that draw `column`, and the interval's width."""
    cols, e = kept(np.asarray(row, np.float64), T, k, p, q)
    run = np.cumsum(e)
    i = int(np.searchsorted(cols, column))
    assert cols[i] == column
    return (run[i] - e[i] / 2) / run[-1], e[i] / run[-1]


def top_p_for(row, T, k, n):
    """A p whose prefix is n long, in the middle of those that are, and the
    share of the n-th mass (with k, of the first k)."""
    row = np.asarray(row, np.float64)
    e = masses(row, order(row), T)
    e = e[:k] if k > 0 else e
    run = np.cumsum(e)
    return (run[n - 1] - e[n - 1] / 2) / run[-1], e[n - 1] / run[-1]
