"""Routing to experts in float64, a row at a time, and how clear each of its
decisions was."""
import numpy as np


def scores(logits, kind):
    """Scores of one row of logits (float64)."""
    l = np.asarray(logits, np.float64)
    with np.errstate(over='ignore', invalid='ignore', divide='ignore'):
        if kind == 'sigmoid':
            return np.where(np.isnan(l), 0.0, 1 / (1 + np.exp(-np.maximum(l, -700.0))))
        live = l[~np.isnan(l)]
        mx = live.max() if live.size else -np.inf
        e = np.where(l == mx, 1.0, np.exp(l - mx))
        e = np.where(np.isnan(l) | (l == -np.inf), 0.0, e)
        return e / e.sum() if e.sum() else e


def route(logits, top, kind='softmax', bias=None, groups=1, kept=1, group_top=1, renormalize=True, scale=1.0):
    """(weights float64 [top], ids [top], the least distance by which an expert
    or a group was picked before the next, relative to the larger)."""
    l = np.asarray(logits, np.float64)
    E = l.size
    s = scores(l, kind)
    with np.errstate(invalid='ignore'):
        c = l.copy() if bias is None else s + np.asarray(bias, np.float64)
    c[np.isnan(c) | np.isnan(l) | (l == -np.inf)] = -np.inf
    clear = np.inf

    def distance(hi, lo):
        return np.inf if lo == -np.inf or hi == np.inf or hi == lo else (hi - lo) / max(abs(hi), abs(lo))

    if kept < groups:
        size, score = E // groups, np.full(groups, -np.inf)
        for g in range(groups):
            at = np.arange(g * size, (g + 1) * size)
            best = sorted((at[c[at] > -np.inf]).tolist(), key=lambda i: (-c[i], i))[:group_top]
            if best:
                # by one best: its c (a logit where there is no bias); by two: sums of scores
                score[g] = c[best[0]] if group_top == 1 else sum((c if bias is not None else s)[best])
        order = sorted(range(groups), key=lambda g: (-score[g], g))
        clear = min(clear, distance(score[order[kept - 1]], score[order[kept]]))
        for g in order[kept:]:
            c[g * size:(g + 1) * size] = -np.inf
    order = sorted(np.flatnonzero(c > -np.inf).tolist(), key=lambda i: (-c[i], i))
    for i in range(min(top, len(order) - 1)):
        clear = min(clear, distance(c[order[i]], c[order[i + 1]]))
    ids = order[:top]
    if kind == 'softmax' and renormalize and ids:
        li = l[ids]
        m = li.max()
        w = np.array([1.0 if v == m else np.exp(v - m) for v in li])
    else:
        w = s[ids]
    if renormalize and ids:
        w = w / w.sum()
    weights, out = np.zeros(top), np.full(top, -1, np.int32)
    weights[:len(ids)], out[:len(ids)] = w * scale, ids
    return weights, out, clear
