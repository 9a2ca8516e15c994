"""Sampling by row (gh_sample) by its definition, in 64 bits, on the CPU."""
import math

import numpy as np


def kept_weights(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """w of every token of a row, zero for those that are left out; None for a row with nothing to pick.  x and the settings in 64 bits."""
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    order = np.argsort(-x, kind="stable")
    top = x[order[0]]
    if not top > -np.inf:
        return None
    out = np.zeros(len(x))
    if not temperature > 0:
        out[order[0]] = 1.0
        return out
    if 0 < top_k < len(x):
        order = order[:top_k]
    with np.errstate(invalid="ignore", over="ignore", under="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / temperature))
    w = np.where(np.isnan(w) | (x[order] == -np.inf) | (w < 2.0 ** -44), 0.0, w)
    if top_p < 1:
        reached = np.cumsum(w)
        before = np.concatenate(([0.0], reached[:-1]))
        w = np.where((before < top_p * math.fsum(w)) | (np.arange(len(w)) == 0), w, 0.0)
    if min_p > 0:
        w = np.where(w >= min(min_p, 1.0), w, 0.0)
    out[order] = w
    return out


def pick(x, u, **settings):
    """(token, probability)."""
    w = kept_weights(x, **settings)
    if w is None:
        return -1, 0.0
    kept = np.flatnonzero(w > 0)
    total = math.fsum(w)
    target = u * total if u > 0 else 0.0
    at = kept[min(int(np.searchsorted(np.cumsum(w[kept]), target)), len(kept) - 1)]
    return int(at), w[at] / total
