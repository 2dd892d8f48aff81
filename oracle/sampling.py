"""Oracle: the next token of a row of logits from a given uniform number.

Test infrastructure only (see ``oracle/__init__.py``).  The reference samples
with torch.topk and torch.multinomial (``src/model/mhc.py:754-772``); the
filters and the draw are restated here by their definition, on a sorted row in
float64.
"""
import numpy as np


def sample_f64(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, margin) of one row: ``margin`` is the smallest relative distance
    of a border (of the draw, of top-p, of min-p) from the value compared with
    it; a token is certain where weights are known to better than that."""
    z = np.asarray(logits, np.float64).copy()
    z[np.isnan(z)] = -np.inf
    if z.max(initial=-np.inf) == -np.inf:
        return -1, 1.0
    if not temperature > 0:
        return int(np.argmax(z)), 1.0
    if z.max() == np.inf:
        w = (z == np.inf).astype(np.float64)
    else:
        w = np.exp((z - z.max()) / temperature)
    order = np.lexsort((np.arange(len(z)), -z))
    if 0 < top_k < len(z):
        order = order[:top_k]
    margin = 1.0
    if top_p < 1.0:
        before = np.concatenate([[0.0], np.cumsum(w[order])])[:-1]
        need = top_p * w[order].sum()
        keep = before < need
        keep[0] = True
        if len(order) > 1:
            margin = min(margin, float(np.abs(before[1:] - need).min() / w.sum()))
        order = order[keep]
    if min_p > 0:
        margin = min(margin, float(np.abs(w[order] - min_p).min() / min_p))
        order = order[w[order] >= min_p]
    if len(order) == 0 or w[order].sum() == 0:
        return -1, margin
    idx = np.sort(order)
    c = np.cumsum(w[idx])
    at = min(max(u, 0.0) * c[-1], np.nextafter(c[-1], 0))
    i = int(np.searchsorted(c, at, side="right"))
    edges = np.concatenate([[0.0], c[:-1]])
    near = np.abs(edges[edges > 0] - at)
    if len(near) and u > 0:
        margin = min(margin, float(near.min() / c[-1]))
    return int(idx[i]), margin
