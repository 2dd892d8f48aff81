"""Oracle: decode attention over a KV cache, and causal self-attention.

Test infrastructure only (see ``oracle/__init__.py``).

``causal_attention_f64``: ``src/model/chassis.py:465`` without a cache,
F.scaled_dot_product_attention(q, k, v, is_causal=True): query t attends to
keys 0..t with scale 1/sqrt(head_dim).

``src/model/chassis.py:441-478`` with a cache (``:262-330``) at T == 1:
F.scaled_dot_product_attention(q, k, v) without a mask, i.e. for every
(sequence, head) o = softmax(q . k_j * scale over the L cached j) @ V with
scale = 1/sqrt(head_dim).

``window_mask`` / ``window_attention_f64`` / ``window_attention_grads_f64``:
attention over the last ``window`` keys and the first ``sinks`` ones (the
reference has none), its gradients by their formulas and, for tolerances, the
sums of magnitudes behind each result.

``paged_rows`` / ``paged_decode_f64``: the same visibility for one new token
over a cache in pages.
"""
import math

import numpy as np


def decode_attention_f64(q, k, v, scale=None) -> np.ndarray:
    """q [B, H, D], k / v [B, H, L, D] -> o [B, H, D] in float64."""
    q = np.asarray(q, np.float64)
    k = np.asarray(k, np.float64)
    v = np.asarray(v, np.float64)
    D = q.shape[-1]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    s = np.einsum('bhd,bhjd->bhj', q, k) * scale
    s = s - s.max(axis=-1, keepdims=True)
    p = np.exp(s)
    p = p / p.sum(axis=-1, keepdims=True)
    return np.einsum('bhj,bhjd->bhd', p, v)


def causal_attention_f64(q, k, v, scale=None) -> np.ndarray:
    """q, k, v [B, H, T, D] -> o [B, H, T, D] in float64."""
    q = np.asarray(q, np.float64)
    k = np.asarray(k, np.float64)
    v = np.asarray(v, np.float64)
    T, D = q.shape[-2], q.shape[-1]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    s = np.einsum('bhtd,bhjd->bhtj', q, k) * scale
    s = np.where(np.tril(np.ones((T, T), bool)), s, -np.inf)
    s = s - s.max(axis=-1, keepdims=True)
    p = np.exp(s)
    p = p / p.sum(axis=-1, keepdims=True)
    return np.einsum('bhtj,bhjd->bhtd', p, v)


def window_mask(Tq, Tk, window, sinks, length=None) -> np.ndarray:
    """[Tq, Tk]: query i at position p = i + Tk - Tq sees key j iff j <= p and
    (j > p - window or j < sinks); nothing from a position past ``length``."""
    p = np.arange(Tq)[:, None] + Tk - Tq
    j = np.arange(Tk)[None, :]
    ok = (j <= p) & ((j > p - window) | (j < sinks) if window > 0 else True)
    return ok & (p < (Tk if length is None else min(max(int(length), 0), Tk)))


def _weights(q, k, scale, ok):
    s = np.where(ok, (q @ k.T) * scale, -np.inf)
    m = s.max(axis=-1, keepdims=True, initial=-np.inf)
    e = np.exp(s - np.where(np.isfinite(m), m, 0.0))
    l = e.sum(axis=-1, keepdims=True)
    with np.errstate(divide='ignore'):
        lse = np.where(l > 0, np.where(np.isfinite(m), m, 0.0) + np.log(l), -np.inf)[:, 0]
    return e / np.where(l > 0, l, 1.0), lse


def window_attention_f64(q, k, v, window, sinks=0, lengths=None, scale=None, go=None) -> dict:
    """q [B, H, Tq, D], k / v [B, G, Tk, D] -> {"o", "lse"}, with ``go`` also
    {"dq", "dk", "dv"}; float64.  "a_*" are the same sums over magnitudes:
    a_o = P |v|, a_dv = P^T |go|, a_dq = scale |P (go v^T - Delta)| |k|, a_dk
    likewise, and e_dq / e_dk the effect of a Delta off by |go| (|o| + a_o)."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    B, H, Tq, D = q.shape
    G, Tk = k.shape[1], k.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    r = {n: np.zeros((B, H, Tq, D)) for n in ("o", "a_o")}
    r["lse"] = np.zeros((B, H, Tq))
    if go is not None:
        go = np.asarray(go, np.float64)
        for n in ("dq", "a_dq", "e_dq"):
            r[n] = np.zeros((B, H, Tq, D))
        for n in ("dk", "dv", "a_dk", "a_dv", "e_dk"):
            r[n] = np.zeros((B, G, Tk, D))
    for b in range(B):
        ok = window_mask(Tq, Tk, window, sinks, None if lengths is None else lengths[b])
        for h in range(H):
            g = h // (H // G)
            p, r["lse"][b, h] = _weights(q[b, h], k[b, g], scale, ok)
            o = p @ v[b, g]
            r["o"][b, h], r["a_o"][b, h] = o, p @ np.abs(v[b, g])
            if go is None:
                continue
            d = go[b, h]
            ds = scale * p * (d @ v[b, g].T - (d * o).sum(-1, keepdims=True))
            ad = scale * p * (np.abs(d) @ np.abs(v[b, g]).T + (np.abs(d) * r["a_o"][b, h]).sum(-1, keepdims=True))
            ed = scale * p * (np.abs(d) * (np.abs(o) + r["a_o"][b, h])).sum(-1, keepdims=True)
            ak, aq = np.abs(k[b, g]), np.abs(q[b, h])
            r["dq"][b, h], r["a_dq"][b, h], r["e_dq"][b, h] = ds @ k[b, g], ad @ ak, ed @ ak
            r["dk"][b, g] += ds.T @ q[b, h]
            r["a_dk"][b, g] += ad.T @ aq
            r["e_dk"][b, g] += ed.T @ aq
            r["dv"][b, g] += p.T @ d
            r["a_dv"][b, g] += p.T @ np.abs(d)
    return r


def paged_rows(pages, table_row, n, page) -> np.ndarray:
    """The n first rows [n, G, D] of a sequence: pages [P, G, page, D]."""
    pages = np.asarray(pages, np.float64)
    out = np.zeros((n,) + (pages.shape[1], pages.shape[3]))
    for j in range(n):
        out[j] = pages[table_row[j // page], :, j % page]
    return out


def paged_decode_f64(q, k_pages, v_pages, table, lengths, window=0, sinks=0, scale=None):
    """q [B, H, D] at position lengths[b] - 1 -> (o, P |v|) [B, H, D]."""
    q = np.asarray(q, np.float64)
    B, H, D = q.shape
    G, page = k_pages.shape[1], k_pages.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    o, a = np.zeros((B, H, D)), np.zeros((B, H, D))
    for b in range(B):
        n = int(lengths[b])
        if n <= 0:
            continue
        k, v = paged_rows(k_pages, table[b], n, page), paged_rows(v_pages, table[b], n, page)
        ok = window_mask(1, n, window, sinks)
        for h in range(H):
            g = h // (H // G)
            p, _ = _weights(q[b, h][None], k[:, g], scale, ok)
            o[b, h], a[b, h] = (p @ v[:, g])[0], (p @ np.abs(v[:, g]))[0]
    return o, a
