"""Token probabilities, embedding gradients and dropout's mask, restated with
numpy in float64 and whole numbers (no counterpart in the reference)."""
import numpy as np


def _rows(logits):
    """(log probabilities, probabilities) [N, V]; a row of -inf alone: -inf and 0."""
    z = np.asarray(logits, np.float64)
    with np.errstate(all="ignore"):
        nothing = np.all(z == -np.inf, axis=1, keepdims=True)
        m = np.where(nothing, 0.0, z.max(1, keepdims=True))
        d = z - m
        logp = np.where(nothing, -np.inf, d - np.log(np.exp(d).sum(1, keepdims=True)))
        return logp, np.exp(logp)


def token_logprobs_f64(logits, tokens, n=0):
    """(logprob [N], entropy [N], top [N, n], index [N, n])."""
    logp, p = _rows(logits)
    N, V = logp.shape
    with np.errstate(all="ignore"):
        H = -np.where(p == 0, 0.0, p * logp).sum(1)
    lp = np.array([0.0 if t < 0 else np.nan if t >= V else logp[r, t] for r, t in enumerate(tokens)])
    z = np.where(np.isnan(logits), -np.inf, np.asarray(logits, np.float64))
    index = np.stack([np.lexsort((np.arange(V), -z[r]))[:n] for r in range(N)]).reshape(N, n)
    top = np.take_along_axis(logp, index, 1)
    dead = np.asarray(tokens) < 0
    H[dead], top[dead], index[dead] = 0.0, -np.inf, -1
    return lp, H, top, index


def token_logprobs_grad_f64(logits, tokens, index, g_lp=None, g_H=None, g_top=None):
    logp, p = _rows(logits)
    N, V = logp.shape
    out = np.zeros((N, V))
    for r, t in enumerate(tokens):
        if t < 0 or np.all(logp[r] == -np.inf):
            continue
        if t >= V:
            out[r] = np.nan
            continue
        g = np.zeros(V)                      # of the row's log probabilities
        if g_lp is not None:
            g[t] += g_lp[r]
        if g_top is not None:
            for j, i in enumerate(index[r]):
                g[i] += g_top[r, j]
        if g_H is not None:
            with np.errstate(all="ignore"):
                g -= g_H[r] * np.where(p[r] == 0, 0.0, p[r] * (1 + logp[r]))
        out[r] = g - p[r] * g.sum()
    return out


def kept(rows, C, drop, seed, stream, first=0):
    """What dropout keeps, element by element of [rows, C] (the rows from
    ``first`` on): the ten-round
    generator of Salmon et al. (SC 2011) on key ``seed``, counter (column / 8,
    row, 0, stream), 16 bits a column."""
    low = 0xFFFFFFFF
    u = np.uint64
    c = [np.broadcast_to(np.arange(-(-C // 8), dtype=u)[None], (rows, -(-C // 8))),
         np.broadcast_to(np.arange(first, first + rows, dtype=u)[:, None], (rows, -(-C // 8)))]
    c += [np.zeros_like(c[0]), np.full_like(c[0], stream)]
    k = [seed & low, (seed >> 32) & low]
    for _ in range(10):
        p, q = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(q >> u(32)) ^ c[1] ^ u(k[0]), q & u(low), (p >> u(32)) ^ c[3] ^ u(k[1]), p & u(low)]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    bits = np.stack([h for w in c for h in (w & u(0xFFFF), w >> u(16))], -1).reshape(rows, -1)
    return bits[:, :C] >= drop


def dropout_f64(x, drop, seed, stream):
    keep = kept(x.shape[0], x.shape[1], drop, seed, stream)
    return np.where(keep, np.asarray(x, np.float64) * (65536.0 / (65536 - drop) if drop < 65536 else 0.0), 0.0)


def embedding_grad_f64(tokens, g, V, padding_idx=None):
    """(sums, sums of the absolute values) [V, C] over the rows of each token."""
    out, size = np.zeros((V, g.shape[1])), np.zeros((V, g.shape[1]))
    for t, row in zip(tokens, np.asarray(g, np.float64)):
        if 0 <= t < V and t != padding_idx:
            out[t] += row
            size[t] += np.abs(row)
    return out, size
