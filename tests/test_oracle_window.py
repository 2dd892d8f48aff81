"""The float64 oracle of windowed and paged attention against independent
forms (CPU): torch's autograd in float64, central differences, a mask written
by its definition, and a paged cache against the rows it was filled from."""
import numpy as np
import pytest
import torch

from oracle import attention as oatt

CASES = [(1, 2, 2, 7, 7, 4, 0, 0, None), (2, 4, 2, 9, 13, 5, 4, 2, [13, 6]), (1, 3, 1, 6, 6, 3, 1, 0, [4]),
         (1, 2, 1, 8, 5, 2, 3, 9, None), (2, 2, 2, 1, 11, 3, 2, 1, [11, 0])]


def _inputs(B, H, G, Tq, Tk, D):
    g = torch.Generator().manual_seed(Tq * 31 + Tk)
    mk = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    return mk(B, H, Tq, D), mk(B, G, Tk, D), mk(B, G, Tk, D), mk(B, H, Tq, D)


def test_window_mask_by_definition():
    for Tq, Tk, W, S, n in ((5, 9, 3, 2, 8), (6, 4, 2, 0, None), (3, 3, 0, 0, 2), (4, 4, 9, 1, 4)):
        m = oatt.window_mask(Tq, Tk, W, S, n)
        for i in range(Tq):
            for j in range(Tk):
                p = i + Tk - Tq
                sees = j <= p and (W <= 0 or p - j < W or j < S) and p < (Tk if n is None else n)
                assert m[i, j] == sees, (Tq, Tk, W, S, n, i, j)


@pytest.mark.parametrize("B,H,G,Tq,Tk,D,W,S,lengths", CASES)
def test_window_attention_against_autograd(B, H, G, Tq, Tk, D, W, S, lengths):
    q, k, v, go = _inputs(B, H, G, Tq, Tk, D)
    r = oatt.window_attention_f64(q, k, v, W, S, lengths, go=go)
    for t in (q, k, v):
        t.requires_grad_(True)
    masks = np.stack([oatt.window_mask(Tq, Tk, W, S, None if lengths is None else lengths[b]) for b in range(B)])
    ok = torch.from_numpy(masks)[:, None]
    s = q @ k.repeat_interleave(H // G, 1).transpose(2, 3) / D ** 0.5
    p = torch.softmax(s.masked_fill(~ok, -1e9), -1) * ok
    o = p @ v.repeat_interleave(H // G, 1)
    grads = torch.autograd.grad(o, (q, k, v), go)
    for n, t in zip(("o", "dq", "dk", "dv"), (o,) + grads):
        assert np.allclose(r[n], t.detach().numpy(), rtol=0, atol=1e-12), n
    live = masks.any(-1)[:, None].repeat(H, 1)
    want = torch.logsumexp(s.masked_fill(~ok, -float("inf")), -1).detach().numpy()
    assert np.allclose(r["lse"][live], want[live], atol=1e-12) and np.all(r["lse"][~live] == -np.inf)
    assert np.all(r["o"][~live] == 0)


def test_window_attention_gradients_against_differences():
    q, k, v, go = (t.numpy() for t in _inputs(1, 2, 1, 6, 8, 3))
    r = oatt.window_attention_f64(q, k, v, 3, 1, [7], go=go)
    f = lambda *a: (oatt.window_attention_f64(*a, 3, 1, [7])["o"] * go).sum()  # noqa: E731
    h = 1e-5
    for n, i in (("dq", 0), ("dk", 1), ("dv", 2)):
        x = [q, k, v]
        for at in np.ndindex(x[i].shape):
            up, dn = x[i].copy(), x[i].copy()
            up[at] += h
            dn[at] -= h
            d = (f(*x[:i], up, *x[i + 1:]) - f(*x[:i], dn, *x[i + 1:])) / (2 * h)
            assert abs(d - r[n][at]) < 1e-7, (n, at)


def test_paged_decode_is_window_attention_of_the_last_row():
    rng = np.random.default_rng(0)
    B, H, G, D, page, n = 3, 4, 2, 5, 4, [9, 0, 4]
    table = np.full((B, 3), -1)
    order = rng.permutation(7)
    table[0, :3], table[2, :1] = order[:3], order[3:4]
    kp, vp = rng.standard_normal((2, 7, G, page, D))
    q = rng.standard_normal((B, H, D))
    for W, S in ((0, 0), (3, 1), (20, 2)):
        o, _ = oatt.paged_decode_f64(q, kp, vp, table, n, W, S)
        assert np.all(o[1] == 0)
        for b in (0, 2):
            k = np.stack([kp[table[b, j // page], :, j % page] for j in range(n[b])], 1)[None]
            v = np.stack([vp[table[b, j // page], :, j % page] for j in range(n[b])], 1)[None]
            want = oatt.window_attention_f64(q[b][None, :, None], k, v, W, S)["o"][0, :, 0]
            assert np.allclose(o[b], want, atol=1e-14)


def test_visible_pairs_by_the_mask():
    from src.model.kernels import visible_pairs
    for Tk in (0, 1, 2, 9, 16):
        for Tq in (0, 1, 5, 9, 16, 20):
            for W in (-1, 0, 1, 3, 9, 15, 16, 30):
                for S in (-2, 0, 1, 4, 9, 20):
                    want = int(oatt.window_mask(Tq, Tk, W, max(S, 0)).sum())
                    assert visible_pairs(Tq, Tk, W, S) == want, (Tq, Tk, W, S)
