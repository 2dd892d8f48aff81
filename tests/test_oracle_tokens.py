"""The token oracle against torch in float64 and the published numbers of the
generator, and the torch forms of the operators against the oracle (CPU)."""
import math

import numpy as np
import pytest
import torch

from oracle import tokens as otok
from src.model import tokens as M

INF = float("inf")


def odd_rows():
    """Rows of 20 logits with every kind of value, their tokens."""
    z = torch.randn(12, 20, generator=torch.Generator().manual_seed(0)) * 3
    z[1, 10:] = -INF
    z[2] = -INF
    z[3, 4] = float("nan")
    z[4, [2, 9]] = INF
    z[5] = torch.finfo(torch.float32).min
    z[6, ::2] = torch.finfo(torch.float32).min
    z[6, 1] = 3.0e38
    z[7] = 0.25
    z[8] = float("nan")                # not counted
    z[9, 1:] = -INF
    return z, torch.tensor([0, 12, 3, 5, 2, 19, 0, 7, -1, 0, 20, 19])


def test_generator_published_numbers():
    """Counter and key of zeros, of ones and of the digits of pi give the
    words of the known-answer tests published with the generator (of which a
    mask takes the halves in order)."""
    def words(c0, c1, c2, c3, k0, k1):
        low = 0xFFFFFFFF
        c, k = [c0, c1, c2, c3], [k0, k1]
        for _ in range(10):
            p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(q >> 32) ^ c[1] ^ k[0], q & low, (p >> 32) ^ c[3] ^ k[1], p & low]
            k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
        return c
    assert words(0, 0, 0, 0, 0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    f = 0xFFFFFFFF
    assert words(f, f, f, f, f, f) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert words(0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344, 0xA4093822, 0x299F31D0) == \
        [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]
    # element (5, 19) of a mask: block 2, half 1 of word 1
    seed, stream = 0x0123456789ABCDEF, 0xFFFFFFFF
    w = words(2, 5, 0, stream, seed & f, seed >> 32)[1] >> 16
    for drop in (w, w + 1):
        assert otok.kept(6, 20, drop, seed, stream)[5, 19] == (w >= drop)
        assert M.kept(6, 20, drop, torch.tensor([seed]), stream)[5, 19] == (w >= drop)


@pytest.mark.parametrize("rows,C,drop,seed,stream", [(1, 1, 32768, 0, 0), (3, 7, 100, 1, 2), (300, 8, 6554, 2 ** 63 - 1, 9),
                                                     (5, 1001, 65535, 12345678901234567, 2 ** 32 - 1), (4, 9, 65536, 7, 0),
                                                     (4, 64, 1, 7, 3), (2, 16, 30000, -5, 3)])
def test_kept(rows, C, drop, seed, stream):
    want = otok.kept(rows, C, drop, seed % 2 ** 64, stream)
    assert np.array_equal(M.kept(rows, C, drop, torch.tensor([seed]), stream).numpy(), want)


def test_kept_share():
    """A share of 1 - p is kept, in every column alike (five standard
    deviations)."""
    rows, C, drop = 4096, 40, 6554
    k = otok.kept(rows, C, drop, 99, 1)
    p = 1 - drop / 65536
    assert abs(k.mean() - p) < 5 * math.sqrt(p * (1 - p) / (rows * C))
    assert np.abs(k.mean(0) - p).max() < 5 * math.sqrt(p * (1 - p) / rows)
    # neighbours, rows and streams agree as independent ones do
    q = p * p + (1 - p) ** 2
    for a, b in ((k[:, 1:], k[:, :-1]), (k[1:], k[:-1]), (k, otok.kept(rows, C, drop, 99, 2)),
                 (k, otok.kept(rows, C, drop, 100, 1))):
        assert abs((a == b).mean() - q) < 5 * math.sqrt(q * (1 - q) / a.size)


def test_logprobs_oracle_against_torch():
    z, t = odd_rows()
    good = [r for r in range(12) if r not in (2, 3, 4, 8, 10)]
    lp, H, top, index = otok.token_logprobs_f64(z.double().numpy(), t.numpy(), 4)
    logp = torch.log_softmax(z.double(), -1)
    assert np.allclose(lp[good], logp[good, t[good]].numpy(), rtol=1e-13)
    assert np.allclose(H[good], torch.special.entr(logp.exp()).sum(-1)[good].numpy(), rtol=1e-13)
    assert np.allclose(top[good], logp[good].topk(4)[0].numpy(), rtol=1e-13)
    assert index[7].tolist() == [0, 1, 2, 3] and index[9].tolist() == [0, 1, 2, 3] and index[8].tolist() == [-1] * 4
    assert lp[2] == -INF and H[2] == 0 and np.isnan(lp[[3, 4, 10]]).all() and lp[8] == H[8] == 0 and H[9] == 0


def same(got, want, rtol):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    # a float32 holds no distance past 3.4e38 (row 6: -6.4e38 and more): infinity
    want = np.where(np.abs(want) > np.finfo(np.float32).max, np.copysign(np.inf, want), want)
    odd = ~np.isfinite(want)
    assert np.array_equal(got[odd], want[odd], equal_nan=True)
    assert np.all(np.abs(got - want)[~odd] <= rtol * np.maximum(1, np.abs(want[~odd])))


@pytest.mark.parametrize("n", [0, 1, 6, 20])
def test_logprobs_plain(n):
    """The torch form (float32: sums of 20 terms and a logarithm, a few
    roundings each of a relative 2^-24) and its autograd."""
    z, t = odd_rows()
    x = z.clone().requires_grad_(True)
    r = M.token_logprobs_plain(x, t, n)
    want = otok.token_logprobs_f64(z.double().numpy(), t.numpy(), n)
    for got, w in zip(r[:3], want):
        same(got.detach().numpy(), w, 64 * 2.0 ** -24)
    assert np.array_equal(r.top_index.numpy(), want[3])
    g = [torch.randn(v.shape, generator=torch.Generator().manual_seed(i)) for i, v in enumerate(r[:3])]
    # rows whose outputs are numbers: autograd of the others multiplies 0 by infinity
    good = [i for i in range(12) if i not in (2, 3, 4, 8, 10)]
    sub = M.token_logprobs_plain(x[good], t[good], n)
    grad, = torch.autograd.grad([v for v in sub[:3] if v.numel()], x, [v[good] for v in g if v.numel()])
    wg = otok.token_logprobs_grad_f64(z.double().numpy(), t.numpy(), want[3], g[0].numpy(), g[1].numpy(), g[2].numpy())
    if n < 20:     # (with all 20 alternatives some have probability 0 and a gradient of their own)
        same(grad[good].numpy(), wg[good], 256 * 2.0 ** -24)
    same(M._logprobs_grad_plain(z, t, r.top_index, *g).numpy(), wg, 256 * 2.0 ** -24)


def test_logprobs_grad_oracle_against_differences():
    g = torch.Generator().manual_seed(3)
    z = torch.randn(2, 9, generator=g).double().numpy()
    t, n = np.array([4, 0]), 3
    gl, gh, gt = (torch.randn(s, generator=g).double().numpy() for s in ((2,), (2,), (2, 3)))

    def f(z):
        lp, H, top, _ = otok.token_logprobs_f64(z, t, n)
        return (gl * lp).sum() + (gh * H).sum() + (gt * top).sum()
    index = otok.token_logprobs_f64(z, t, n)[3]
    want = otok.token_logprobs_grad_f64(z, t, index, gl, gh, gt)
    h = 1e-6
    for r in range(2):
        for i in range(9):
            e = np.zeros_like(z)
            e[r, i] = h
            assert abs((f(z + e) - f(z - e)) / (2 * h) - want[r, i]) < 1e-8


def test_dropout_and_embedding_plain():
    g = torch.Generator().manual_seed(4)
    x, r, seed = torch.randn(5, 3, 13, generator=g), torch.randn(5, 3, 13, generator=g), torch.tensor([77])
    x[0, 0] = float("nan")
    y = M.counter_dropout_plain(x, 0.25, seed, 3, r)
    keep = torch.from_numpy(otok.kept(15, 13, 16384, 77, 3)).view(5, 3, 13)
    want = torch.where(keep, x * (65536 / 49152), torch.zeros_like(x)) + r
    assert torch.allclose(y, want, rtol=4 * 2.0 ** -24, atol=4 * 2.0 ** -24, equal_nan=True)
    assert M.counter_dropout_plain(x, 1.0, seed).abs().max() == 0
    w = torch.randn(11, 13, generator=g, requires_grad=True)
    t = torch.tensor([[3, 3, 10, 0], [-1, 11, 5, 3]])
    y = M.token_embedding_plain(t, w, 2.5, 5, None, 0.25, seed, 3)
    gy = torch.randn(y.shape, generator=g)
    gw, = torch.autograd.grad(y, w, gy)
    keep = torch.from_numpy(otok.kept(8, 13, 16384, 77, 3))
    f = 2.5 * 65536 / 49152
    want = torch.where(keep.view(2, 4, 13), w.detach()[t.clamp(0, 10)] * f, torch.zeros(2, 4, 13))
    want[(t < 0) | (t > 10)] = float("nan")
    assert torch.allclose(y.detach(), want, rtol=4 * 2.0 ** -24, atol=0, equal_nan=True)
    sums, size = otok.embedding_grad_f64(t.reshape(-1).numpy(), (gy.reshape(8, 13) * keep * f).numpy(), 11, 5)
    assert np.all(np.abs(gw.numpy() - sums) <= 8 * 2.0 ** -24 * size)
