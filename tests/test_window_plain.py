"""Windowed attention from torch's operations (what transforms, traces and
forward-mode derivatives take) against the float64 oracle, on the CPU.

Tolerances: h half a step of the tensors' type for the one rounding of each
result; the rest is float32: a score is off by 2^-24 D c |q| |k|, sums over n
terms by n 2^-24 of their magnitudes, which rho adds up and which enters in
two places (the weights and their gradients)."""
import numpy as np
import pytest
import torch

from oracle import attention as oatt

CASES = [  # B, H, G, Tq, Tk, D, W, S, lengths
    (1, 2, 2, 7, 7, 16, 0, 0, None), (2, 4, 2, 9, 13, 16, 4, 2, [13, 6]), (1, 3, 1, 6, 6, 32, 1, 0, [4]),
    (1, 2, 1, 8, 5, 16, 3, 9, None), (2, 2, 2, 1, 11, 16, 2, 1, [11, 0]), (3, 6, 2, 40, 40, 64, 10, 5, [40, 1, 23]),
    (1, 1, 1, 3, 0, 16, 2, 1, None)]
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def inputs(B, H, G, Tq, Tk, D, dtype, lengths):
    g = torch.Generator().manual_seed(Tq * 31 + Tk)
    q, go = (torch.randn(B, H, Tq, D, generator=g).to(dtype) for _ in range(2))
    k, v = (torch.randn(B, G, Tk, D, generator=g).to(dtype) for _ in range(2))
    return q, k, v, go, None if lengths is None else torch.tensor(lengths, dtype=torch.int32)


def f64(*ts):
    return [t.detach().double().numpy() for t in ts]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H,G,Tq,Tk,D,W,S,lengths", CASES)
def test_plain_window_attention_and_gradients(B, H, G, Tq, Tk, D, W, S, lengths, dtype):
    from src.model.attention import window_attention_plain
    q, k, v, go, ln = inputs(B, H, G, Tq, Tk, D, dtype, lengths)
    if Tk == 0:
        assert not window_attention_plain(q, k, v, W, S, ln).any()
        return
    for t in (q, k, v):
        t.requires_grad_(True)
    o = window_attention_plain(q, k, v, W, S, ln)
    grads = torch.autograd.grad(o, (q, k, v), go)
    r = oatt.window_attention_f64(*f64(q, k, v), W, S, lengths, go=f64(go)[0])
    h = HALF[dtype]
    reach = float((q.detach().abs().amax((0, 1, 2)).double() * k.detach().abs().amax((0, 1, 2)).double()).sum()) * D ** -0.5
    rho = 2.0 ** -24 * (2 * D * reach + max(Tq, Tk) * (H // G) + 4 * D + 64)
    assert o.dtype == dtype
    for n, t in zip(("o", "dq", "dk", "dv"), (o,) + grads):
        tol = h * np.abs(r[n]) + 2 * rho * r["a_" + n] + (rho * r["e_" + n] if n in ("dq", "dk") else 0)
        assert (np.abs(f64(t)[0] - r[n]) <= tol).all(), n


def test_plain_window_attention_of_padding():
    """NaN and infinities in rows without a key and past the lengths reach
    neither the outputs nor any gradient."""
    from src.model.attention import window_attention_plain
    outs = []
    for fill in (0.0, float("nan"), float("inf")):
        q, k, v, go, ln = inputs(2, 4, 2, 12, 9, 16, torch.float32, [9, 4])
        q[:, :, :3] = go[:, :, :3] = fill
        for t, at in ((q, 7), (go, 7), (k, 4), (v, 4)):
            t[1, :, at:] = fill
        x = [t.requires_grad_(True) for t in (q, k, v)]
        o = window_attention_plain(*x, 4, 1, ln)
        outs.append([o.detach()] + list(torch.autograd.grad(o, x, go)))
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))
    assert not outs[0][0][:, :, :3].any() and not outs[0][0][1, :, 7:].any()


def test_plain_window_attention_both_modes_agree():
    """go . J t forward equals (J^T go) . t backward; a trace follows its
    inputs; autocast changes nothing."""
    import torch.autograd.forward_ad as fw
    from src.model.attention import window_attention_plain
    q, k, v, go, ln = inputs(2, 4, 2, 9, 13, 16, torch.float32, [13, 6])
    f = lambda *x: window_attention_plain(*x, 4, 2, ln)  # noqa: E731
    t = [torch.randn(a.shape, generator=torch.Generator().manual_seed(9)) for a in (q, k, v)]
    with fw.dual_level():
        do = fw.unpack_dual(f(*(fw.make_dual(a, b) for a, b in zip((q, k, v), t)))).tangent
    x = [a.clone().requires_grad_(True) for a in (q, k, v)]
    grads = torch.autograd.grad(f(*x), x, go)
    forward, backward = float((do.double() * go).sum()), sum(float((a.double() * b).sum()) for a, b in zip(grads, t))
    size = sum(float((a.double() * b).abs().sum()) for a, b in zip(grads, t))
    assert abs(forward - backward) <= 2.0 ** -24 * 1000 * size
    traced = torch.jit.trace(f, (q, k, v), check_trace=False)
    assert torch.allclose(traced(go, v, k), f(go, v, k), rtol=0, atol=1e-6)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        assert torch.equal(f(q, k, v), f(*(a.clone() for a in (q, k, v))))
        cast = f(q, k, v)
    assert torch.equal(cast, f(q, k, v))


def test_window_attention_under_a_mode_refuses_the_cpu_too():
    import torch.autograd.forward_ad as fw
    from src.model.attention import window_attention
    q = torch.zeros(1, 1, 3, 16)
    with fw.dual_level():
        with pytest.raises(RuntimeError, match="GPU"):
            window_attention(fw.make_dual(q, q), q, q, 2)
