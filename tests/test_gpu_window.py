"""Windowed attention and its gradients on the GPU against the float64 oracle
on the same (rounded) inputs, element by element.

Tolerances.  h is half a step of the tensors' type (2^-8 bf16, 2^-24
float32): o is rounded once, and bf16 weights P and their gradients dS once
for the products, so with a_x the sums of magnitudes of result x
    |o - o*|   <= h |o*| + h a_o,          |dv - dv*| <= h |dv*| + h a_dv
    |dq - dq*| <= h |dq*| + h a_dq + h e_dq  (e_dq: Delta from an o and a P
                                              that are rounded), dk likewise.
Everything else is float32: a score c q k is off by D 2^-24 c |q| |k|, which
moves P by as much relatively; sums over n keys or queries are off by
n 2^-24 of their magnitudes, exponentials by a few steps.  rho below adds
these, and 2 rho a_x covers the two places (P, Delta) where it enters.
"""
import numpy as np
import pytest
import torch

from oracle import attention as oatt

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def make(B, H, G, Tq, Tk, D, dtype, seed, layout="bthd"):
    g = torch.Generator().manual_seed(seed)

    def mk(h, t):
        if layout == "bthd":
            return torch.randn(B, t, h, D, generator=g).to(dtype).cuda().transpose(1, 2)
        return torch.randn(B, h, t, D, generator=g).to(dtype).cuda()
    return mk(H, Tq), mk(G, Tk), mk(G, Tk), mk(H, Tq)


def rho(q, k, Tq, Tk, scale):
    D = q.shape[-1]
    qa, ka = q.detach().double().abs().amax(dim=(0, 1, 2)), k.detach().double().abs().amax(dim=(0, 1, 2))
    reach = float((qa * ka).sum()) * scale
    return 2.0 ** -24 * (2 * D * reach + max(Tq, Tk) * (q.shape[1] // k.shape[1]) + 4 * D + 64)


def check(name, got, want, tol):
    got = got.double().cpu().numpy()
    assert got.shape == want.shape and np.isfinite(got).all(), name
    over = np.abs(got - want) / np.maximum(tol, 1e-30)
    print(f"{name}: worst error / bound {over.max(initial=0):.3f}", flush=True)
    assert (np.abs(got - want) <= tol).all(), (name, over.max())


def check_all(q, k, v, go, o, grads, W, S, lengths, scale=None):
    Tq, Tk, D = q.shape[2], k.shape[2], q.shape[3]
    c = D ** -0.5 if scale is None else scale
    h, p = HALF[q.dtype], rho(q, k, Tq, Tk, c)
    ln = None if lengths is None else lengths.cpu().numpy()
    r = oatt.window_attention_f64(*(t.detach().double().cpu().numpy() for t in (q, k, v)), W, S, ln, c,
                                  None if go is None else go.double().cpu().numpy())
    check("o", o.detach(), r["o"], h * np.abs(r["o"]) + (h + 2 * p) * r["a_o"])
    if go is not None:
        for n, t in zip(("dq", "dk", "dv"), grads):
            tol = h * np.abs(r[n]) + (h + 2 * p) * r["a_" + n] + ((h + p) * r["e_" + n] if n != "dv" else 0)
            check(n, t, r[n], tol)
    return r


# sizes on both sides of the tiles (32 queries a wavefront, 128 a workgroup, 64 keys a chunk), shared heads, windows
# inside, at and past a tile, first tokens in and past the first chunk, rows that see nothing, padded sequences
SHAPES = [
    # B, H, G, Tq, Tk, D, W, S, lengths
    (1, 1, 1, 1, 1, 16, 0, 0, None),
    (2, 4, 2, 33, 33, 32, 8, 0, None),
    (1, 2, 1, 130, 130, 64, 64, 4, None),
    (2, 3, 3, 257, 257, 128, 100, 3, [257, 70]),
    (1, 4, 1, 200, 331, 64, 63, 70, None),
    (2, 2, 2, 129, 64, 16, 33, 1, None),          # more queries than keys: the first rows see nothing
    (3, 2, 2, 96, 96, 16, 1, 0, [0, 1, 96]),
    (1, 8, 8, 513, 513, 16, 0, 0, None),
    (1, 2, 2, 64, 300, 128, 300, 2, [299]),
    (1, 2, 1, 400, 400, 32, 17, 130, None),
    (1, 1, 1, 700, 700, 128, 65, 1, None),
    # enough rows that a workgroup takes 128 queries instead of 32
    (3, 32, 8, 300, 333, 16, 70, 5, [333, 100, 1]),
    (2, 33, 11, 520, 520, 32, 130, 0, None),
    (3, 32, 32, 300, 300, 64, 0, 0, [17, 300, 299]),
    (2, 48, 6, 400, 390, 128, 150, 66, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H,G,Tq,Tk,D,W,S,lengths", SHAPES)
def test_window_attention_and_gradients(B, H, G, Tq, Tk, D, W, S, lengths, dtype):
    from src.model.attention import window_attention
    print(f"case {B} {H}/{G} {Tq}/{Tk} {D} W={W} S={S} {lengths} {dtype}", flush=True)
    q, k, v, go = make(B, H, G, Tq, Tk, D, dtype, Tq + 7 * D, "bthd" if W % 2 else "bhtd")
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    with torch.no_grad():
        o0 = window_attention(q, k, v, W, S, ln)
    torch.cuda.synchronize()
    for t in (q, k, v):
        t.requires_grad_(True)
    o = window_attention(q, k, v, W, S, ln)
    grads = torch.autograd.grad(o, (q, k, v), go)
    again = torch.autograd.grad(window_attention(q, k, v, W, S, ln), (q, k, v), go)
    torch.cuda.synchronize()
    assert torch.equal(o0, o.detach()) and all(torch.equal(a, b) for a, b in zip(grads, again))
    check_all(q, k, v, go, o, grads, W, S, ln)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_window_attention_log_sums(dtype):
    from src.model import kernels
    q, k, v, _ = make(2, 4, 2, 90, 150, 64, dtype, 5)
    ln = torch.tensor([150, 100], dtype=torch.int32, device="cuda")
    _, lse = kernels.window_attention(q, k, v, 30, 2, ln, need_lse=True)
    r = oatt.window_attention_f64(q.double().cpu(), k.double().cpu(), v.double().cpu(), 30, 2, [150, 100])["lse"]
    lse = lse.double().cpu().numpy()
    assert (np.isneginf(lse) == np.isneginf(r)).all()
    ok = np.isfinite(r)
    # a relative error of the sum is an absolute one of its logarithm
    assert np.abs(lse[ok] - r[ok]).max() <= 2 * rho(q, k, 90, 150, 64 ** -0.5) + 2.0 ** -22 * np.abs(r[ok]).max()


@pytest.mark.gpu
def test_window_attention_layouts_and_partial_gradients():
    """Rows at strides and offsets that the kernels do not read are copied;
    only the gradients that are asked for come back; an expanded output
    gradient is one tensor's worth of values."""
    from src.model.attention import window_attention
    B, H, G, T, D = 2, 4, 2, 70, 32
    base, k, v, _ = make(B, H, G, T, T, D, torch.bfloat16, 9)
    wide = torch.zeros(B, T, H, D + 3, dtype=torch.bfloat16, device="cuda")
    wide[..., 1:D + 1] = base.transpose(1, 2)
    odd = wide[..., 1:D + 1].transpose(1, 2)
    want = window_attention(base, k, v, 20, 2)
    assert torch.equal(window_attention(odd, k, v, 20, 2), want)
    assert torch.equal(window_attention(base, k, v.contiguous(), 20, 2), want)
    # one head's and one sequence's keys for all (expanded), and rows far apart
    ke, ve = k[:1, :1].expand(B, G, T, D), v[:1, :1].expand(B, G, T, D)
    assert torch.equal(window_attention(base, ke, ve, 20, 2), window_attention(base, ke.contiguous(), ve.contiguous(), 20, 2))
    kr = k[:1, :1].detach().clone().requires_grad_(True)
    (dk,) = torch.autograd.grad(window_attention(base, kr.expand(B, G, T, D), ve, 20, 2).sum(), (kr,))
    kx = kr.detach().expand(B, G, T, D).contiguous().requires_grad_(True)
    (dx,) = torch.autograd.grad(window_attention(base, kx, ve.contiguous(), 20, 2).sum(), (kx,))
    assert torch.equal(dk, dx.sum((0, 1), keepdim=True))
    far = torch.zeros(T, (1 << 22) + 8, dtype=torch.bfloat16, device="cuda")
    far = far.as_strided((1, 1, T, D), (0, 0, (1 << 22) + 8, 1))
    far.copy_(k[:1, :1])
    assert torch.equal(window_attention(base[:1, :2], far, v[:1, :1], 20, 2),
                       window_attention(base[:1, :2], k[:1, :1], v[:1, :1], 20, 2))
    vr = v.detach().requires_grad_(True)
    o = window_attention(base, k, vr, 20, 2)
    (dv,) = torch.autograd.grad(o.sum(), (vr,))
    check_all(base, k, vr, None, o, (), 20, 2, None)
    r = oatt.window_attention_f64(*(t.detach().double().cpu().numpy() for t in (base, k, vr)), 20, 2,
                                  go=np.ones((B, H, T, D)))
    h, p = 2.0 ** -8, rho(base, k, T, T, D ** -0.5)
    check("dv", dv, r["dv"], h * np.abs(r["dv"]) + (h + 2 * p) * r["a_dv"])


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,D", [(1, 150, 64), (80, 130, 32)])
def test_window_attention_rest_of_the_output(B, T, D):
    """What rounding took from the output: at most half a step of it, nothing
    in rows that see nothing; the backward's row sums come closer with it."""
    from src.model import kernels
    q, k, v, go = make(B, 4, 2, T, T, D, torch.bfloat16, 12)
    ln = torch.full((B,), T - 7, dtype=torch.int32, device="cuda")
    o, lse, rest = kernels.window_attention(q, k, v, 50, 3, ln, need_rest=True)
    assert torch.equal(o, kernels.window_attention(q, k, v, 50, 3, ln)) and rest.shape == o.shape
    assert (rest.float().abs() <= 2.0 ** -8 * o.float().abs()).all() and rest.any() and not rest[:, :, T - 7:].any()
    r = oatt.window_attention_f64(*(t.detach().double().cpu().numpy() for t in (q[:2], k[:2], v[:2])), 50, 3,
                                  ln[:2].cpu().numpy(), go=go[:2].double().cpu().numpy())
    err = []
    for x in (rest, None):
        dq, dk, dv = kernels.window_attention_bwd(q, k, v, o, lse, go, 50, 3, ln, rest=x)
        err.append([float(np.linalg.norm(a[:2].double().cpu().numpy() - r[n]) / np.linalg.norm(r[n]))
                    for a, n in ((dq, "dq"), (dk, "dk"), (dv, "dv"))])
    print(err, flush=True)
    assert err[0][0] < err[1][0] and err[0][1] < err[1][1] and err[0][2] == err[1][2]
    o32, lse, rest = kernels.window_attention(q.float(), k.float(), v.float(), 50, 3, need_rest=True)
    assert rest is None and lse is not None
    with pytest.raises(AssertionError, match="rest"):
        kernels.window_attention_bwd(q, k, v, o, lse, go, 50, 3, ln, rest=o[:, :, 1:])


@pytest.mark.gpu
def test_window_attention_padding_may_hold_anything():
    """Positions past a sequence's length hold no values: NaN and infinities
    there reach neither outputs nor gradients of the others."""
    from src.model.attention import window_attention
    q, k, v, go = make(2, 2, 2, 150, 150, 64, torch.bfloat16, 3)
    ln = torch.tensor([77, 150], dtype=torch.int32, device="cuda")
    clean = [t.clone() for t in (q, k, v)]
    dirty = [t.clone() for t in (q, k, v)]
    for t in dirty:
        t[0, :, 77:] = float("nan")
        t[0, :, 100:] = float("inf")
    god = go.clone()
    god[0, :, 77:] = float("nan")
    outs = []
    for x, g in ((clean, go), (dirty, god)):
        for t in x:
            t.requires_grad_(True)
        o = window_attention(*x, 40, 3, ln)
        outs.append([o.detach()] + list(torch.autograd.grad(o, x, g)))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
        assert not a[0, :, 77:].any()


@pytest.mark.gpu
def test_window_attention_rows_before_the_first_key_may_hold_anything():
    """More queries than keys: the first rows see nothing, and what they and
    their output gradients hold reaches nothing."""
    from src.model.attention import window_attention
    q, k, v, go = make(1, 2, 1, 90, 50, 32, torch.float32, 4)
    outs = []
    for fill in (0.0, float("nan")):
        q[:, :, :40] = go[:, :, :40] = fill
        x = [t.clone().requires_grad_(True) for t in (q, k, v)]
        o = window_attention(*x, 20, 1)
        outs.append([o.detach()] + list(torch.autograd.grad(o, x, go)))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert not outs[0][0][:, :, :40].any() and not outs[0][1][:, :, :40].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B", [1, 80])
def test_window_attention_of_infinite_scores_is_no_number(B, dtype):
    """Rows that see scores of -inf alone have no weights: not a number, in
    few and in many work items; rows that see others are as without."""
    from src.model.attention import window_attention
    q, k, v, _ = make(B, 4, 2, 40, 40, 32, dtype, 8)
    q = q.abs()
    k2 = k.clone()
    k2[:, :, :10] = float("-inf")
    o = window_attention(q, k2, v, 6)
    assert o[:, :, :10].isnan().all()
    want = window_attention(q, k, v, 6)
    assert torch.equal(o[:, :, 15:], want[:, :, 15:])


@pytest.mark.gpu
def test_window_attention_in_a_graph():
    """Forward and backward captured once and replayed on changing inputs,
    with eager work between the replays."""
    from src.model import kernels
    q, k, v, go = make(1, 4, 2, 200, 200, 64, torch.bfloat16, 11, "bhtd")
    args = (48, 2)

    def step():
        o, lse = kernels.window_attention(q, k, v, *args, need_lse=True)
        return (o, lse) + kernels.window_attention_bwd(q, k, v, o, lse, go, *args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        for t in (q, k, v, go):
            t.copy_(torch.randn(t.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)))
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i


def test_window_attention_refusals():
    """Checks made on the host, before the library is called."""
    from src.model import kernels
    q, k = torch.zeros(2, 4, 3, 16), torch.zeros(2, 2, 3, 16)
    with pytest.raises(RuntimeError, match="GPU"):
        kernels.window_attention(q, k, k, 4)


def test_window_entry_points_check_before_they_launch():
    """Sizes that a launch does not hold, strides and workspaces are refused
    by the library itself (no pointer is followed)."""
    import os
    from src.model import _hip
    if not os.path.exists(_hip.LIB_PATH):
        pytest.skip("library not built")
    L = _hip.lib()
    p = 4096

    def fwd(B=1, H=2, G=1, Tq=8, Tk=8, D=64, st=64, q=p, scale=0.1, dtype=1, rest=None):
        return L.walsh_window_attention_fwd(q, 1 << 20, 1 << 16, st, p, p, 1 << 20, 1 << 16, 64, B, H, G, Tq, Tk, D, 4,
                                            1, None, scale, p, 1 << 20, 1 << 16, 64, p, rest, dtype, None)

    def bwd(Tq=8, Tk=8, work=1 << 30, dq=p):
        return L.walsh_window_attention_bwd(p, 1 << 20, 1 << 16, 64, p, p, 1 << 20, 1 << 16, 64, p, 1 << 20, 1 << 16, 64,
                                            p, 1 << 20, 1 << 16, 64, p, None, 1, 2, 1, Tq, Tk, 64, 4, 1, None, 0.1, dq, p, p,
                                            1, p, work, None)
    for kw, rc in ((dict(H=3, G=2), -1), (dict(Tq=(1 << 24) + 1), -1), (dict(D=24), -2), (dict(st=60), -2),
                   (dict(st=1 << 23), -2), (dict(q=p + 8), -2), (dict(rest=p + 8), -2), (dict(scale=0.0), -1), (dict(dtype=5), -2),
                   (dict(B=1 << 14, H=1 << 10, Tq=128), -2), (dict(B=1 << 60, H=1 << 30), -2),
                   (dict(B=4, H=32, Tq=1 << 24, Tk=1 << 24), -2)):
        assert fwd(**kw) == rc, kw
        assert L.walsh_last_error()
    assert fwd(B=0) == fwd(Tq=0) == 0
    assert bwd(Tq=0) == bwd(Tk=0) == bwd(work=16) == -1
    assert bwd(dq=p + 4) == -2


@pytest.mark.gpu
def test_window_attention_refusals_on_the_gpu():
    from src.model import _hip, kernels
    from src.model.attention import window_attention
    z = lambda *s, dt=torch.float32: torch.zeros(*s, device="cuda", dtype=dt)  # noqa: E731
    q, k = z(2, 4, 3, 16), z(2, 2, 3, 16)
    with pytest.raises(AssertionError, match="evenly"):
        kernels.window_attention(q, z(2, 3, 3, 16), z(2, 3, 3, 16), 4)
    with pytest.raises(AssertionError, match="does not fit"):
        kernels.window_attention(q, z(1, 2, 3, 16), z(1, 2, 3, 16), 4)
    with pytest.raises(ValueError, match="head_dim 24"):
        kernels.window_attention(z(1, 1, 2, 24), z(1, 1, 2, 24), z(1, 1, 2, 24), 4)
    with pytest.raises(TypeError, match="one dtype"):
        kernels.window_attention(q, k.bfloat16(), k.bfloat16(), 4)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        kernels.window_attention(q.half(), k.half(), k.half(), 4)
    with pytest.raises(TypeError, match="int32"):
        kernels.window_attention(q, k, k, 4, lengths=torch.ones(2, device="cuda", dtype=torch.int64))
    with pytest.raises(RuntimeError, match="tensors on"):
        kernels.window_attention(q, k, k, 4, lengths=torch.ones(2, dtype=torch.int32))
    for bad in (0.0, -1.0, float("nan"), 1e9):
        with pytest.raises(_hip.WalshHipError, match="scale"):
            kernels.window_attention(q, k, k, 4, scale=bad)
    # nothing to do: no rows, no keys
    assert window_attention(q[:, :, :0], k, k, 4).shape == (2, 4, 0, 16)
    assert not window_attention(q, k[:, :, :0], k[:, :, :0], 4).any()
    # the gradient of a gradient, and batched gradients, are refused
    qr = q.clone().requires_grad_(True)
    o = window_attention(qr, k, k, 4)
    (g,) = torch.autograd.grad(o.sum(), (qr,), create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    o = window_attention(qr, k, k, 4)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(o, (qr,), torch.ones(2, *o.shape, device="cuda"), is_grads_batched=True)


# What a kernel call would hide from those who look at each operation: dual
# numbers, traces, transforms and dispatch modes take the plain operations.

def _small(dtype, seed=21):
    q, k, v, go = make(2, 4, 2, 20, 26, 16, dtype, seed, "bhtd")
    return q, k, v, go, (7, 2, torch.tensor([26, 13], dtype=torch.int32, device="cuda"))


def _jvp_f64(q, k, v, args, t):
    """The oracle's derivative along the tangents t: the sum of its gradients
    against them, an output's unit direction at a time, by differences."""
    x = [a.double().cpu().numpy() for a in (q, k, v)]
    t = [a.double().cpu().numpy() for a in t]
    f = lambda e: oatt.window_attention_f64(*(a + e * b for a, b in zip(x, t)), args[0], args[1],  # noqa: E731
                                            args[2].cpu().numpy())["o"]
    h = 1e-4
    return (8 * (f(h) - f(-h)) - (f(2 * h) - f(-2 * h))) / (12 * h)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("grad", [False, True])
def test_window_attention_in_forward_mode(grad, dtype):
    """A dual number's tangent arrives, whether or not a gradient is asked for
    as well.  float32 sums of 26 keys and 16 elements: a score is off by 2^-24
    times 16 |q| |k| / 4, a few 1e-6 of it, and the tangent's terms by as much
    relatively; bf16 adds one rounding of the result."""
    import torch.autograd.forward_ad as fw
    from src.model.attention import window_attention
    q, k, v, _, args = _small(dtype)
    t = [torch.randn_like(a) for a in (q, k, v)]
    want = _jvp_f64(q, k, v, args, t)
    with fw.dual_level():
        x = [fw.make_dual(a.requires_grad_(grad), b) for a, b in zip((q, k, v), t)]
        o, do = fw.unpack_dual(window_attention(*x, *args))
    assert do is not None and do.dtype == dtype
    got = do.detach().double().cpu().numpy()
    assert (np.abs(got - want) <= HALF[dtype] * np.abs(want) + 2e-4).all() and np.abs(want).max() > 1
    with torch.no_grad():
        plain = window_attention(q, k, v, *args)
    assert (o.detach().float() - plain.float()).abs().max() <= (0.05 if dtype == torch.bfloat16 else 1e-5)


@pytest.mark.gpu
def test_window_attention_traced():
    """A trace computes the operator of the inputs that it is given."""
    from src.model.attention import window_attention
    q, k, v, _, args = _small(torch.float32)
    traced = torch.jit.trace(lambda *x: window_attention(*x, *args), (q, k, v), check_trace=False)
    for seed in (1, 2):
        x = _small(torch.float32, seed)[:3]
        want = window_attention(*x, *args)
        assert (traced(*x) - want).abs().max() <= 1e-5 and want.abs().max() > 0.1


@pytest.mark.gpu
def test_window_attention_under_transforms():
    """torch.func's grad, jvp and vmap, against the kernels' results."""
    from src.model.attention import window_attention
    q, k, v, go, args = _small(torch.float32)
    x = [a.clone().requires_grad_(True) for a in (q, k, v)]
    want = torch.autograd.grad(window_attention(*x, *args), x, go)
    got = torch.func.grad(lambda *x: (window_attention(*x, *args) * go).sum(), argnums=(0, 1, 2))(q, k, v)
    assert all((a - b).abs().max() <= 1e-4 for a, b in zip(got, want))
    _, do = torch.func.jvp(lambda q: window_attention(q, k, v, *args), (q,), (go,))
    assert np.abs(do.double().cpu().numpy() - _jvp_f64(q, k, v, args, [go, 0 * k, 0 * v])).max() <= 2e-4
    many = torch.stack([q, go, q + go])
    got = torch.func.vmap(lambda q: window_attention(q, k, v, *args))(many)
    for a, b in zip(got, many):
        assert (a - window_attention(b, k, v, *args)).abs().max() <= 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("whole", [False, True])
def test_window_attention_under_a_dispatch_mode(whole):
    """A mode that counts operations sees products (over the backward alone,
    or both), and the results are the kernels'."""
    from torch.utils.flop_counter import FlopCounterMode
    from src.model.attention import window_attention
    q, k, v, go, args = _small(torch.float32)
    x = [a.requires_grad_(True) for a in (q, k, v)]
    want = torch.autograd.grad(window_attention(*x, *args), x, go)
    o = None if whole else window_attention(*x, *args)
    with FlopCounterMode(display=False) as count:
        if whole:
            o = window_attention(*x, *args)
            assert count.get_total_flops() > 0
        got = torch.autograd.grad(o, x, go)
    assert count.get_total_flops() > 0
    assert all((a - b).abs().max() <= 1e-4 for a, b in zip(got, want))


@pytest.mark.gpu
def test_windowed_attention_layer_in_forward_mode():
    """A layer's single token over a dense cache, too."""
    import torch.autograd.forward_ad as fw
    from src.model import WalshConfig
    from src.model.chassis import CausalSelfAttention
    layer = CausalSelfAttention(WalshConfig(n_layer=1, n_head=8, n_embd=256, algebra="hadamard", head_mixing=False,
                                            attn_window=8, attn_sinks=1)).cuda().eval()
    g = torch.Generator().manual_seed(3)
    q, k, v, t = (torch.randn(2, 8, n, 32, generator=g).cuda() for n in (1, 30, 30, 1))
    want = _jvp_f64(q, k, v, (8, 1, torch.full((2,), 30)), [t, 0 * k, 0 * v])
    with torch.no_grad(), fw.dual_level():
        do = fw.unpack_dual(layer._windowed(fw.make_dual(q, t), k, v, 0, True)).tangent
    assert np.abs(do.double().cpu().numpy() - want).max() <= 2e-4 and np.abs(want).max() > 0.1


@pytest.mark.gpu
@pytest.mark.parametrize("H,G,T,D,W,S,lengths", [(4, 2, 300, 16, 0, 0, None), (4, 2, 300, 32, 70, 3, [300, 129]),
                                                 (4, 4, 513, 64, 0, 0, [513, 33]), (2, 1, 513, 64, 100, 40, None),
                                                 (4, 2, 300, 128, 0, 0, [300, 1]), (4, 2, 700, 128, 65, 1, [700, 290])])
def test_window_attention_query_gradients_of_keys_with_an_offset(H, G, T, D, W, S, lengths):
    """A vector added to all keys moves all of a row's scores alike and
    changes no gradient of q, whose weights dS sum to nothing: roundings that
    leave a rest of the sum would be multiplied by it.  The keys are multiples
    of 2^-5 within 1, so that 4 plus a key is a bf16 number: both calls have
    the same exact result, and their errors, of roundings of the same sizes,
    differ by less than 2."""
    from src.model.attention import window_attention
    q, k, v, go = make(2, H, G, T, T, D, torch.bfloat16, D + T, "bhtd")
    k = (torch.rand(k.shape, generator=torch.Generator().manual_seed(T)).mul(64).floor().sub(32) / 32).bfloat16().cuda()
    far = (k.float() + 4).bfloat16()
    assert torch.equal(far.float() - 4, k.float())
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want = oatt.window_attention_f64(*(t.double().cpu().numpy() for t in (q, k, v)), W, S, lengths,
                                     go=go.double().cpu().numpy())["dq"]
    err = []
    for keys in (k, far):
        x = q.clone().requires_grad_(True)
        (dq,) = torch.autograd.grad(window_attention(x, keys, v, W, S, ln), (x,), go)
        err.append(np.linalg.norm(dq.double().cpu().numpy() - want) / np.linalg.norm(want))
    print(f"relative error {err[0]:.2e}, with the offset {err[1]:.2e}", flush=True)
    assert err[1] <= 2 * err[0] and err[0] <= 2.0 ** -8


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,G,T,D,W,S", [(2, 4, 2, 300, 16, 64, 2), (2, 4, 2, 300, 32, 0, 0), (2, 4, 4, 300, 64, 0, 0),
                                           (2, 2, 1, 513, 128, 100, 2), (2, 8, 4, 40, 128, 4, 2), (3, 32, 8, 300, 64, 70, 0)])
def test_window_attention_gradients_of_values_with_an_offset(B, H, G, T, D, W, S):
    """A vector added to all values moves every output alike, and with it
    Delta and each go v^T: dS, dQ and dK do not change.  They would by what
    the output's weights, rounded and not normalised as rounded, have too much
    or too little.  Values are multiples of 2^-5 within 1, 4 plus them bf16
    numbers; the roundings left are of the same sizes, so errors differ by less
    than 2."""
    from src.model.attention import window_attention
    q, k, v, go = make(B, H, G, T, T, D, torch.bfloat16, D + T, "bhtd")
    v = (torch.rand(v.shape, generator=torch.Generator().manual_seed(T)).mul(64).floor().sub(32) / 32).bfloat16().cuda()
    far = (v.float() + 4).bfloat16()
    go = (go.float() + 1).bfloat16()
    assert torch.equal(far.float() - 4, v.float())
    r = oatt.window_attention_f64(*(t.double().cpu().numpy() for t in (q, k, v)), W, S, go=go.double().cpu().numpy())
    err = []
    for values in (v, far):
        x = [t.clone().requires_grad_(True) for t in (q, k)]
        grads = torch.autograd.grad(window_attention(*x, values, W, S), x, go)
        err.append([np.linalg.norm(t.double().cpu().numpy() - r[n]) / np.linalg.norm(r[n]) for n, t in zip(("dq", "dk"), grads)])
    print(f"relative errors {err[0]}, with the offset {err[1]}", flush=True)
    assert all(b <= 2 * a and a <= 2.0 ** -7 for a, b in zip(*err))


@pytest.mark.gpu
@pytest.mark.parametrize("H,G,T,D,W", [(4, 4, 300, 16, 64), (4, 4, 142, 32, 17), (4, 2, 513, 128, 100)])
def test_window_attention_query_gradients_of_large_scores_in_float32(H, G, T, D, W):
    """Queries and keys with an offset of twelve times their spread: scores
    near 36 sqrt(D), whose float32 steps move each weight by some 1e-6
    relatively.  That error enters dQ, dK and dV alike, term by term; the keys'
    offset multiplies it in dQ unless a row's dS sum to nothing."""
    from src.model.attention import window_attention
    q, k, v, go = make(2, H, G, T, T, D, torch.float32, D + T, "bhtd")
    x = [t.mul_(0.25).add_(3).requires_grad_(True) for t in (q, k)] + [v.requires_grad_(True)]
    grads = torch.autograd.grad(window_attention(*x, W, 2), x, go)
    r = oatt.window_attention_f64(*(t.detach().double().cpu().numpy() for t in x), W, 2, go=go.double().cpu().numpy())
    err = [np.linalg.norm(t.double().cpu().numpy() - r[n]) / np.linalg.norm(r[n]) for n, t in zip(("dq", "dk", "dv"), grads)]
    print("relative errors", err, flush=True)
    assert err[0] <= 1.6 * max(err[1:])
