"""Log probabilities, entropies and alternatives on the GPU, and their
gradients, against the float64 oracle.

Bounds: a weight exp(l - m) is formed with three roundings of its exponent and
one of the exponential, relatively 2^-24 (3 |log2 w| + 2); a lane adds at most
V / 256 of them one after the other and moves its sums to a new maximum (three
roundings) at most once for every 2,048 tokens and twice at the end; 24 more
additions join lanes and wavefronts.  Weighted by w, |log2 w| averages to at
most log2 V < 18.  So the sum S, and with it log S, is within
    unit(V) = 2^-24 (V / 256 + 3 V / 2048 + 100)
of itself, and what is formed from it within a few units."""
import numpy as np
import pytest
import torch

from oracle import tokens as otok

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
INF, NAN = float("inf"), float("nan")


def unit(V):
    return 2.0 ** -24 * (V / 256 + 3 * V / 2048 + 100)


def rows(N, V, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(N, V, generator=g) * (0.5 + 4 * torch.rand(N, 1, generator=g))).to(dtype)
    t = torch.randint(V, (N,), generator=g)
    best = torch.rand(N, generator=g) < 0.5
    return z, torch.where(best, z.float().argmax(-1), t)


def in_float(want):
    """Float64 numbers as float32 can hold them: no distance past 3.4e38."""
    want = np.asarray(want, np.float64)
    return np.where(np.abs(want) > np.finfo(np.float32).max, np.copysign(np.inf, want), want)


def close(got, want, bound, what):
    got, want = got.double().cpu().numpy(), in_float(want)
    odd = ~np.isfinite(want)
    assert np.array_equal(got[odd], want[odd], equal_nan=True), what
    with np.errstate(invalid="ignore"):
        off = np.abs(got - want) / np.broadcast_to(bound, want.shape)
    assert np.all(off[~odd] <= 1), (what, float(off[~odd].max()))


def check(z, t, n, got, V):
    """``got`` of token_logprobs against the oracle."""
    lp, H, top, index = otok.token_logprobs_f64(z.double().cpu().numpy(), t.cpu().numpy(), n)
    fin = lambda x: np.where(np.isfinite(x), np.abs(x), 0)  # noqa: E731
    close(got[0], lp, unit(V) + 4 * 2.0 ** -24 * fin(lp), "logprob")
    close(got[1], H, unit(V) * 40, "entropy")
    close(got[2], top, unit(V) + 4 * 2.0 ** -24 * fin(top), "top")
    assert np.array_equal(got[3].cpu().numpy(), index)
    return index


def run(z, t, n=0):
    from src.model import kernels
    return kernels.token_logprobs(z.cuda(), t.cuda(), n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V", [(1, 1), (3, 2), (5, 7), (4, 8), (2, 9), (7, 63), (3, 64), (3, 65), (2, 511), (4, 512),
                                 (3, 1021), (2, 2049), (5, 4096), (3, 8191), (3, 8200), (2, 16391), (4, 32003),
                                 (300, 1000), (6, 50257), (2, 131077)])
def test_forward(N, V, dtype):
    z, t = rows(N, V, dtype, V)
    for n in sorted({0, 1, min(V, 5), min(V, 64)}):
        print(f"N={N} V={V} n={n} {dtype}", flush=True)
        check(z, t, n, run(z, t, n), V)


@pytest.mark.parametrize("dtype", DTYPES)
def test_odd_values(dtype):
    """Masked tails, rows of nothing, NaN, infinities, lowest values, equal
    logits, uncounted rows, tokens outside."""
    for V in (40, 3000, 20011):
        z, t = rows(13, V, dtype, V)
        low = torch.finfo(dtype).min
        z[1, V // 3:] = -INF
        t[1] = V - 1
        z[2] = -INF
        z[3, 4] = NAN
        z[4, [2, 9]] = INF
        z[5] = low
        z[6, ::2] = low
        z[6, 1] = 3e38
        z[7] = 0.25
        z[8] = NAN
        t[8] = -1
        z[9, 1:] = -INF
        t[9] = 0
        t[10] = V
        z[11] = NAN
        t[12] = -(2 ** 60)
        for n in (0, 3, 20):
            check(z, t, n, run(z, t, n), V)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1500, 50257])
def test_equal_and_ordered(V, dtype):
    """Thousands of equal logits, and rows whose largest lie side by side, in
    order, or all in one lane's tokens."""
    z = torch.zeros(8, V)
    z[1, ::3] = 1.0
    z[2] = torch.arange(V) / V
    z[3] = -torch.arange(V) / V
    z[4, 700:1400] = torch.arange(700) / 64.0
    z[5, :] = -torch.arange(V).remainder(8192).div(8, rounding_mode="floor").float()     # the first lane has the largest
    z[6] = torch.randn(V, generator=torch.Generator().manual_seed(1)).round()
    z[7, -70:] = 5.0
    z = z.to(dtype)
    t = torch.arange(8) * (V // 9)
    for n in (1, 17, 64):
        check(z, t, n, run(z, t, n), V)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [100, 4099, 50257])
def test_few_tokens_allowed(V, dtype):
    """Rows that a grammar has masked, by -inf and by the type's lowest value:
    fewer tokens left than alternatives are asked for, or all left side by side;
    and values that no usual logit has below them."""
    g = torch.Generator().manual_seed(V)
    low = torch.finfo(dtype).min
    z = torch.full((9, V), -INF)
    z[:, torch.randperm(V, generator=g)[:3]] = torch.tensor([1.0, -2.0, 1.0])
    z[1][z[1] == -INF] = low
    z[2, :90] = torch.randn(90, generator=g)
    z[3, V - 64:] = torch.randn(64, generator=g)
    z[4, 10:14] = torch.tensor([-1e35, -2e35, -1e35, -1e30])
    z[5, 20:80] = low
    z[6] = -INF
    z[6, V // 2] = 0.0
    z[7, ::2] = -1e30
    z[8, 1::3] = NAN
    z = z.to(dtype)
    t = z.float().nan_to_num(-INF).argmax(-1)
    for n in (1, 3, 4, 20, 64):
        check(z, t, n, run(z, t, n), V)


def test_layouts():
    """Rows of a wider matrix, at odd addresses, transposed, expanded, with
    several leading dimensions; tokens and outputs keep theirs."""
    from src.model import kernels
    base, t = rows(6, 1207, torch.bfloat16, 5)
    views = [base.cuda()[:, 3:1003], base.cuda().t().contiguous().t()[:, :1000], base.cuda()[:1, :1000].expand(6, 1000),
             torch.cat([torch.zeros(1, dtype=base.dtype), base[:, :1000].reshape(-1)]).cuda()[1:].view(6, 1000)]
    t = t.clamp(0, 999)
    for v in views:
        check(v, t, 4, kernels.token_logprobs(v, t.cuda(), 4), 1000)
        g = torch.ones(6, device="cuda")
        got = kernels.token_logprobs(v, t.cuda(), 0, need_stats=True)
        d = kernels.token_logprobs_bwd(v, t.cuda(), got[3], got[4], g)
        want = otok.token_logprobs_grad_f64(v.double().cpu().numpy(), t.numpy(), None, np.ones(6))
        close(d, want, 1e-3 * unit(1000) + np.abs(want) * (2.0 ** -8 + 4 * unit(1000)), "gradient")
    v3 = base.view(2, 3, 1207).cuda()
    got = kernels.token_logprobs(v3, t.view(2, 3).cuda(), 2)
    assert got[0].shape == (2, 3) and got[2].shape == (2, 3, 2)
    check(base, t, 2, [x.flatten(0, 1) for x in got], 1207)
    twice = t.cuda().repeat_interleave(2)[::2]
    assert torch.equal(kernels.token_logprobs(base.cuda(), twice, 0)[0], kernels.token_logprobs(base.cuda(), t.cuda(), 0)[0])
    # nothing at all
    for shape in ((0, 7), (3, 0, 7)):
        got = kernels.token_logprobs(torch.zeros(shape, device="cuda"), torch.zeros(shape[:-1], device="cuda").long(), 3)
        assert got[2].shape == shape[:-1] + (3,) and got[0].numel() == 0


def grad_bound(z, t, index, gs, want, dtype, V):
    # (rows that are not counted hold anything and give exact zeros)
    logp, p = otok._rows(torch.where(torch.from_numpy(t >= 0)[:, None], z.double(), 0.0).numpy())
    p[t < 0] = 0
    gl, gh, gt = gs
    G = np.abs(gl) + (np.abs(gt).sum(1) if gt is not None else 0)
    with np.errstate(invalid="ignore"):
        lp = np.where(p > 0, np.abs(logp), 0)
        inner = p * (G[:, None] + np.abs(gh)[:, None] * (lp + 20))
        size = inner * (3 * lp * 2.0 ** -24 + 3 * unit(V))
    special = np.zeros_like(p)
    for r in range(len(p)):
        if 0 <= t[r] < V:
            special[r, t[r]] += abs(gl[r])
        if gt is not None and t[r] >= 0:
            np.add.at(special[r], index[r], np.abs(gt[r]))
    half = torch.finfo(dtype).eps / 2
    with np.errstate(invalid="ignore"):
        return size + 3 * 2.0 ** -24 * (special + inner) + half * np.where(np.isfinite(want), np.abs(want), 0) + 1e-37


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V", [(1, 1), (3, 2), (5, 9), (4, 64), (3, 511), (2, 1021), (5, 8192), (3, 8200), (4, 32003),
                                 (3, 50257), (2, 131077)])
def test_backward(N, V, dtype):
    from src.model import token_logprobs
    z, t = rows(N, V, dtype, V)
    if N > 2:
        t[1] = -1
        z[1] = NAN
        z[2, V // 2:] = -INF
    for n in sorted({0, 1, min(V, 20)}):
        print(f"N={N} V={V} n={n} {dtype}", flush=True)
        g = torch.Generator().manual_seed(n)
        gs = [torch.randn(N, generator=g), torch.randn(N, generator=g), torch.randn(N, n, generator=g) if n else None]
        x = z.cuda().requires_grad_(True)
        r = token_logprobs(x, t.cuda(), n)
        out = [r.logprob, r.entropy] + ([r.top_logprob] if n else [])
        d, = torch.autograd.grad(out, x, [v.cuda() for v in gs if v is not None])
        assert d.dtype == dtype and d.shape == x.shape
        index = r.top_index.cpu().numpy()
        nums = [None if v is None else v.double().numpy() for v in gs]
        want = otok.token_logprobs_grad_f64(z.double().numpy(), t.numpy(), index, *nums)
        close(d, want, grad_bound(z, t.numpy(), index, nums, want, dtype, V), "gradient")


def test_backward_odd_values():
    from src.model import token_logprobs
    V = 2500
    z, t = rows(8, V, torch.float32, 3)
    z[1] = -INF
    z[2, 7] = NAN
    z[3, 7] = INF
    t[4] = V
    z[5] = torch.finfo(torch.float32).min
    z[6, 1:] = torch.finfo(torch.float32).min
    z[7, :] = 1.5
    x = z.cuda().requires_grad_(True)
    for n in (0, 3):
        r = token_logprobs(x, t.cuda(), n)
        gs = [torch.full((8,), 2.0), torch.full((8,), -3.0)]
        d, = torch.autograd.grad([r.logprob, r.entropy], x, [v.cuda() for v in gs])
        index = r.top_index.cpu().numpy()
        nums = [v.double().numpy() for v in gs] + [None]
        want = otok.token_logprobs_grad_f64(z.double().numpy(), t.numpy(), index, *nums)
        want[[2, 3]] = NAN
        close(d, want, grad_bound(z, t.numpy(), index, nums, want, torch.float32, V), "gradient")


def test_backward_of_some_outputs():
    """Gradients of one output alone, expanded ones, and none."""
    from src.model import token_logprobs
    z, t = rows(4, 300, torch.float32, 8)
    x = z.cuda().requires_grad_(True)
    zero = np.zeros(4)
    r = token_logprobs(x, t.cuda(), 2)
    index = r.top_index.cpu().numpy()
    for i, loss in enumerate((r.logprob.sum(), r.entropy.sum(), r.top_logprob.sum())):
        d, = torch.autograd.grad(loss, x, retain_graph=True)
        nums = [np.ones(4) if i == 0 else zero, np.ones(4) if i == 1 else zero, np.ones((4, 2)) if i == 2 else None]
        want = otok.token_logprobs_grad_f64(z.double().numpy(), t.numpy(), index, *nums)
        close(d, want, grad_bound(z, t.numpy(), index, nums, want, torch.float32, 300), i)
    assert not r.top_index.requires_grad
    # differences of the operator itself: rounding of the outputs over the step
    h = 2.0 ** -6
    e = torch.zeros_like(z)
    e[:, 5] = h
    up, down = (token_logprobs((z + s * e).cuda(), t.cuda()).entropy.double() for s in (1, -1))
    d, = torch.autograd.grad(r.entropy.sum(), x)
    assert ((up - down) / (2 * h) - d[:, 5].double()).abs().max() <= 80 * unit(300) / h + h * h


@pytest.mark.parametrize("n", [0, 3])
def test_derivatives_of_the_gradient_and_transforms(n):
    """Second derivatives, forward mode, vmap and vectorised Jacobians take
    torch's operations and agree with the kernels' first derivatives."""
    from src.model import token_logprobs
    z, t = rows(3, 50, torch.float32, 4)
    z, t = z.cuda(), t.cuda()

    def loss(x):
        r = token_logprobs(x, t, n)
        return (r.logprob * 2 + r.entropy.square()).sum() + r.top_logprob.square().sum()
    x = z.clone().requires_grad_(True)
    d, = torch.autograd.grad(loss(x), x)
    d2, = torch.autograd.grad(loss(x), x, create_graph=True)
    v = torch.randn(z.shape, generator=torch.Generator().manual_seed(1)).cuda()
    hv, = torch.autograd.grad((d2 * v).sum(), x)
    close(d2.detach(), d.double().cpu().numpy(), 1e-4 * (1 + d.abs().cpu().numpy()), "first derivatives")
    h = 2.0 ** -8
    y = [(z + s * h * v).requires_grad_(True) for s in (1, -1)]
    up, down = (torch.autograd.grad(loss(w), w)[0].double() for w in y)
    # (second-order truncation, and rounding of gradients of a few units over 2 h)
    close(hv, ((up - down) / (2 * h)).cpu().numpy(), 0.05 + 0 * hv.cpu().numpy(), "second derivatives")
    g = torch.func.grad(loss)(z)
    close(g, d.double().cpu().numpy(), 1e-4 * (1 + d.abs().cpu().numpy()), "func.grad")
    _, jv = torch.func.jvp(loss, (z,), (v,))
    assert abs(jv - (d * v).sum()) <= 1e-3 * (1 + (d * v).abs().sum())
    each = torch.func.vmap(lambda a, b: token_logprobs(a, b, n).logprob)(z, t)
    assert (each - token_logprobs(z, t).logprob).abs().max() <= 2 * unit(50) * 16
    J = torch.autograd.functional.jacobian(lambda a: token_logprobs(a, t, n).logprob, z, vectorize=True)
    J2 = torch.autograd.functional.jacobian(lambda a: token_logprobs(a, t, n).logprob, z)
    assert (J - J2).abs().max() <= 1e-5


def test_rows_past_2_31_elements():
    """The last rows of logits of more than 2^31 elements, and their gradient."""
    from src.model import kernels
    V, N = 50257, 42800
    z = torch.empty(N, V, device="cuda", dtype=torch.bfloat16).normal_(generator=torch.Generator("cuda").manual_seed(0))
    t = torch.full((N,), -1, device="cuda")
    t[-2:] = torch.tensor([0, V - 1], device="cuda")
    got = kernels.token_logprobs(z, t, 3, need_stats=True)
    check(z[-2:], t[-2:], 3, [x[-2:] for x in got[:4]], V)
    d = kernels.token_logprobs_bwd(z, t, got[3][:, :0], got[4], torch.ones(N, device="cuda"))
    want = otok.token_logprobs_grad_f64(z[-2:].double().cpu().numpy(), t[-2:].cpu().numpy(), None, np.ones(2))
    close(d[-2:], want, np.abs(want) * (2.0 ** -8 + 4 * unit(V)), "gradient")
    assert not d[:-2].any()


def test_streams_and_graphs():
    """Two calls on two streams, and a captured forward and backward replayed
    with new logits, tokens and eager work in between."""
    from src.model import kernels
    z, t = rows(64, 5003, torch.bfloat16, 6)
    z, t = z.cuda(), t.cuda()
    z2, t2 = z.flip(0).contiguous(), t.flip(0).contiguous()
    want, want2 = kernels.token_logprobs(z, t, 8), kernels.token_logprobs(z2, t2, 8)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(a):
            x = kernels.token_logprobs(z, t, 8)
        with torch.cuda.stream(b):
            y = kernels.token_logprobs(z2, t2, 8)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(x, want)) and all(torch.equal(p, q) for p, q in zip(y, want2))
    zs, ts, g = z.clone(), t.clone(), torch.ones(64, device="cuda")

    def step():
        r = kernels.token_logprobs(zs, ts, 8, need_stats=True)
        return r, kernels.token_logprobs_bwd(zs, ts, r[3], r[4], g, g, r[2])
    with torch.cuda.stream(a):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r, d = step()
    for k in range(4):
        zs.copy_(z if k % 2 else z2)
        ts.copy_(t if k % 2 else t2)
        graph.replay()
        e, de = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(r, e)) and torch.equal(d, de), k


def test_refusals():
    from src.model import kernels, token_logprobs
    z, t = torch.zeros(2, 9, device="cuda"), torch.zeros(2, device="cuda").long()
    for f in (kernels.token_logprobs, token_logprobs):
        with pytest.raises(ValueError, match="alternatives"):
            f(z, t, 10)
        with pytest.raises(ValueError, match="alternatives"):
            f(torch.zeros(2, 100, device="cuda"), t, 65)
        with pytest.raises(ValueError, match="alternatives"):
            f(z, t, -1)
        with pytest.raises(TypeError, match="int64"):
            f(z, t.int())
        with pytest.raises(TypeError, match="dtype"):
            f(z.half(), t)
        with pytest.raises(AssertionError):
            f(z, t[:1])
        with pytest.raises(RuntimeError):
            f(z.cpu(), t)
        with pytest.raises(RuntimeError):
            f(z, t.cpu())
    r = kernels.token_logprobs(z, t, 2, need_stats=True)
    with pytest.raises(AssertionError):
        kernels.token_logprobs_bwd(z, t, r[3], r[4][:1], torch.ones(2, device="cuda"))
    with pytest.raises(AssertionError):
        kernels.token_logprobs_bwd(z, t, r[3], r[4], torch.ones(2, device="cuda").double())
    with pytest.raises(AssertionError):
        kernels.token_logprobs_bwd(z, t, r[3][:1], r[4], torch.ones(2, device="cuda"))
