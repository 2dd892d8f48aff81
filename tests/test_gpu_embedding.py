"""Scaled embedding lookup with dropout and its gradient on the GPU against the
float64 oracle.  A looked-up value has the factor's rounding and the product's
(2^-24 each); a gradient's element is a float32 sum of n terms, off by at most
(n + 3) 2^-24 of the sum of their absolute values; both are rounded to their
type once."""
import numpy as np
import pytest
import torch

from oracle import tokens as otok

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def seed_of(v):
    return torch.tensor([v], device="cuda")


def check_grad(got, tokens, g, V, pad=None):
    t = tokens.reshape(-1).cpu().numpy()
    sums, size = otok.embedding_grad_f64(t, g, V, pad)
    n = np.bincount(t[(t >= 0) & (t < V)], minlength=V)[:, None]
    bound = (n + 3) * 2.0 ** -24 * size + torch.finfo(got.dtype).eps / 2 * np.abs(sums)
    assert np.all(np.abs(got.double().cpu().numpy() - sums) <= bound)


def some_tokens(N, V, kind, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "uniform":
        return torch.randint(V, (N,), generator=g)
    if kind == "words":
        return ((V + 1) ** torch.rand(N, generator=g) - 1).long().clamp(0, V - 1)
    if kind == "one":
        return torch.full((N,), V // 2)
    # mostly one token, runs of others, and some outside the vocabulary
    t = torch.randint(V, (N,), generator=g)
    t[N // 8:N // 2] = V - 1
    t[N // 2:3 * N // 4] = 0
    t[::7] = torch.tensor([-1, V, 2 ** 62, -(2 ** 62)]).repeat(N)[:len(t[::7])]
    return t


@pytest.mark.parametrize("wt,ot", [(F32, F32), (BF16, BF16), (F32, BF16), (BF16, F32)])
@pytest.mark.parametrize("N,V,C,kind", [(1, 1, 1, "uniform"), (3, 5, 7, "uniform"), (70, 11, 8, "words"),
                                        (1000, 65, 33, "words"), (33, 300, 64, "one"), (64, 3, 16, "one"),
                                        (5000, 257, 24, "mixed"), (2049, 70001, 20, "words"), (9000, 700, 12, "one"),
                                        (512, 513, 1021, "uniform"), (130, 1000, 4096, "mixed"),
                                        (40000, 2, 9, "uniform"), (31, 1, 5, "one"), (32, 1, 5, "one"), (33, 1, 5, "one")])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_lookup_and_gradient(N, V, C, kind, p, wt, ot):
    from src.model import token_embedding
    print(f"N={N} V={V} C={C} {kind} p={p} {wt} {ot}", flush=True)
    t = some_tokens(N, V, kind, V)
    g = torch.Generator().manual_seed(C)
    w, gy = torch.randn(V, C, generator=g).to(wt), torch.randn(N, C, generator=g).to(ot)
    wd = w.cuda().requires_grad_(True)
    y = token_embedding(t.cuda(), wd, 1.7, out_dtype=ot, p=p, seed=seed_of(31), stream=2)
    drop = round(p * 65536)
    keep = otok.kept(N, C, drop, 31, 2) * (65536 / (65536 - drop))
    out = ((t < 0) | (t >= V)).numpy()
    want = w.double().numpy()[t.clamp(0, V - 1).numpy()] * 1.7 * keep
    got = y.detach().double().cpu().numpy()
    assert np.isnan(got[out]).all()
    assert np.all(np.abs(got - want)[~out] <= (2 * 2.0 ** -24 + torch.finfo(ot).eps / 2) * np.abs(want)[~out])
    d, = torch.autograd.grad(y, wd, gy.cuda(), retain_graph=True)
    assert d.dtype == wt and d.shape == (V, C)
    check_grad(d, t, gy.double().numpy() * 1.7 * keep, V)
    assert torch.equal(d, torch.autograd.grad(y, wd, gy.cuda())[0])


def test_same_as_torch():
    """Without a scale a lookup is a copy, and a gradient of few tokens torch's."""
    from src.model import token_embedding
    w = torch.randn(50, 24, device="cuda", requires_grad=True)
    t = torch.randint(50, (4, 9), device="cuda")
    y = token_embedding(t, w)
    assert y.shape == (4, 9, 24) and torch.equal(y, torch.nn.functional.embedding(t, w))
    gy = torch.randn_like(y)
    a, = torch.autograd.grad(y, w, gy)
    b, = torch.autograd.grad(torch.nn.functional.embedding(t, w), w, gy)
    assert torch.allclose(a, b, rtol=0, atol=2.0 ** -20)
    a, = torch.autograd.grad(token_embedding(t, w, padding_idx=int(t[0, 0])), w, gy)
    b, = torch.autograd.grad(torch.nn.functional.embedding(t, w, padding_idx=int(t[0, 0])), w, gy)
    assert torch.allclose(a, b, rtol=0, atol=2.0 ** -20) and not a[t[0, 0]].any()


def test_dropout_of_rows_is_dropout():
    """The lookup's mask is counter_dropout's of the rows."""
    from src.model import counter_dropout, token_embedding
    w, t, s = torch.randn(40, 77, device="cuda"), torch.randint(40, (3, 20), device="cuda"), seed_of(8)
    a = token_embedding(t, w, p=0.4, seed=s, stream=5)
    assert torch.equal(a, counter_dropout(token_embedding(t, w), 0.4, s, 5))


def test_layouts():
    """Strided and transposed weights, tokens and gradients, odd addresses."""
    from src.model import kernels
    g = torch.Generator().manual_seed(0)
    t = torch.randint(30, (40,), generator=g).cuda()
    base = torch.randn(31, 80, generator=g).cuda()
    for dt in (F32, BF16):
        for w in (base.to(dt)[:30, 3:70], base.to(dt).t().contiguous().t()[:30], base.to(dt)[:1].expand(30, 80),
                  base.to(dt).flatten()[1:1 + 30 * 41].view(30, 41)):
            want = kernels.embedding(t, w.contiguous(), 0.5)
            assert torch.equal(kernels.embedding(t, w, 0.5), want)
            assert torch.equal(kernels.embedding(t.repeat_interleave(2)[::2], w, 0.5), want)
        gy = torch.randn(40, 90, generator=g).to(dt).cuda()
        for v in (gy[:, 1:70], gy.t().contiguous().t(), gy[:1].expand(40, 90), gy[:, ::2]):
            want = kernels.embedding_bwd(t, v.contiguous(), 30, 0.5)
            assert torch.equal(kernels.embedding_bwd(t, v, 30, 0.5), want)
    gy = torch.randn(2, 5, 4, 16, generator=g).cuda().transpose(0, 1)
    want = kernels.embedding_bwd(t.view(5, 2, 4), gy.contiguous(), 30)
    assert torch.equal(kernels.embedding_bwd(t.view(5, 2, 4), gy, 30), want)
    # nothing at all: every row of the gradient is still written
    for _ in range(3):
        torch.full((30, 16), float("nan"), device="cuda")
        assert not kernels.embedding_bwd(t[:0], gy.new_zeros(0, 16), 30).any()
    assert kernels.embedding(t[:0], base).shape == (0, 80) and kernels.embedding_bwd(t, gy.new_zeros(40, 0), 30).shape == (30, 0)


def test_odd_gradients():
    """NaN and infinities reach the token's row alone, and not from what is
    dropped or not counted."""
    from src.model import kernels
    t = torch.tensor([3, 4, 3, -1, 9], device="cuda")
    gy = torch.ones(5, 16, device="cuda")
    gy[1] = float("nan")
    gy[3] = float("inf")
    d = kernels.embedding_bwd(t, gy, 10)
    assert d[4].isnan().all() and torch.equal(d[3], torch.full_like(d[3], 2)) and d[9].eq(1).all()
    assert not d[[0, 1, 2, 5, 6, 7, 8]].any()
    d = kernels.embedding_bwd(t, torch.full_like(gy, float("nan")), 10, p=1.0, seed=seed_of(1))
    assert not d.any()
    d = kernels.embedding_bwd(t, gy, 10, padding_idx=4)
    assert not d[4].any()


def test_derivatives_of_the_gradient_and_transforms():
    from src.model import token_embedding
    s, t = seed_of(4), torch.tensor([[1, 1, 5], [0, -1, 5]], device="cuda")
    w = torch.randn(6, 10, device="cuda", requires_grad=True)
    v = torch.randn(2, 3, 10, device="cuda")

    def f(a):
        y = token_embedding(t, a, 2.0, 5, p=0.25, seed=s)
        return torch.where(y.isnan(), 0.0, y).square()
    d, = torch.autograd.grad(f(w), w, v)
    d2, = torch.autograd.grad(f(w), w, v, create_graph=True)
    assert torch.allclose(d, d2.detach(), rtol=1e-5, atol=1e-5) and not d[5].any()
    u = torch.randn_like(w)
    hv, = torch.autograd.grad((d2 * u).sum(), w)
    k = torch.from_numpy(otok.kept(6, 10, 16384, 4, 0)).view(2, 3, 10).cuda() * (2.0 * 65536 / 49152)
    want = torch.zeros(6, 10, device="cuda")
    for i in range(2):
        for j in range(3):
            if t[i, j] in (0, 1):
                want[t[i, j]] += 2 * v[i, j] * k[i, j] ** 2 * u[t[i, j]]
    assert torch.allclose(hv, want, rtol=1e-5, atol=1e-5)
    _, jv = torch.func.jvp(f, (w.detach(),), (u,))
    assert torch.allclose((jv * v).sum(), (d * u).sum() + ((2 * w * u)[5] * (v * k * k)[t == 5]).sum() * 0, rtol=1e-3, atol=1e-3)
    assert torch.allclose(torch.func.grad(lambda a: (f(a) * v).sum())(w.detach()), d, rtol=1e-5, atol=1e-5)


def test_rows_past_2_31_elements():
    from src.model import kernels
    V, C = 131072, 16400
    w = torch.zeros(V, C, device="cuda", dtype=BF16)
    w[-1] = 1.5
    t = torch.tensor([V - 1, 0, V - 1], device="cuda")
    y = kernels.embedding(t, w, 2.0)
    assert y[0].eq(3).all() and not y[1].any()
    d = kernels.embedding_bwd(t, y, V)
    assert d[-1].eq(6).all() and not d[-3:-1].any() and not d[1::4096].any()


@pytest.mark.parametrize("dtype,C", [(BF16, 2001), (F32, 1001), (BF16, 4096)])
def test_gradients_past_the_caches(dtype, C):
    """Weights of more than 256 MB, whose gradient is streamed, at odd widths:
    rows that occur once, often and not at all."""
    from src.model import kernels
    V, N = 70001, 3000
    g = torch.Generator().manual_seed(C)
    t = torch.cat([torch.randint(V, (N - 700,), generator=g), torch.full((600,), V - 1), torch.arange(100)])
    gy = torch.randn(N, C, generator=g).to(dtype)
    d = kernels.embedding_bwd(t.cuda(), gy.cuda(), V, 0.5, padding_idx=7)
    rows = torch.unique(t)
    some = rows[torch.randperm(len(rows), generator=g)[:40]].tolist() + [V - 1, 7, 0, 99]
    for v in some:
        mine = gy[t == v].double() * 0.5
        want, size = mine.sum(0), mine.abs().sum(0)
        if v == 7:
            want = size = torch.zeros(C, dtype=torch.float64)
        bound = (len(mine) + 3) * 2.0 ** -24 * size + torch.finfo(dtype).eps / 2 * want.abs()
        assert ((d[v].double().cpu() - want).abs() <= bound).all(), v
    none = torch.ones(V, dtype=torch.bool)
    none[rows] = False
    assert not d[none.cuda()].any()


def test_streams_and_graphs():
    """Captured with the seed and tokens in place and replayed with others; two
    backward passes on two streams have a workspace each."""
    from src.model import kernels, token_embedding
    V, C = 900, 136
    w, s = torch.randn(V, C, device="cuda", requires_grad=True), seed_of(1)
    t, t2 = some_tokens(5000, V, "mixed", 1).cuda(), some_tokens(5000, V, "words", 2).cuda()
    gy = torch.randn(5000, C, device="cuda")
    ts = t.clone()

    def step():
        y = token_embedding(ts, w, 3.0, p=0.2, seed=s)
        return y.detach(), torch.autograd.grad(y, w, gy)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, d = step()
    for k in range(4):
        s.fill_(50 + k)
        ts.copy_(t2 if k % 2 else t)
        graph.replay()
        with torch.no_grad():
            want = kernels.embedding(ts, w, 3.0, None, 0.2, s), kernels.embedding_bwd(ts, gy, V, 3.0, None, None, 0.2, s)
        torch.cuda.synchronize()
        assert torch.equal(y.nan_to_num(7), want[0].nan_to_num(7)) and torch.equal(d, want[1]), k
    want = [kernels.embedding_bwd(a, gy, V) for a in (t, t2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for a, st in zip((t, t2), streams):
            with torch.cuda.stream(st):
                got.append(kernels.embedding_bwd(a, gy, V))
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals():
    from src.model import kernels, token_embedding
    w, t, s = torch.zeros(5, 8, device="cuda"), torch.zeros(3, device="cuda").long(), seed_of(1)
    for f in (lambda *a, **k: token_embedding(a[1], a[0], **k), lambda *a, **k: kernels.embedding(a[1], a[0], **k)):
        with pytest.raises(TypeError, match="int64"):
            f(w, t.int())
        with pytest.raises(TypeError, match="dtype"):
            f(w.half(), t)
        with pytest.raises(TypeError, match="dtype"):
            f(w, t, out_dtype=torch.float16)
        with pytest.raises(AssertionError):
            f(w[0], t)
        with pytest.raises(AssertionError):
            f(w[:0], t)
        with pytest.raises(ValueError, match="seed"):
            f(w, t, p=0.5)
        with pytest.raises(ValueError, match="probability"):
            f(w, t, p=-0.5, seed=s)
        with pytest.raises(RuntimeError):
            f(w, t.cpu())
        with pytest.raises(RuntimeError):
            f(w.cpu(), t.cpu())
    for pad in (-1, 5):
        with pytest.raises(ValueError, match="padding_idx"):
            token_embedding(t, w, padding_idx=pad)
    with pytest.raises(AssertionError):
        kernels.embedding_bwd(t, w, 5)
    with pytest.raises(AssertionError):
        kernels.embedding_bwd(t, w[:3], 0)
