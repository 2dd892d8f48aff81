"""Dropout without a mask on the GPU against the oracle: what is kept is equal
element by element, values within their roundings (the factor's and the
product's 2^-24 each, the sum's, and the output type's)."""
import numpy as np
import pytest
import torch

from oracle import tokens as otok

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def seed_of(v):
    return torch.tensor([v], device="cuda")


def close(got, want, size, dtype):
    got = got.double().cpu().numpy()
    assert np.all(np.abs(got - want) <= 3 * 2.0 ** -24 * size + torch.finfo(dtype).eps / 2 * np.abs(want))


@pytest.mark.parametrize("xt,rt", [(F32, None), (BF16, None), (F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("M,C,p", [(1, 1, 0.5), (3, 7, 0.1), (5, 8, 0.9), (2, 9, 0.3), (300, 33, 0.25), (64, 512, 0.1),
                                   (7, 1365, 0.5), (3, 4096, 0.2), (1, 70001, 0.7), (40000, 3, 0.4), (2, 300003, 0.1)])
def test_values(M, C, p, xt, rt):
    from src.model import counter_dropout
    print(f"M={M} C={C} p={p} {xt} {rt}", flush=True)
    g = torch.Generator().manual_seed(C)
    x = torch.randn(M, C, generator=g).to(xt)
    r = None if rt is None else torch.randn(M, C, generator=g).to(rt)
    seed, stream, drop = 2 ** 62 + 12345 * C, C % 11, round(p * 65536)
    xd = x.cuda().requires_grad_(True)
    rd = None if r is None else r.cuda().requires_grad_(True)
    y = counter_dropout(xd, p, seed_of(seed), stream, rd)
    out = xt if rt in (None, xt) else F32
    assert y.dtype == out and y.is_contiguous()
    d = otok.dropout_f64(x.double().numpy(), drop, seed, stream)
    res = np.zeros((M, C)) if r is None else r.double().numpy()
    close(y.detach(), d + res, np.abs(d) + np.abs(res), out)
    if r is None:
        keep = otok.kept(M, C, drop, seed, stream)
        assert np.array_equal((y.detach() != 0).cpu().numpy(), keep & (x != 0).numpy())
    gy = torch.randn(M, C, generator=g).to(out)
    grads = torch.autograd.grad(y, [xd] + ([] if rd is None else [rd]), gy.cuda())
    d = otok.dropout_f64(gy.double().numpy(), drop, seed, stream)
    close(grads[0], d, np.abs(d), xt)
    if r is not None:
        assert torch.equal(grads[1].cpu(), gy.to(rt))


def test_ends_of_the_range():
    """Nothing dropped, everything, the smallest shares; NaN and infinities in
    dropped places."""
    from src.model import counter_dropout
    x = torch.randn(50, 40, device="cuda")
    assert torch.equal(counter_dropout(x, 0.0, None), x)
    assert torch.equal(counter_dropout(x, 2.0 ** -18, None, residual=x), x + x)
    s = seed_of(5)
    assert not counter_dropout(torch.full_like(x, float("nan")), 1.0, s).any()
    assert torch.equal(counter_dropout(x, 1.0, s, residual=x), x)
    keep = torch.from_numpy(otok.kept(50, 40, 32768, 5, 0)).cuda()
    y = counter_dropout(torch.where(keep, x, torch.full_like(x, float("inf"))), 0.5, s)
    assert torch.equal(y, torch.where(keep, x * 2, torch.zeros_like(x)))
    y = counter_dropout(torch.where(keep, torch.full_like(x, float("nan")), x), 0.5, s)
    assert torch.equal(y.isnan(), keep) and not y[~keep].any()
    assert counter_dropout(x[:0], 0.5, s).shape == (0, 40) and counter_dropout(x[:, :0], 0.5, s).shape == (50, 0)


@pytest.mark.parametrize("seed,stream", [(-5, 2 ** 32 - 1), (-(2 ** 63), 0), (2 ** 63 - 1, 1), (0, 0)])
def test_every_seed_is_one(seed, stream):
    from src.model import counter_dropout
    y = counter_dropout(torch.ones(33, 50, device="cuda"), 0.5, seed_of(seed), stream)
    assert np.array_equal((y != 0).cpu().numpy(), otok.kept(33, 50, 32768, seed % 2 ** 64, stream))


def test_tensors_past_the_caches():
    """bf16 rows of more than 256 MB, whose loads are streamed, at an odd width."""
    from src.model import counter_dropout
    M, C = 70003, 2001
    g = torch.Generator("cuda").manual_seed(1)
    x, r = (torch.empty(M, C, device="cuda", dtype=BF16).normal_(generator=g) for _ in range(2))
    y = counter_dropout(x, 0.25, seed_of(6), 3, r)
    for at in (0, 1, 35001, M - 2, M - 1):
        keep = otok.kept(1, C, 16384, 6, 3, first=at)[0]
        d = np.where(keep, x[at].double().cpu().numpy() * (65536 / 49152), 0)
        want = d + r[at].double().cpu().numpy()
        close(y[at], want, np.abs(d) + np.abs(want - d), BF16)


def test_layouts():
    """Strided, transposed and expanded rows, odd addresses, several leading
    dimensions, one: the mask goes by row and column, not by address."""
    from src.model import counter_dropout
    s = seed_of(2 ** 63 - 1)
    base = torch.randn(12, 1003, device="cuda")
    r = torch.randn(12, 1003, device="cuda")
    views = [base[:, 1:900], base.t()[:700].t(), base[:1].expand(12, 1003)[:, :77], base.view(3, 4, 1003)[:, 1:3], base[3],
             torch.cat([base.reshape(-1), base.new_zeros(1)])[1:].view(12, 1003), base[:, ::2]]
    for v in views:
        for t in (v, v.bfloat16(), v.bfloat16()[..., 1:]):
            want = counter_dropout(t.clone(memory_format=torch.contiguous_format), 0.3, s, 4)
            assert torch.equal(counter_dropout(t, 0.3, s, 4), want)
        rr = r.flatten()[:v.numel()].view(v.shape)
        want = counter_dropout(v.contiguous(), 0.3, s, 4, rr)
        assert torch.equal(counter_dropout(v, 0.3, s, 4, rr), want)
        assert torch.equal(counter_dropout(v, 0.3, s, 4, rr.t().contiguous().t() if rr.dim() == 2 else rr), want)


def test_derivatives_of_the_gradient_and_transforms():
    from src.model import counter_dropout
    s = seed_of(9)
    x = torch.randn(6, 21, device="cuda", requires_grad=True)
    v = torch.randn(6, 21, device="cuda")

    def f(a):
        return counter_dropout(a.square(), 0.4, s, 1, a)
    y = f(x)
    d, = torch.autograd.grad(y, x, v)
    d2, = torch.autograd.grad(f(x), x, v, create_graph=True)
    keep = torch.from_numpy(otok.kept(6, 21, 26214, 9, 1)).cuda()
    k = keep * (65536 / (65536 - 26214))
    assert torch.allclose(d, v * (2 * k * x + 1), rtol=1e-6, atol=1e-6)
    assert torch.allclose(d2, d, rtol=1e-6, atol=1e-6)
    dd, = torch.autograd.grad(d2.sum(), x)
    assert torch.allclose(dd, 2 * k * v, rtol=1e-6, atol=1e-6)
    _, jv = torch.func.jvp(f, (x.detach(),), (v,))
    assert torch.allclose(jv, d, rtol=1e-6, atol=1e-6)
    assert torch.allclose(torch.func.grad(lambda a: (f(a) * v).sum())(x.detach()), d, rtol=1e-6, atol=1e-6)


def test_rows_past_2_31_elements():
    from src.model import kernels
    M, C, s = 33000, 65551, seed_of(3)
    x = torch.ones(M, C, device="cuda", dtype=BF16)
    y = kernels.dropout(x, 0.5, s, 2)
    for r in (0, 32765, M - 1):
        assert np.array_equal((y[r] != 0).cpu().numpy(), otok.kept(1, C, 32768, 3, 2, first=r)[0])


def test_streams_and_graphs():
    """The seed is read when a graph replays; two streams do not meet."""
    from src.model import counter_dropout
    s, x = seed_of(1), torch.randn(100, 515, device="cuda", dtype=BF16, requires_grad=True)
    gy = torch.randn(100, 515, device="cuda", dtype=BF16)

    def step():
        y = counter_dropout(x, 0.3, s, 6)
        return y, torch.autograd.grad(y, x, gy)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        del_ = step()
        del del_
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, d = step()
    y, d = y.detach(), d.detach()
    for k in range(4):
        s.fill_(1000 + k)
        graph.replay()
        with torch.no_grad():
            want = counter_dropout(x, 0.3, s, 6), counter_dropout(gy, 0.3, s, 6)
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(d, want[1]), k
    seeds = [seed_of(11), seed_of(12)]
    want = [counter_dropout(x.detach(), 0.3, t) for t in seeds]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for t, st in zip(seeds, streams):
        with torch.cuda.stream(st):
            got.append(counter_dropout(x.detach(), 0.3, t))
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_seed_changed_before_the_backward():
    """Its mask would be another one: autograd refuses."""
    from src.model import counter_dropout
    s, x = seed_of(1), torch.randn(4, 8, device="cuda", requires_grad=True)
    y = counter_dropout(x, 0.5, s)
    s.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


def test_refusals():
    from src.model import counter_dropout
    x, s = torch.zeros(2, 9, device="cuda"), seed_of(1)
    with pytest.raises(ValueError, match="probability"):
        counter_dropout(x, 1.5, s)
    with pytest.raises(ValueError, match="probability"):
        counter_dropout(x, float("nan"), s)
    with pytest.raises(ValueError, match="seed"):
        counter_dropout(x, 0.5, None)
    with pytest.raises(TypeError, match="seed"):
        counter_dropout(x, 0.5, 7)
    with pytest.raises(TypeError, match="seed"):
        counter_dropout(x, 0.5, s.int())
    with pytest.raises(AssertionError):
        counter_dropout(x, 0.5, torch.cat([s, s]))
    with pytest.raises(ValueError, match="stream"):
        counter_dropout(x, 0.5, s, -1)
    with pytest.raises(ValueError, match="stream"):
        counter_dropout(x, 0.5, s, 1 << 32)
    with pytest.raises(AssertionError):
        counter_dropout(x, 0.5, s, residual=x[:1])
    with pytest.raises(TypeError, match="dtype"):
        counter_dropout(x.half(), 0.5, s)
    with pytest.raises(RuntimeError):
        counter_dropout(x.cpu(), 0.5, s.cpu())
    with pytest.raises(RuntimeError):
        counter_dropout(x, 0.5, s.cpu())
    with pytest.raises(AssertionError):
        counter_dropout(x[0, 0], 0.5, s)
