"""Sampling on the GPU against the float64 oracle: tokens are equal.

A weight on the GPU is off by at most 2^-22 (1 + log2 of its distance from
the largest) relatively, under 2^-17 for the rows here, and those errors have
no common sign; a row whose nearest border lies closer than 2^-17 is not
decided by the definition and may fall on either side (none of these do)."""
import numpy as np
import pytest
import torch

from oracle.sampling import sample_f64

SURE = 2.0 ** -17


def rows(B, V, dtype, seed):
    """Language-model-like rows: weights that fall with the rank."""
    g = torch.Generator().manual_seed(seed)
    rank = torch.rand(B, V, generator=g).argsort(-1).float() + 1
    z = (4 - 1.1 * rank.log() + 0.5 * torch.randn(B, V, generator=g)).to(dtype)
    return z, torch.rand(B, generator=g)


def check(z, u, T, k, p, m, got):
    B = z.shape[0]
    val = lambda s, b: float(s[b]) if torch.is_tensor(s) else s  # noqa: E731
    unsure = 0
    for b in range(B):
        want, margin = sample_f64(z[b].double().numpy(), float(u[b]), val(T, b), int(val(k, b)), val(p, b), val(m, b))
        if margin < SURE:
            unsure += 1
            continue
        assert got[b] == want, (b, int(got[b]), want, margin, val(T, b), val(k, b), val(p, b), val(m, b))
    return unsure


def run(z, u, T=1.0, k=0, p=1.0, m=0.0):
    from src.model import kernels
    dev = lambda s: s.cuda() if torch.is_tensor(s) else s  # noqa: E731
    return kernels.sample(z.cuda(), u.cuda(), dev(T), dev(k), dev(p), dev(m)).cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (5, 63), (4, 64), (3, 65), (2, 1023), (7, 1025), (3, 16385), (4, 50257),
                                 (2, 131072), (1, 200000)])
def test_sample_against_oracle(B, V, dtype):
    """Every filter alone and together, each row with its own settings."""
    z, u = rows(B, V, dtype, V)
    g = torch.Generator().manual_seed(V)
    T = 0.5 + torch.rand(B, generator=g)
    k = torch.tensor([1, 2, 7, 50, 400, 5000, 0, V])[torch.randint(0, 8, (B,), generator=g)].int()
    p = torch.tensor([0.95, 0.5, 0.1, 1.0, 0.999, 0.0])[torch.randint(0, 6, (B,), generator=g)]
    m = torch.tensor([0.0, 0.05, 0.3, 0.001])[torch.randint(0, 4, (B,), generator=g)]
    close = 0
    for args in ((1.0, 0, 1.0, 0.0), (T, 0, 1.0, 0.0), (T, k, 1.0, 0.0), (T, 0, p, 0.0), (T, 0, 1.0, m), (T, k, p, 0.0),
                 (T, k, p, m), (0.0, k, p, m), (2.0, min(40, V), 0.9, 0.02)):
        print(f"V={V} {dtype} settings {[('tensor' if torch.is_tensor(a) else a) for a in args]}", flush=True)
        close += check(z, u, *args, run(z, u, *args))
    print(f"{close} of {9 * B} rows too close to a border")


@pytest.mark.gpu
def test_sample_frequencies():
    """Evenly spaced numbers give every token its share (the draw's borders
    are exact to one number)."""
    z = torch.randn(1, 37, generator=torch.Generator().manual_seed(1)) * 2
    n = 1 << 16
    u = (torch.arange(n) + 0.5) / n
    got = torch.bincount(run(z.expand(n, 37), u, T=0.7), minlength=37).double() / n
    want = torch.softmax(z[0].double() / 0.7, 0)
    assert (got - want).abs().max() <= 1.0 / n + 2.0 ** -20


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sample_ties(dtype):
    """Equal logits: the lowest indexes stay, and borders at exact shares."""
    V = 4096
    z = torch.zeros(6, V, dtype=dtype)
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1.0 - 2.0 ** -13, 2.0 ** -12])
    assert run(z, u).tolist() == [int(x * V) for x in u]
    assert run(z, u, k=1000).tolist() == [int(np.floor(float(x) * 1000)) for x in u]
    assert run(z, u, p=0.5).tolist() == [int(x * V // 2) for x in u]
    # 2,000 equal ones below one larger, and the cut inside them
    z[:, 1:2001] = -1.0
    z[:, 2001:] = -3.0
    z[:, 3000] = 2.0
    got = run(z, u, k=500)
    assert check(z, u, 1.0, 500, 1.0, 0.0, got) == 0 and got.max() <= 3000
    got = run(z, u, p=0.7, k=1500)
    assert check(z, u, 1.0, 1500, 0.7, 0.0, got) <= 1


@pytest.mark.gpu
def test_sample_odd_values():
    """-inf (masked), NaN, infinities, huge and tiny values, an empty row."""
    inf, nan = float("inf"), float("nan")
    V = 300
    base = torch.randn(9, V, generator=torch.Generator().manual_seed(2))
    base[0] = -inf
    base[1] = nan
    base[2, :] = -inf
    base[2, 123] = -7.0
    base[3, ::2] = -inf
    base[4, 5:200] = nan
    base[5, [7, 250]] = inf
    base[6] *= 1e30
    base[7] *= 1e-38
    base[8] = torch.finfo(torch.float32).min
    u = torch.tensor([0.3, 0.4, 0.9, 0.6, 0.7, 0.75, 0.5, 0.31, 0.5])
    for args in ((1.0, 0, 1.0, 0.0), (0.7, 20, 1.0, 0.0), (1.3, 0, 0.8, 0.0), (1.0, 100, 0.9, 0.01), (0.0, 0, 1.0, 0.0)):
        got = run(base, u, *args)
        assert got[0] == got[1] == -1 and got[2] == 123
        # rows whose weights are all 1 or 0: sums and borders are exact on both sides
        exact = [5, 7, 8] if args[2] == 1.0 else [5]
        for b in exact:
            assert got[b] == sample_f64(base[b].double().numpy(), float(u[b]), *args)[0], b
        rest = [b for b in range(9) if b not in (5, 7, 8)]
        assert check(base[rest], u[rest], *args, got[rest]) == 0
        check(base, u, *args, got)
    # numbers outside [0, 1) take the nearest token
    z = torch.zeros(3, V)
    assert run(z, torch.tensor([-1.0, 1.0, 2.0])).tolist() == [0, V - 1, V - 1]


@pytest.mark.gpu
@pytest.mark.parametrize("V", [40, 3000, 20000, 60000])
def test_sample_more_asked_for_than_there_are_numbers(V):
    """top-k above the number of logits that are numbers: NaN counts as -inf,
    so the others stay, all of them."""
    z, u = rows(4, V, torch.float32, V)
    keep = torch.rand(4, V, generator=torch.Generator().manual_seed(V)) < 0.2
    keep[:, 7] = True
    z[~keep] = float("nan")
    for args in ((1.0, V // 2, 1.0, 0.0), (0.8, V // 2, 0.9, 0.0), (1.0, V - 1, 0.95, 0.01), (1.0, 0, 0.9, 0.0)):
        # (how many rows lie too close to a border depends on the rows and settings alone)
        print(args, check(z, u, *args, run(z, u, *args)), "undecided", flush=True)
    assert torch.equal(run(z, u, 1.0, V // 2), run(z, u))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 300, 20000, 60000])
def test_sample_top_p_of_nothing_and_less_keeps_the_first(V, dtype):
    """A top_p at or below 0, for every row or for some of them, leaves the
    largest logit alone; one that is no number leaves all."""
    z, u = rows(6, V, dtype, V + 1)
    first = torch.from_numpy(np.array([np.argmax(r) for r in z.double().numpy()]))
    each = torch.tensor([-0.5, 0.9, 0.0, -1.0, -float("inf"), float("nan")])
    for k in (0, 1, 40, V):
        for m in (0.0, 0.05):
            for p in (0.0, -1e-30, -0.5, -1.0, -3.0, -float("inf")):
                assert torch.equal(run(z, u, 0.8, k, p, m), first), (k, m, p)
            got = run(z, u, 0.8, k, each, m)
            assert torch.equal(got[[0, 2, 3, 4]], first[[0, 2, 3, 4]]), (k, m)
            assert torch.equal(got[[1]], run(z, u, 0.8, k, 0.9, m)[[1]])
            assert torch.equal(got[[5]], run(z, u, 0.8, k, 1.0, m)[[5]])
            check(z[:5], u[:5], 0.8, k, each[:5], m, got[:5])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sample_masks_of_the_lowest_value_at_any_temperature(dtype):
    """Logits masked with the type's lowest value have no weight, at
    temperatures where their distance passes float32, too."""
    V = 2000
    z, u = rows(3, V, dtype, 5)
    z[:, ::3] = torch.finfo(dtype).min
    for T in (1.0, 1e-3, 1e-10, 3e-30, 1e-38):
        for k, p, m in ((0, 1.0, 0.0), (300, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.02)):
            got = run(z, u, T, k, p, m)
            print(T, k, p, m, check(z, u, T, k, p, m, got), "undecided", flush=True)
            if T < 1e-6:
                assert torch.equal(z.gather(1, got[:, None])[:, 0], z.amax(-1))


@pytest.mark.gpu
def test_sample_strides_streams_and_graph():
    from src.model import kernels
    z, u = rows(4, 5000, torch.bfloat16, 3)
    want = run(z, u, 0.9, 50, 0.95, 0.0)
    wide = torch.zeros(4, 5003, dtype=torch.bfloat16)
    wide[:, 1:5001] = z
    got = kernels.sample(wide.cuda()[:, 1:5001], u.cuda(), 0.9, 50, 0.95)
    assert torch.equal(got.cpu(), want)
    assert torch.equal(kernels.sample(z.t().contiguous().cuda().t(), u.cuda(), 0.9, 50, 0.95).cpu(), want)
    s = torch.cuda.Stream()
    zc, uc = z.cuda(), u.cuda()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = kernels.sample(zc, uc, 0.9, 50, 0.95)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got.cpu(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kernels.sample(zc, uc, 0.9, 50, 0.95)
    for i in range(4):
        zn, un = rows(4, 5000, torch.bfloat16, 10 + i)
        zc.copy_(zn)
        uc.copy_(un)
        want = kernels.sample(zc, uc, 0.9, 50, 0.95)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_sample_refuses_the_cpu():
    from src.model import kernels
    with pytest.raises(RuntimeError, match="GPU"):
        kernels.sample(torch.zeros(1, 4), torch.zeros(1))


@pytest.mark.gpu
def test_sample_refusals():
    from src.model import _hip, kernels
    z, u = torch.zeros(2, 8, device="cuda"), torch.zeros(2, device="cuda")
    with pytest.raises(AssertionError):
        kernels.sample(z, u[:1])
    with pytest.raises(TypeError, match="u is float32"):
        kernels.sample(z, u.double())
    with pytest.raises(TypeError, match="top_k"):
        kernels.sample(z, u, top_k=u)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        kernels.sample(z.half(), u)
    with pytest.raises(ValueError, match="min_p"):
        kernels.sample(z, u, min_p=1.5)
    with pytest.raises(RuntimeError, match="tensors on"):
        kernels.sample(z, u.cpu())
    with pytest.raises(_hip.WalshHipError, match="V="):
        kernels.sample(z[:, :0], u)
    with pytest.raises(_hip.WalshHipError, match="V="):
        kernels.sample(torch.zeros(2, 1 << 20, device="cuda"), u)
    # the most that are taken: equal ones, whose sum stays within 64 bits
    assert kernels.sample(torch.zeros(1, (1 << 20) - 1, device="cuda"), u[:1] + 0.5).item() == ((1 << 20) - 1) // 2
    assert kernels.sample(z[:0], u[:0]).shape == (0,)
