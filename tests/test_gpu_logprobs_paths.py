"""Token probabilities at the sizes that take a kernel of their own: logits and
gradients that are streamed, rows of more steps than are told apart, many long
rows; sampled rows against the float64 oracle, with test_gpu_logprobs's bounds."""
import pytest
import torch

from oracle import tokens as otok
from test_gpu_logprobs import check, close, grad_bound

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
INF = float("inf")
SIZE = {F32: 4, BF16: 2}
MiB = 1 << 20


def many(N, V, dtype, seed):
    """Logits and tokens on the device, some rows masked in half, some not counted."""
    g = torch.Generator("cuda").manual_seed(seed)
    z = torch.empty(N, V, device="cuda", dtype=dtype).normal_(0, 3, generator=g)
    t = torch.randint(V, (N,), device="cuda", generator=g)
    z[1::7, : V // 2] = -INF
    t[3::11] = -1
    return z, t


def sample_of(N):
    return sorted({0, 1, 2, 3, 8, N // 2, N // 2 + 1, N - 2, N - 1})


@pytest.mark.parametrize("n", [0, 20])
@pytest.mark.parametrize("dtype,N,V", [(BF16, 2700, 50257), (F32, 1401, 50257), (BF16, 14001, 9999)])
def test_streamed_forward(dtype, N, V, n):
    from src.model import kernels
    assert N * V * SIZE[dtype] > 256 * MiB
    z, t = many(N, V, dtype, N + n)
    got = kernels.token_logprobs(z, t, n)
    at = sample_of(N)
    check(z[at].cpu(), t[at].cpu(), n, [x[at] for x in got], V)
    # every row as the kernel that keeps what the gradient reads
    held = kernels.token_logprobs(z, t, n, need_stats=True)
    assert all(torch.equal(a, b) for a, b in zip(got, held))


@pytest.mark.parametrize("n", [0, 20])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("least,most", [(0, 128), (128, 256), (256, 400)])
def test_gradients_of_every_size(dtype, least, most, n):
    """The gradient with alternatives where neither side, one or both are streamed."""
    from src.model import kernels
    V = 32003
    N = (least + 40) * MiB // (V * SIZE[dtype])
    assert least * MiB < N * V * SIZE[dtype] < most * MiB
    z, t = many(N, V, dtype, N + n)
    r = kernels.token_logprobs(z, t, n, need_stats=True)
    g = torch.Generator("cuda").manual_seed(n)
    gs = [torch.randn(N, device="cuda", generator=g), torch.randn(N, device="cuda", generator=g),
          torch.randn(N, n, device="cuda", generator=g) if n else None]
    d = kernels.token_logprobs_bwd(z, t, r[3], r[4], *gs)
    at = sample_of(N)
    nums = [None if v is None else v[at].double().cpu().numpy() for v in gs]
    zs, ts, index = z[at].cpu(), t[at].cpu().numpy(), r[3][at].cpu().numpy()
    check(zs, t[at].cpu(), n, [x[at] for x in r[:4]], V)
    want = otok.token_logprobs_grad_f64(zs.double().numpy(), ts, index, *nums)
    close(d[at], want, grad_bound(zs, ts, index, nums, want, dtype, V), "gradient")
    assert not d[3::11].any()


@pytest.mark.parametrize("dtype,N,V", [(BF16, 300, 140003), (F32, 300, 140003), (BF16, 1, 600011), (F32, 1, 600011)])
def test_rows_of_many_steps(dtype, N, V):
    """The largest logits in the steps behind those that are told apart, and in
    steps that share their place with an earlier one."""
    from src.model import kernels
    z, t = many(N, V, dtype, V)
    wide = 8192 if N > 256 else 32768          # tokens of a step
    assert V > 16 * wide
    for i, r in enumerate((0, 2, N // 2, N - 2, N - 1) if N > 2 else (0,)):
        z[r, 16 * wide + 5:16 * wide + 40:3] = 17.0 + i
        z[r, 9 + i * wide // 2] = 30.0
        z[r, -3:] = 18.5
        z[r, :200] -= 20
        t[r] = 16 * wide + 5
    for n in (1, 12, 40):
        got = kernels.token_logprobs(z, t, n)
        at = [r for r in (0, 1, 2, N // 2, N - 2, N - 1) if 0 <= r < N]
        check(z[at].cpu(), t[at].cpu(), n, [x[at] for x in got], V)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_long_rows(dtype):
    """Four wavefronts to a row of more than 8,192 tokens."""
    from src.model import kernels
    z, t = many(300, 20011, dtype, 5)
    z[4] = 0.5
    z[5, 3:] = -INF
    z[6, ::2] = torch.finfo(dtype).min
    for n in (0, 7, 64):
        got = kernels.token_logprobs(z, t, n, need_stats=True)
        at = [0, 1, 2, 3, 4, 5, 6, 150, 298, 299]
        check(z[at].cpu(), t[at].cpu(), n, [x[at] for x in got[:4]], 20011)
