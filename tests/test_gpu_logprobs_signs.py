"""What no rounding may make of a row of logits: a log probability above 0, an
entropy below, a weight above 1; on rows that are sure of a token.  Values are
held to test_gpu_logprobs's bounds."""
import pytest
import torch

from test_gpu_logprobs import check

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
INF = float("inf")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N,V", [(4000, 40), (2000, 3000), (200, 20011)])
def test_sure_rows_have_no_probability_above_one(N, V, dtype):
    """Rows that are sure of a token: no rounding makes its log probability
    positive, or the entropy negative, nor its weight in the gradient above 1."""
    from src.model import kernels, token_logprobs
    from src.model.tokens import token_logprobs_plain
    g = torch.Generator().manual_seed(V)
    z = torch.randn(N, V, generator=g)
    best = torch.randint(V, (N,), generator=g)
    z[torch.arange(N), best] = 30 + 900 * torch.rand(N, generator=g)
    z[::3] -= 700
    z[1::4] = torch.where(torch.arange(V) == best[1::4, None], z[1::4], torch.tensor(-INF))
    z, best = z.to(dtype).cuda(), best.cuda()
    for n in (0, min(5, V)):
        for r in (kernels.token_logprobs(z, best, n), token_logprobs_plain(z, best, n)):
            assert r[0].max() <= 0 and r[1].min() >= 0 and (n == 0 or r[2].max() <= 0)
        check(z.cpu(), best.cpu(), n, kernels.token_logprobs(z, best, n), V)
    x = z.requires_grad_(True)
    d, = torch.autograd.grad(token_logprobs(x, best).logprob.sum(), x)
    # 1 - p of the token, and -p of the others
    assert d.gather(-1, best[:, None]).min() >= 0
