"""Scores of texts against what stands before each token: later tokens,
padding and the padded width reach none of them, whatever the layers."""
import pytest
import torch

pytestmark = pytest.mark.gpu
MODELS = ["Walsh", "mHCWalsh"]
LAYERS = [dict(), dict(use_moe=True), dict(use_channel_mod=True), dict(algebra="octonion"),
          dict(attn_window=8, attn_sinks=2)]


def model(kind, **kw):
    import src.model as S
    torch.manual_seed(0)
    cfg = S.WalshConfig(**{**dict(block_size=64, vocab_size=97, n_layer=2, n_head=8, n_embd=128, algebra="hadamard"), **kw})
    m = getattr(S, kind)(cfg).cuda().eval()
    with torch.no_grad():
        for name, p in m.named_parameters():
            if "context_mlp" in name:        # (initial weights move a row by a thousandth alone)
                p.mul_(20)
    return m


def texts(B, T, seed=1):
    return torch.randint(97, (B, T), generator=torch.Generator().manual_seed(seed)).cuda()


# Two forwards of one text at two widths differ by the float32 rounding of two
# layers and a softmax: some hundred roundings of 2^-24 of numbers up to 10.
ROUNDED = 1e-4


@pytest.mark.parametrize("kw", LAYERS)
@pytest.mark.parametrize("kind", MODELS)
def test_later_tokens_reach_no_score(kind, kw):
    m, a = model(kind, **kw), texts(2, 13)
    b = a.clone()
    b[:, 8:] = (b[:, 8:] + 1 + texts(2, 5, 2) % 90) % 97
    with torch.no_grad():
        ra, rb = m.score(a, top_n=3), m.score(b, top_n=3)
    # (the distribution at k is that behind k + 1 tokens)
    assert (ra.logprob - rb.logprob)[:, :7].abs().max() <= ROUNDED
    assert (ra.entropy - rb.entropy)[:, :8].abs().max() <= ROUNDED
    assert (ra.top_logprob - rb.top_logprob)[:, :8].abs().max() <= ROUNDED
    assert (ra.logprob - rb.logprob)[:, 7:].abs().max() > 1e-2


@pytest.mark.parametrize("kw", LAYERS)
@pytest.mark.parametrize("kind", MODELS)
def test_padding_reaches_no_score(kind, kw):
    """Each text of a padded batch, its padding of any number, as alone."""
    m = model(kind, **kw)
    idx, lengths = texts(4, 17), [9, 17, 1, 2]
    for i, n in enumerate(lengths):
        idx[i, n:] = (-7, 0, 10 ** 12, 96)[i]
    with torch.no_grad():
        r = m.score(idx, lengths, 3)
        wide = m.score(torch.cat([idx, idx.new_full((4, 4), -1)], 1), torch.tensor(lengths, device="cuda"), 3)
        for i, n in enumerate(lengths):
            for got in (r, wide):
                assert not got.logprob[i, n - 1:].any() and not got.entropy[i, n - 1:].any()
                assert got.top_index[i, n - 1:].eq(-1).all()
            if n < 2:
                continue
            alone = m.score(idx[i:i + 1, :n], top_n=3)
            for got in (r, wide):
                assert (got.logprob[i, :n - 1] - alone.logprob[0]).abs().max() <= ROUNDED
                assert (got.entropy[i, :n - 1] - alone.entropy[0]).abs().max() <= ROUNDED
                assert (got.top_logprob[i, :n - 1] - alone.top_logprob[0]).abs().max() <= ROUNDED


@pytest.mark.parametrize("kw", LAYERS)
def test_scores_are_those_of_the_generated(kw):
    """What generate without a cache says of its tokens, score says of the text."""
    m = model("mHCWalsh", **kw)
    torch.manual_seed(3)
    out, r = m.generate(texts(2, 5), 6, logprobs=2)
    with torch.no_grad():
        s = m.score(out, top_n=2)
    assert (r.logprob - s.logprob[:, 4:]).abs().max() <= ROUNDED
    assert (r.entropy - s.entropy[:, 4:]).abs().max() <= ROUNDED


def test_gradients_of_scores_with_channel_modulation():
    """The scores' gradient against a difference of the scores, along a step of
    the output weights and the norms (what is not quantised)."""
    m, idx = model("mHCWalsh", use_channel_mod=True), texts(2, 7)
    loss = lambda: m.score(idx, [7, 4]).logprob.sum()  # noqa: E731
    p = [m.norm.weight, m.layers[0].channel_mod_norm.weight]
    g = torch.autograd.grad(loss(), p)
    step = [torch.randn(q.shape, generator=torch.Generator().manual_seed(i)).cuda() for i, q in enumerate(p)]
    want = sum((a * b).sum().double() for a, b in zip(g, step))
    h = 2.0 ** -9
    with torch.no_grad():
        ends = []
        for s in (h, -2 * h):
            for q, d in zip(p, step):
                q.add_(s * d)
            ends.append(loss().double())
    # nine scores, each off by ROUNDED, over the step; and the third derivative's share
    assert abs((ends[0] - ends[1]) / (2 * h) - want) <= 9 * ROUNDED / (2 * h) + 1e-2 * want.abs()
