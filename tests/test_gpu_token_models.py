"""Models with a scaled embedding, dropout of tokens' rows and of layers'
outputs, token scores and generated tokens' probabilities: the operators
together, as a training step and a generation use them."""
import numpy as np
import pytest
import torch

from oracle import tokens as otok

pytestmark = pytest.mark.gpu
MODELS = ["Walsh", "mHCWalsh"]


def model(kind, dtype=torch.float32, **kw):
    import src.model as S
    torch.manual_seed(0)
    cfg = S.WalshConfig(block_size=64, vocab_size=97, n_layer=2, n_head=4, n_embd=64, algebra="hadamard", **kw)
    return getattr(S, kind)(cfg).cuda().to(dtype)


def texts(B=3, T=17, seed=1):
    return torch.randint(97, (B, T), generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("kind", MODELS)
def test_defaults_are_the_reference_path(kind, monkeypatch):
    """Without the new fields no new operator runs and no random number is drawn."""
    from src.model import tokens
    m = model(kind).train()

    def never(*a, **k):
        raise AssertionError("called")
    monkeypatch.setattr(tokens, "token_embedding", never)
    monkeypatch.setattr(tokens, "counter_dropout", never)
    monkeypatch.setattr(tokens, "fresh_seed", never)
    idx = texts()
    m(idx, idx)[1].backward()
    state = torch.cuda.get_rng_state()
    m(idx, idx)
    assert torch.equal(torch.cuda.get_rng_state(), state)


@pytest.mark.parametrize("kind", MODELS)
def test_scale_is_a_scaled_embedding(kind):
    """A factor of 8 is the model whose rows are 8 times as large (a power of
    two: the same numbers)."""
    a, b = model(kind, embed_scale=8.0).eval(), model(kind).eval()
    idx = texts()
    with torch.no_grad():
        b.tok_embeddings.weight = torch.nn.Parameter(b.tok_embeddings.weight * 8)
        ha, hb = a(idx, return_hidden=True)[2], b(idx, return_hidden=True)[2]
    assert torch.equal(ha, hb)


@pytest.mark.parametrize("kind", MODELS)
def test_training_with_dropout_repeats(kind):
    """The same generator state gives the same loss and gradients, another one
    others; evaluation drops nothing; checkpointed layers compute their masks
    again."""
    m = model(kind, embed_scale=2.0, embed_dropout=0.1, resid_dropout=0.2).train()
    idx, tgt = texts(), texts(seed=2)

    def step(seed):
        torch.manual_seed(seed)
        m.zero_grad(set_to_none=True)
        loss = m(idx, tgt)[1]
        loss.backward()
        return loss.detach(), [p.grad.clone() for p in m.parameters() if p.grad is not None]
    (l0, g0), (l1, g1), (l2, _) = step(5), step(5), step(6)
    assert torch.equal(l0, l1) and l0 != l2 and len(g0) == len(g1) > 5
    assert all(torch.equal(x, y) for x, y in zip(g0, g1))
    if kind == "mHCWalsh":
        m.gradient_checkpointing = True
        l3, g3 = step(5)
        assert torch.equal(l0, l3) and all(torch.allclose(x, y, rtol=1e-4, atol=1e-5) for x, y in zip(g0, g3))
    m.eval()
    with torch.no_grad():
        assert torch.equal(m(idx, tgt)[1], m(idx, tgt)[1])


@pytest.mark.parametrize("kind", MODELS)
def test_training_agrees_with_the_torch_forms(kind, monkeypatch):
    """Loss and gradients of a step through lookup, dropout and token
    probabilities, kernels against torch's operations on the same seeds: equal
    up to the float32 rounding of a network this size."""
    from src.model import tokens
    m = model(kind, embed_scale=2.0, embed_dropout=0.1, resid_dropout=0.2).train()
    idx, lengths = texts(), [17, 9, 12]

    def step():
        torch.manual_seed(3)
        m.zero_grad(set_to_none=True)
        r = m.score(idx, lengths, 4)
        (-r.logprob.sum() / 35 - 0.01 * r.entropy.sum() + 0.1 * r.top_logprob[:, :8].mean()).backward()
        return r, [p.grad.clone() for p in m.parameters() if p.grad is not None]
    r0, g0 = step()
    monkeypatch.setattr(tokens, "_kernel_tensors", lambda *a: False)
    r1, g1 = step()
    assert torch.allclose(r0.logprob, r1.logprob, atol=1e-4) and torch.allclose(r0.entropy, r1.entropy, atol=1e-4)
    for x, y in zip(g0, g1):
        assert (x - y).norm() <= 1e-3 * y.norm() + 1e-6


@pytest.mark.parametrize("kw", [dict(), dict(use_moe=True), dict(use_channel_mod=True), dict(algebra="octonion"),
                                dict(attn_window=8, attn_sinks=2)])
@pytest.mark.parametrize("kind", MODELS)
def test_every_kind_of_layer_trains_with_dropout(kind, kw):
    """Under bf16 autocast: finite losses and gradients that the same generator
    state gives again."""
    import src.model as S
    torch.manual_seed(0)
    cfg = S.WalshConfig(**{**dict(block_size=64, vocab_size=97, n_layer=2, n_head=8, n_embd=128, algebra="hadamard",
                                  embed_dropout=0.1, resid_dropout=0.1, embed_scale=4.0), **kw})
    m = getattr(S, kind)(cfg).cuda().train()
    idx = texts(2, 24)

    def step():
        torch.manual_seed(4)
        m.zero_grad(set_to_none=True)
        with torch.autocast("cuda", torch.bfloat16):
            loss = m(idx, texts(2, 24, 2))[1] - m.score(idx).logprob.mean()
        loss.backward()
        return loss.detach(), [p.grad.clone() for p in m.parameters() if p.grad is not None]
    (l0, g0), (l1, g1) = step(), step()
    assert l0.isfinite() and torch.equal(l0, l1) and all(x.isfinite().all() for x in g0)
    # (atomics of torch's own operations aside)
    assert all((x - y).norm() <= 1e-2 * x.norm() + 1e-6 for x, y in zip(g0, g1))


@pytest.mark.parametrize("kind", MODELS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_score(kind, dtype):
    """Scores are the log probabilities of the model's own logits, padding
    counts nothing whatever it holds, and autocast works."""
    m = model(kind).eval()
    idx = texts()
    with torch.no_grad(), torch.autocast("cuda", torch.bfloat16, enabled=dtype == torch.bfloat16):
        logits = m.all_logits(idx[:, :-1])
        r = m.score(idx, top_n=3)
        assert r.logprob.shape == (3, 16) and r.top_index.shape == (3, 16, 3)
        want = otok.token_logprobs_f64(logits.flatten(0, 1).double().cpu().numpy(), idx[:, 1:].flatten().cpu().numpy(), 3)
        assert np.abs(r.logprob.flatten().double().cpu().numpy() - want[0]).max() < 1e-5
        assert np.array_equal(r.top_index.flatten(0, 1).cpu().numpy(), want[3])
        one, _ = m(idx[:, :5])
        assert torch.allclose(one[:, -1].float(), logits[:, 4].float(), rtol=0.05, atol=0.05)
        padded = idx.clone()
        padded[1, 9:] = -5
        padded[2, 12:] = 10 ** 9
        q = m.score(padded, torch.tensor([17, 9, 12], device="cuda"), 3)
        assert torch.equal(q.logprob[0], r.logprob[0]) and torch.equal(q.logprob[1, :8], r.logprob[1, :8])
        assert not q.logprob[1, 8:].any() and q.top_index[2, 11:].eq(-1).all() and not q.entropy[2, 11:].any()
    with pytest.raises(ValueError, match="two tokens"):
        m.score(idx[:, :1])
    with pytest.raises(ValueError, match="lengths"):
        m.score(idx, [3, 4])


def test_generate_with_probabilities():
    """The reference's loop, the filtered one and the cached one give the new
    tokens' log probabilities under the model itself."""
    from src.model import PagedKVCache
    m = model("mHCWalsh").eval()
    idx = texts(2, 6)
    cache = PagedKVCache(2, 8, 4, 16, 32, "cuda", dtype=torch.float32, batch=2, page_size=16)
    for kw in (dict(), dict(top_k=5), dict(top_p=0.9, temperature=0.7), dict(kv_cache=cache, min_p=0.02)):
        torch.manual_seed(9)
        out, r = m.generate(idx, 5, logprobs=2, **kw)
        torch.manual_seed(9)
        if "kv_cache" in kw:
            cache.reset()
        assert torch.equal(m.generate(idx, 5, **kw), out)
        assert r.logprob.shape == (2, 5) and r.top_index.shape == (2, 5, 2)
        with torch.no_grad():
            want = m.score(out, top_n=2)
        assert torch.allclose(r.logprob, want.logprob[:, 5:], atol=1e-3)
        assert torch.allclose(r.entropy, want.entropy[:, 5:], atol=1e-3)
        assert (r.logprob <= r.top_logprob[..., 0]).all()
    # padded prompts: the same probabilities as each prompt alone
    cache.reset()
    torch.manual_seed(9)
    padded = idx.clone()
    padded[1, 4:] = 0
    out, r = m.generate(padded, 3, temperature=0.0, top_p=0.9, kv_cache=cache, lengths=[6, 4], logprobs=2)
    cache.reset()
    with torch.no_grad():
        alone = m.score(torch.cat([padded[1:, :4], out[1:, 6:]], 1), top_n=2)
    assert torch.allclose(r.logprob[1], alone.logprob[0, 3:], atol=1e-3)
    out, r = m.generate(idx, 0, logprobs=3)
    assert torch.equal(out, idx) and r.top_logprob.shape == (2, 0, 3) and r.top_index.dtype == torch.int64
    for bad in (-1, 65):
        with pytest.raises(ValueError, match="logprobs"):
            m.generate(idx, 2, logprobs=bad)


def test_captured_training_step():
    """A step with dropout and token probabilities in one graph: each replay
    draws a seed of its own and matches an eager step on it."""
    from src.model import kernels, token_embedding, token_logprobs
    from src.model.tokens import counter_dropout, fresh_seed
    V, C = 300, 64
    g = torch.Generator().manual_seed(2)
    w = torch.randn(V, C, generator=g).cuda().requires_grad_(True)
    head = (0.1 * torch.randn(C, V, generator=g)).cuda()
    t, nxt = torch.randint(V, (40,), generator=g).cuda(), torch.randint(V, (40,), generator=g).cuda()

    def step(seed):
        h = token_embedding(t, w, 2.0, p=0.1, seed=seed)
        h = counter_dropout(h.tanh(), 0.2, seed, 1, h)
        r = token_logprobs(h @ head, nxt)
        return r.logprob, torch.autograd.grad(-r.logprob.mean() - 0.1 * r.entropy.mean(), w)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fresh_seed("cuda"))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        seed = fresh_seed("cuda")
        lp, d = step(seed)
    lp = lp.detach()
    seen = set()
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        seen.add(int(seed))
        elp, ed = step(seed.clone())
        assert torch.allclose(lp, elp, atol=1e-5) and torch.allclose(d, ed, rtol=1e-4, atol=1e-6)
        assert not kernels.token_logprobs(head, nxt.new_zeros(C))[0].isnan().any()
    assert len(seen) == 4
