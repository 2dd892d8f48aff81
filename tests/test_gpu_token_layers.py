"""Scaled rows and dropout in a model beside what else a model may have:
channel modulation, hooks and layers of its own, weights of an earlier time."""
import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu
MODELS = ["Walsh", "mHCWalsh"]


def model(kind, dtype=torch.float32, **kw):
    import src.model as S
    torch.manual_seed(0)
    cfg = S.WalshConfig(**{**dict(block_size=64, vocab_size=97, n_layer=2, n_head=4, n_embd=64, algebra="hadamard"), **kw})
    return getattr(S, kind)(cfg).cuda().to(dtype)


def texts(B=3, T=17, seed=1):
    return torch.randint(97, (B, T), generator=torch.Generator().manual_seed(seed)).cuda()


# ------------------------------------------------------------------ channel modulation

@pytest.mark.parametrize("grad", [True, False])
def test_everything_a_layer_adds_is_dropped(grad):
    """Of layers that drop all, channel modulation adds no more than the rest."""
    m = model("mHCWalsh", use_channel_mod=True, resid_dropout=1.0).train()
    idx = texts()
    with torch.set_grad_enabled(grad):
        a = m(idx, return_hidden=True)[2]
        for layer in m.layers:
            layer.use_channel_mod = False
        b = m(idx, return_hidden=True)[2]
    # (the streams' update is fused with what follows it in the one, not in the other)
    assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)


def test_channel_modulation_has_masks_of_its_own():
    """Its dropped rows are those of a stream number that no other output has,
    and evaluation drops none."""
    from src.model import tokens
    seen = []
    m = model("mHCWalsh", use_channel_mod=True, resid_dropout=0.25).train()
    drop, tokens.counter_dropout = tokens.counter_dropout, lambda y, p, s, n, r=None: (seen.append((p, n)), drop(y, p, s, n, r))[1]
    try:
        m(texts())
        assert len(seen) == 6 == len(set(seen)) and {p for p, _ in seen} == {0.25}
        # (attention and feed-forward keep the numbers that they have without it)
        assert {1, 2, 3, 4} < {n for _, n in seen}
        m.eval()
        with torch.no_grad():
            m(texts())
        assert len(seen) == 6
    finally:
        tokens.counter_dropout = drop


def test_training_with_channel_modulation_repeats():
    m, idx, tgt = model("mHCWalsh", use_channel_mod=True, resid_dropout=0.2).train(), texts(), texts(seed=2)

    def step(seed):
        torch.manual_seed(seed)
        m.zero_grad(set_to_none=True)
        loss = m(idx, tgt)[1]
        loss.backward()
        return loss.detach(), [p.grad.clone() for p in m.parameters() if p.grad is not None]
    (l0, g0), (l1, g1) = step(5), step(5)
    m.gradient_checkpointing = True
    l2, g2 = step(5)
    assert torch.equal(l0, l1) and torch.equal(l0, l2)
    for x, y, z in zip(g0, g1, g2):
        assert torch.allclose(x, y, rtol=1e-4, atol=1e-5) and torch.allclose(x, z, rtol=1e-4, atol=1e-5)


# ------------------------------------------------------------------ the embedding module

class Shifted(nn.Embedding):
    def forward(self, tokens):
        return super().forward(tokens) + 1.0


def changed(how, m):
    """Changes what the model's embedding gives; its rows then."""
    e, idx = m.tok_embeddings, texts()
    if how == "forward hook":
        e.register_forward_hook(lambda mod, args, out: out + 1.0)
    elif how == "pre-hook":
        e.register_forward_pre_hook(lambda mod, args: ((args[0] + 1) % 97,))
    elif how == "global hook":
        return nn.modules.module.register_module_forward_hook(
            lambda mod, args, out: out + 1.0 if isinstance(mod, nn.Embedding) else None)
    elif how == "subclass":
        m.tok_embeddings = Shifted(97, 64).cuda()
    elif how == "own forward":
        e.forward = lambda tokens: nn.functional.embedding(tokens, e.weight) + 1.0
    elif how == "max_norm":
        e.max_norm = 0.05
    return None


CHANGES = ["forward hook", "pre-hook", "global hook", "subclass", "own forward", "max_norm"]


@pytest.mark.parametrize("how", CHANGES)
@pytest.mark.parametrize("kind", MODELS)
def test_hooks_and_own_embeddings_are_run(kind, how):
    """A factor (a power of two) and dropout of everything apply to what the
    module gives, whatever it is: the same as rows that are that much larger."""
    a, b = model(kind, embed_scale=8.0).eval(), model(kind).eval()
    handles = [changed(how, m) for m in (a, b)]
    if how == "subclass":
        b.tok_embeddings.load_state_dict(a.tok_embeddings.state_dict())
    hook = b.tok_embeddings.register_forward_hook(lambda mod, args, out: out * 8)
    try:
        with torch.no_grad():
            if how == "global hook":
                [h.remove() for h in handles[1:]]         # (there are two, and each is called for both)
            ha, hb = a(texts(), return_hidden=True)[2], b(texts(), return_hidden=True)[2]
            plain = model(kind, embed_scale=8.0).eval()(texts(), return_hidden=True)[2] if how != "global hook" else None
        assert torch.equal(ha, hb)
        assert plain is None or not torch.allclose(ha, plain, atol=1e-3)
    finally:
        hook.remove()
        [h.remove() for h in handles if h is not None]


def test_gradients_and_dropout_through_a_hook():
    """A hook that changes nothing changes nothing: rows, masks and gradients."""
    got = []
    for hooked in (False, True):
        m = model("mHCWalsh", embed_scale=2.0, embed_dropout=0.25).train()
        calls = []
        if hooked:
            m.tok_embeddings.register_forward_hook(lambda *a: calls.append(1))
        torch.manual_seed(4)
        loss = m(texts(), texts(seed=2))[1]
        loss.backward()
        assert len(calls) == hooked
        got.append((loss.detach(), m.tok_embeddings.weight.grad.clone()))
    # (2 times 4 / 3 is one factor in the kernel, two here)
    assert torch.allclose(got[0][0], got[1][0], rtol=1e-5)
    assert (got[0][1] - got[1][1]).norm() <= 1e-4 * got[0][1].norm()


def test_padding_row_learns_nothing():
    """An embedding with a padding_idx keeps it with a factor."""
    m = model("mHCWalsh", embed_scale=2.0).train()
    m.tok_embeddings = nn.Embedding(97, 64, padding_idx=5).cuda()
    idx = texts()
    idx[:, ::3] = 5
    m(idx, texts(seed=2))[1].backward()
    g = m.tok_embeddings.weight.grad
    assert not g[5].any() and g[idx[0, 1]].any()


# ------------------------------------------------------------------ what a model is given

@pytest.mark.parametrize("kind", MODELS)
def test_tokens_of_32_bits(kind):
    """A model takes the tokens that its embedding takes, with a factor too."""
    for kw in (dict(), dict(embed_scale=2.0), dict(embed_scale=2.0, embed_dropout=0.5)):
        m = model(kind, **kw).eval()
        with torch.no_grad():
            a, b = m(texts())[0], m(texts().int())[0]
            assert torch.equal(a, b)
            assert torch.equal(m.score(texts()).logprob, m.score(texts().int()).logprob)
            assert torch.equal(m.score(texts(), [17, 4, 9]).logprob, m.score(texts().int(), [17, 4, 9]).logprob)


@pytest.mark.parametrize("field", ["embed_dropout", "resid_dropout"])
@pytest.mark.parametrize("p", [-0.1, 1.5, float("nan")])
@pytest.mark.parametrize("kind", MODELS)
def test_probabilities_that_are_none(kind, p, field):
    m = model(kind, **{field: p})
    with pytest.raises(ValueError, match="probability"):
        m.train()(texts(), texts())


@pytest.mark.parametrize("kind", MODELS)
def test_layers_of_an_earlier_time(kind):
    """Modules that were stored before there was a dropout of outputs."""
    m = model(kind).train()
    want = m(texts(), texts(seed=2))[1]
    for layer in m.layers:
        layer.__dict__.pop("resid_dropout", None)
    assert torch.equal(m(texts(), texts(seed=2))[1], want)


def test_no_new_tokens_have_float32_probabilities():
    m = model("mHCWalsh").eval()
    torch.set_default_dtype(torch.bfloat16)
    try:
        _, r = m.generate(texts(), 0, logprobs=2)
    finally:
        torch.set_default_dtype(torch.float32)
    assert all(x.dtype == torch.float32 for x in r[:3]) and r.top_index.dtype == torch.int64


@pytest.mark.parametrize("kind", MODELS)
def test_lengths_that_no_text_has(kind):
    """As generate's: whole numbers from 1 to the width, one a text, on either side."""
    m = model(kind).eval()
    for bad in ([17, 0, 3], [17, -1, 3], [18, 3, 3], [3, 4], [17.0, 3.0, 3.0], [[17, 3, 3]]):
        for lengths in (bad, torch.tensor(bad), torch.tensor(bad, device="cuda")):
            with pytest.raises((ValueError, TypeError), match="lengths"):
                m.score(texts(), lengths)
