"""Scaled rows and dropout in a model beside what else a model may have:
channel modulation, hooks and layers of its own, weights of an earlier time."""
import pytest
import torch

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
