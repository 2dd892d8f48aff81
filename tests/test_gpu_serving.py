"""The windowed attention, the paged cache and the sampling as a model uses
them, together: cached against uncached, windowed against a masked attention,
captured against eager.  Bars as of the other model tests: float32 within 1e-5
relative, bf16 against the float32 forward within max(1e-2, 1.25 x the uncached
bf16 forward's own distance)."""
import pytest
import torch
from torch.nn.attention import SDPBackend, sdpa_kernel

pytestmark = pytest.mark.gpu


def rel(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return float((a - b).norm() / b.norm().clamp_min(1e-30))


def make(C=512, n_layer=2, n_head=32, seed=0, cls="mHCWalsh", **kw):
    import src.model as M
    torch.manual_seed(seed)
    args = dict(block_size=64, vocab_size=1000, n_layer=n_layer, n_head=n_head, n_embd=C, algebra="hadamard",
                head_mixing=n_head % 32 == 0)
    args.update(kw)
    return getattr(M, cls)(M.WalshConfig(**args)).cuda().eval()


def tokens(B, T, seed=1):
    return torch.randint(0, 1000, (B, T), generator=torch.Generator().manual_seed(seed)).cuda()


def paged(model, batch, pages=64, dtype=torch.float32, page_size=16, max_seq_len=128):
    from src.model import PagedKVCache
    cfg = model.config
    return PagedKVCache(cfg.n_layer, pages, cfg.n_head, cfg.n_embd // cfg.n_head, max_seq_len, "cuda", dtype, batch,
                        page_size)


@pytest.mark.parametrize("cls,kw", [("mHCWalsh", dict(attn_window=16, attn_sinks=2)), ("mHCWalsh", dict(attn_window=24)),
                                    ("Walsh", dict(attn_window=16, attn_sinks=3, use_moe=True)),
                                    ("mHCWalsh", dict(C=256, n_head=8, algebra="octonion", attn_window=9, attn_sinks=1))])
def test_windowed_model_against_masked_attention(cls, kw, monkeypatch):
    """Logits and gradients with the window on the kernels equal those with
    the mask given to torch's attention (float32)."""
    from src.model import kernels
    model = make(cls=cls, **kw)
    idx, tgt = tokens(2, 60), tokens(2, 60, 2)

    def step():
        model.train()
        model.zero_grad()
        with sdpa_kernel(SDPBackend.MATH):      # float32 products throughout
            logits, loss = model(idx, targets=tgt)
            loss.backward()
        model.eval()
        return [logits.detach()] + [p.grad.clone() for p in model.parameters() if p.grad is not None]
    own = step()
    monkeypatch.setattr(kernels, "window_attention_supported", lambda q: False)
    ref = step()
    # gradients that all but cancel (the stream mappings': their inputs are
    # equal streams at the start) hold little but rounding: they are left out
    most = max(g.norm() for g in ref[1:])
    full = [rel(a, b) for a, b in zip(own, ref) if b.norm() > 1e-3 * most]
    print(f"{cls} {kw}: logits {full[0]:.2e}, worst of {len(full) - 1} gradients {max(full[1:]):.2e}")
    # the octonion layers compute with bf16 operands whatever the model's type:
    # a difference of one float32 step may move a rounding, as in a bf16 model
    own_bf16 = kw.get("algebra") == "octonion"
    assert full[0] <= (1e-2 if own_bf16 else 1e-5) and max(full[1:]) <= (2e-2 if own_bf16 else 1e-4)
    monkeypatch.undo()
    model.layers[0].attention.window = 0
    assert rel(step()[0], ref[0]) > 1e-3    # the window matters at this length


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kw", [dict(), dict(attn_window=16, attn_sinks=2), dict(attn_window=8, attn_sinks=0)])
def test_dense_cache_decode_matches_uncached(kw, dtype):
    from src.model import KVCache
    model = make(**kw)
    B, T0, steps = 3, 30, 6
    idx = tokens(B, T0 + steps)
    kv = KVCache(2, 64, 32, 16, torch.device("cuda"), dtype=dtype, batch=B)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16, enabled=dtype == torch.bfloat16):
        for a, e in [(0, 20), (20, T0)] + [(T0 + s, T0 + s + 1) for s in range(steps)]:
            lg, _ = model(idx[:, a:e], kv_cache=kv, start_pos=a)
            kv.increment(e - a)
            compare(model, idx[:, :e], lg, dtype, f"{kw} to {e}")


def compare(model, idx, got, dtype, what):
    ref, _ = model(idx)
    if dtype == torch.float32:
        r = rel(got, ref)
        print(f"{what}: {r:.2e}")
        assert r <= (1e-2 if model.config.algebra == "octonion" else 1e-5)   # octonion layers: bf16 operands
        return
    with torch.autocast("cuda", enabled=False):
        ref32, _ = model(idx)
    own, unc = rel(got, ref32), rel(ref, ref32)
    print(f"{what}: cached {own:.2e}, uncached {unc:.2e} from float32")
    assert own <= max(1e-2, 1.25 * unc)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kw", [dict(), dict(attn_window=16, attn_sinks=2), dict(C=256, n_head=8, use_moe=True),
                                dict(C=256, n_head=8, algebra="octonion", attn_window=20, attn_sinks=1),
                                dict(cls="Walsh", attn_window=8)])
def test_paged_cache_matches_uncached_sequences(kw, dtype):
    """Prompts of unequal lengths, padded, then one token at a time; one
    sequence ends and its pages go to another; every step's logits equal the
    uncached forward of that sequence alone."""
    model = make(**kw)
    B, T0 = 3, 30
    lens = [30, 7, 18]
    idx = tokens(B, 60)
    kv = paged(model, B, pages=8, dtype=dtype, max_seq_len=60)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16, enabled=dtype == torch.bfloat16):
        kv.reserve(lens)
        lg, _ = model(idx[:, :T0], kv_cache=kv)
        kv.increment()
        at = list(lens)
        seqs = [idx[b:b + 1] for b in range(B)]
        for s in range(8):
            for b in range(B):
                if at[b]:
                    compare(model, seqs[b][:, :at[b]], lg[b:b + 1], dtype, f"{kw} step {s} row {b}")
            if s == 3:
                kv.release(1)
                at[1] = 0
                seqs[1] = tokens(1, 60, 5)
            take = [1, 0 if s == 5 else 1, 1]
            kv.reserve(take)
            lg, _ = model(torch.cat([q[:, n:n + 1] for q, n in zip(seqs, at)]), kv_cache=kv)
            kv.increment()
            lg = lg.clone()
            at = [n + c for n, c in zip(at, take)]
            if s == 5:
                lg[1] = model(seqs[1][:, :at[1]])[0]      # took no token: nothing to compare
    assert kv.seq_lens == at


@pytest.mark.parametrize("kw", [dict(), dict(attn_window=16, attn_sinks=2)])
def test_prompts_in_parts(kw):
    """A second part of several tokens behind cached ones, of two of three
    sequences."""
    model = make(**kw)
    idx = tokens(3, 50)
    kv = paged(model, 3)
    with torch.no_grad():
        kv.reserve([20, 20, 5])
        model(idx[:, :20], kv_cache=kv)
        kv.increment()
        kv.reserve([30, 11, 0])
        lg, _ = model(idx[:, 20:50], kv_cache=kv)
        kv.increment()
        for b, n in ((0, 50), (1, 31)):
            compare(model, idx[b:b + 1, :n], lg[b:b + 1], torch.float32, f"{kw} part two, row {b}")
        kv.reserve([0, 0, 1])
        lg, _ = model(idx[:, 5:6], kv_cache=kv)
        kv.increment()
        compare(model, idx[2:, :6], lg[2:], torch.float32, f"{kw} row 2")


def test_generate_with_the_paged_cache():
    """The largest logit each time: the same tokens as without a cache, for
    prompts alone and padded together; and drawn ones from the same random
    numbers as the sampling called by hand."""
    from src.model import kernels
    model = make(attn_window=16, attn_sinks=2)
    idx = tokens(3, 20)
    want = idx.clone()
    with torch.no_grad():
        for _ in range(12):
            want = torch.cat([want, model(want)[0][:, -1].argmax(-1, keepdim=True)], 1)
    got = model.generate(idx, 12, temperature=0.0, kv_cache=paged(model, 3))
    assert torch.equal(got, want)
    lens = [20, 4, 11]
    got = model.generate(idx, 6, temperature=0.0, kv_cache=paged(model, 3), lengths=lens)
    for b, n in enumerate(lens):
        w = idx[b:b + 1, :n]
        with torch.no_grad():
            for _ in range(6):
                w = torch.cat([w, model(w)[0][:, -1].argmax(-1, keepdim=True)], 1)
        assert torch.equal(got[b, 20:], w[0, n:]), b
    settings = dict(temperature=0.9, top_k=50, top_p=0.9, min_p=0.01)
    torch.manual_seed(3)
    got = model.generate(idx, 5, kv_cache=paged(model, 3), **settings)
    torch.manual_seed(3)
    w = idx
    with torch.no_grad():
        for _ in range(5):
            t = kernels.sample(model(w)[0][:, -1], torch.rand(3, device="cuda"), **settings)
            w = torch.cat([w, t[:, None]], 1)
    assert torch.equal(got, w)
    torch.manual_seed(3)
    assert torch.equal(model.generate(idx, 5, **settings), w)


def test_generate_without_new_arguments_is_the_old_loop():
    model = make()
    idx = tokens(2, 10)
    torch.manual_seed(5)
    got = model.generate(idx, 4, temperature=0.8, top_k=20)
    torch.manual_seed(5)
    with torch.no_grad():
        for _ in range(4):
            z = model(idx)[0][:, -1].float() / 0.8
            z[z < torch.topk(z, 20)[0][:, [-1]]] = -float("inf")
            idx = torch.cat([idx, torch.multinomial(torch.softmax(z, -1), 1)], 1)
    assert torch.equal(got, idx)


def test_captured_decode_step_with_sampling():
    """Model, cache and sampling of one token captured once and replayed as
    the sequences grow, with eager work in between, against eager steps."""
    from src.model import kernels
    model = make(attn_window=24, attn_sinks=2)
    B, lens, steps = 3, [20, 3, 11], 10
    idx = tokens(B, 20)
    g = torch.Generator().manual_seed(0)
    us = torch.rand(steps, B, generator=g).cuda()
    runs = []
    for captured in (False, True):
        kv = paged(model, B, dtype=torch.bfloat16)
        u, tok = us[0].clone(), torch.zeros(B, 1, dtype=torch.int64, device="cuda")

        def step():
            with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
                lg, _ = model(tok, kv_cache=kv)
            return kernels.sample(lg[:, -1], u, 0.9, 100, 0.95)
        with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
            kv.reserve(lens)
            lg, _ = model(idx, kv_cache=kv)
            kv.increment()
        tok.copy_(lg[:, -1].argmax(-1, keepdim=True))
        graph, out = None, []
        for s in range(steps):
            u.copy_(us[s])
            kv.reserve(1)
            if captured and graph is None:
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    step()
                torch.cuda.current_stream().wait_stream(side)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    new = step()
            if captured:
                graph.replay()
                torch.randn(256, 256, device="cuda").sum().item()
            else:
                new = step()
            kv.increment()
            tok.copy_(new[:, None])
            out.append(new.clone())
        runs.append(torch.stack(out))
    assert torch.equal(*runs)


def test_paged_cache_refusals_in_a_model():
    model = make()
    idx = tokens(2, 5)
    kv = paged(model, 2)
    with torch.no_grad():
        with pytest.raises(RuntimeError, match="reserved"):
            model(idx, kv_cache=kv)
        kv.reserve([5, 5])
        with pytest.raises(AssertionError, match="2 sequences"):
            model(idx[:1], kv_cache=kv)
        with pytest.raises(ValueError, match="rotary"):
            model(idx, kv_cache=paged(model, 2, max_seq_len=1000))
        kv.reset()
        with pytest.raises(ValueError, match="lengths"):
            model.generate(idx, 2, kv_cache=kv, lengths=[6, 1])
        with pytest.raises(ValueError, match="kv_cache"):
            model.generate(idx, 2, lengths=[5, 1])
        with pytest.raises(ValueError, match="positions"):
            model.generate(idx, 125, kv_cache=kv)
        kv.reserve(1)
        kv.increment()
        with pytest.raises(ValueError, match="not empty"):
            model.generate(idx, 2, kv_cache=kv)
    kv.reset()
    kv.reserve(5)
    with pytest.raises(RuntimeError, match="no_grad"):
        model(idx, kv_cache=kv)


def test_generate_survives_logits_that_are_no_numbers():
    """Such rows have no token; what follows them is some token of the
    vocabulary."""
    model = make()
    with torch.no_grad():
        model.output.weight[999] = float("nan")
        model.invalidate_weight_caches()
        bad = tokens(2, 6)
        bad[1, :] = 999
        got = model.generate(bad, 4, temperature=0.0, top_p=1.0)
    assert int(got.min()) >= 0 and int(got.max()) < 1000


def test_generate_takes_lengths_as_a_tensor_and_no_other_cache():
    model = make(n_layer=1)
    idx = tokens(2, 6)
    want = model.generate(idx, 3, temperature=0.0, kv_cache=paged(model, 2), lengths=[6, 2])
    got = model.generate(idx, 3, temperature=0.0, kv_cache=paged(model, 2), lengths=torch.tensor([6, 2]))
    assert torch.equal(got, want)
    with pytest.raises(TypeError, match="PagedKVCache"):
        model.generate(idx, 3, kv_cache=object())


def test_windowed_single_token_keeps_the_gradients_of_its_keys(monkeypatch):
    """Keys and values that are trained while the queries are frozen: a single
    token over a dense cache gives them their gradients."""
    from src.model import KVCache, kernels
    layer = make(C=256, n_head=8, attn_window=8, attn_sinks=1).layers[0].attention
    for p in layer.wq.parameters():
        p.requires_grad_(False)
    g = torch.Generator().manual_seed(4)
    x = torch.randn(2, 13, 256, generator=g).cuda()
    # rotary angle 0 throughout: cos 1, sin 0
    freqs = torch.polar(torch.ones(13, 16), torch.zeros(13, 16)).cuda()

    def step():
        kv = KVCache(1, 64, 8, 32, torch.device("cuda"), dtype=torch.float32, batch=2)
        with torch.no_grad():
            layer(x[:, :12], freqs[:12], kv)
            kv.increment(12)
        layer.zero_grad()
        layer(x[:, 12:], freqs[12:], kv).square().sum().backward()
        return {n: p.grad for n, p in layer.named_parameters() if n.startswith(("wk", "wv")) and p.grad is not None}
    own = step()
    monkeypatch.setattr(kernels, "window_attention_supported", lambda q: False)
    with sdpa_kernel(SDPBackend.MATH):
        ref = step()
    assert ref and own.keys() == ref.keys()
    for n in ref:
        print(n, rel(own[n], ref[n]), flush=True)
        assert rel(own[n], ref[n]) <= 1e-4 or ref[n].norm() < 1e-6


@pytest.mark.parametrize("kw", [dict(), dict(attn_window=16, attn_sinks=2)])
def test_padding_past_the_rotary_table(kw):
    """Parts and prompts padded past the model's 128 rotary positions, whose
    tokens that count lie within them."""
    model = make(**kw)
    idx = tokens(2, 160)
    kv = paged(model, 2)
    with torch.no_grad():
        kv.reserve([110, 110])
        model(idx[:, :110], kv_cache=kv)
        kv.increment()
        kv.reserve([10, 18])
        lg, _ = model(idx[:, 110:140], kv_cache=kv)
        kv.increment()
        for b, n in ((0, 120), (1, 128)):
            compare(model, idx[b:b + 1, :n], lg[b:b + 1], torch.float32, f"{kw} row {b}")
    lens = [100, 50]
    want = model.generate(idx[:, :100], 4, temperature=0.0, kv_cache=paged(model, 2), lengths=lens)
    got = model.generate(idx[:, :150], 4, temperature=0.0, kv_cache=paged(model, 2), lengths=lens)
    assert torch.equal(got[:, 150:], want[:, 100:])


def test_generate_takes_settings_per_row():
    """Each of the sampling's settings as a tensor with one value per row."""
    from src.model import kernels
    model = make(n_layer=1)
    idx = tokens(3, 9)
    settings = dict(temperature=torch.tensor([0.7, 1.0, 1.3]).cuda(), top_p=torch.tensor([0.9, 1.0, 0.5]).cuda(),
                    min_p=torch.tensor([0.0, 0.02, 0.01]).cuda())
    for k in (torch.tensor([0, 3, 40], dtype=torch.int32).cuda(), 0, None):
        torch.manual_seed(7)
        w = idx
        with torch.no_grad():
            for _ in range(4):
                t = kernels.sample(model(w)[0][:, -1], torch.rand(3, device="cuda"), top_k=0 if k is None else k, **settings)
                w = torch.cat([w, t[:, None]], 1)
        torch.manual_seed(7)
        assert torch.equal(model.generate(idx, 4, top_k=k, **settings), w)
        torch.manual_seed(7)
        assert torch.equal(model.generate(idx, 4, top_k=k, kv_cache=paged(model, 3), **settings), w)


def test_generate_whatever_the_default_dtype():
    """The drawn numbers are float32, which the sampling takes, also where
    new tensors are something else by default."""
    model = make(n_layer=1)
    idx = tokens(2, 6)
    torch.manual_seed(1)
    want = model.generate(idx, 3, top_p=0.9)
    try:
        torch.set_default_dtype(torch.float64)
        torch.manual_seed(1)
        got = model.generate(idx, 3, top_p=0.9)
    finally:
        torch.set_default_dtype(torch.float32)
    assert torch.equal(got, want)


def test_generate_refuses_before_it_draws():
    """A pool that would run out of pages on the way, and a cache of another
    batch, are refused with nothing drawn and nothing taken; a pool that is
    just large enough serves to the end."""
    model = make(n_layer=1)
    idx = tokens(2, 20)
    # 20 + 13 - 1 = 32 and 4 + 12 = 16 positions of pages of 16: 3 pages; one token more needs 5
    lens, steps = [20, 4], 13
    kv = paged(model, 2, pages=3)
    state = torch.cuda.get_rng_state()
    for n in (steps + 1, 100):
        with pytest.raises(RuntimeError, match="pages"):
            model.generate(idx, n, kv_cache=kv, lengths=lens)
    for other in (1, 3):
        kv2 = paged(model, other, pages=40)
        for ln in (None, lens):
            with pytest.raises(ValueError, match="sequences"):
                model.generate(idx, 2, kv_cache=kv2, lengths=ln)
        assert kv2.free_pages == 40 and not kv2.counts.any()
    assert torch.equal(torch.cuda.get_rng_state(), state) and kv.free_pages == 3 and kv.seq_lens == [0, 0]
    got = model.generate(idx, steps, temperature=0.0, kv_cache=kv, lengths=lens)
    assert torch.equal(got, model.generate(idx, steps, temperature=0.0, kv_cache=paged(model, 2), lengths=lens))
    assert kv.free_pages == 0
    # pages that a sequence holds already count as its own
    kv.reset()
    kv.reserve([17, 1])
    assert torch.equal(model.generate(idx, steps, temperature=0.0, kv_cache=kv, lengths=lens), got)


def test_paged_single_token_refuses_dropout():
    """The kernel drops nothing: in training mode with dropout the step raises
    instead of leaving it out."""
    model = make(n_layer=1, dropout=0.5).train()
    kv = paged(model, 2)
    with torch.no_grad():
        kv.reserve(1)
        with pytest.raises(RuntimeError, match="dropout"):
            model(tokens(2, 1), kv_cache=kv)
        kv.reset()
        kv.reserve(1)
        assert model.eval()(tokens(2, 1), kv_cache=kv)[0].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_windowed_model_with_dropout_trains(dtype):
    """Dropout takes the masked attention of the library: it runs, its result
    is random in training and the kernels' in evaluation."""
    model = make(n_layer=1, dropout=0.3, attn_window=8, attn_sinks=2).train()
    idx, tgt = tokens(2, 40), tokens(2, 40, 2)
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=dtype == torch.bfloat16):
        a, loss = model(idx, targets=tgt)
        loss.backward()
        b, _ = model(idx, targets=tgt)
        assert not torch.equal(a, b)
    assert all(p.grad.isfinite().all() for p in model.parameters() if p.grad is not None)


def test_launch_timing_names_the_kernels_that_ran():
    """Labels are the kernels that the library picked, with the operations of
    the pairs that the mask leaves."""
    from src.model import _hip, kernels
    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731

    def ran(f):
        with _hip.LaunchTimer() as lt:
            f()
        (name, d), = lt.summary().items()
        return name, d["flops"]
    few, many = z(1, 2, 100, 16), z(64, 32, 100, 16)
    assert ran(lambda: kernels.window_attention(few, few, few, 0)) == ("window_fwd_split_kernel", 4 * 2 * 16 * 5050)
    assert ran(lambda: kernels.window_attention(many, many, many, 10, 2)) == \
        ("window_fwd_kernel", 4 * 64 * 32 * 16 * (55 + 90 * 10 + 2 * 90 - 1))
    table, n = z(1, 1).int(), z(1).int() + 64
    for H, name in ((2, "paged_decode_rows_kernel"), (8, "paged_decode_kernel")):
        pages = z(1, 1, 64, 16)
        assert ran(lambda: kernels.paged_decode_attention(z(1, H, 1, 16), pages, pages, table, n))[0] == name


@pytest.mark.parametrize("cls,kw", [("mHCWalsh", dict(attn_window=16, attn_sinks=2)),
                                    ("Walsh", dict(C=1024, n_head=16, attn_window=24, attn_sinks=1, head_mixing=False))])
def test_windowed_model_trains_under_bf16_autocast(cls, kw, monkeypatch):
    """Logits and gradients of a training step on the kernels are as near to
    the float32 step as those of masked attention in bf16."""
    from src.model import kernels
    model = make(cls=cls, **kw).train()
    idx, tgt = tokens(3, 60), tokens(3, 60, 2)

    def step(bf16):
        model.zero_grad()
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=bf16):
            logits, loss = model(idx, targets=tgt)
            loss.backward()
        return logits.detach(), torch.cat([p.grad.reshape(-1) for p in model.parameters() if p.grad is not None])
    own = step(True)
    monkeypatch.setattr(kernels, "window_attention_supported", lambda q: False)
    lib = step(True)
    with sdpa_kernel(SDPBackend.MATH):
        ref = step(False)
    for n, a, b, r in zip(("logits", "gradients"), own, lib, ref):
        print(f"{cls} {n}: {rel(a, r):.2e}, masked attention in bf16 {rel(b, r):.2e}")
        assert rel(a, r) <= max(1e-2, 1.25 * rel(b, r))


@pytest.mark.parametrize("cls", ["mHCWalsh", "Walsh"])
def test_padding_need_not_be_tokens(cls):
    """Prompts padded with -1 and with numbers past the vocabulary, and an idle
    sequence's place, give what padding with a token gives."""
    model = make(n_layer=1, cls=cls)
    idx = tokens(3, 20)
    lens = [20, 4, 11]
    pad = torch.arange(20, device="cuda") >= torch.tensor(lens, device="cuda")[:, None]
    outs = []
    for fill in (0, -1, 2 ** 33):
        kv = paged(model, 3)
        with torch.no_grad():
            kv.reserve(lens)
            a, _ = model(idx.masked_fill(pad, fill), kv_cache=kv)
            kv.increment()
            kv.reserve([1, 0, 1])
            last = idx[:, :1].clone()
            last[1] = fill
            b, _ = model(last, kv_cache=kv)
            kv.increment()
        outs.append((a, b[[0, 2]]))
        if cls == "mHCWalsh":
            new = model.generate(idx.masked_fill(pad, fill), 3, temperature=0.0, kv_cache=paged(model, 3), lengths=lens)
            outs[-1] += (new[:, 20:],)
    for other in outs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(outs[0], other))


@pytest.mark.parametrize("bf16", [False, True])
def test_logits_of_the_last_token_as_before(bf16):
    """Without a paged cache each model forms its last logits from the rows it
    always did: bitwise, where the library's product goes by their strides (a
    weight without gradients, or autocast's copy of one)."""
    kw = dict(n_layer=1, C=512, vocab_size=50257, algebra="octonion", n_head=16)
    idx = tokens(8, 60)
    for cls, rows in (("Walsh", lambda h: h[:, [-1], :]), ("mHCWalsh", lambda h: h[:, -1:, :])):
        model = make(cls=cls, **kw).requires_grad_(False)
        with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16, enabled=bf16):
            logits, _, h = model(idx, return_hidden=True)
            w = model.output.weight.bfloat16() if bf16 else model.output.weight
            assert torch.equal(logits, torch.nn.functional.linear(rows(h), w)), cls
