"""Bookkeeping of the paged key-value cache (CPU: no kernel runs)."""
import pytest
import torch

from src.model import PagedKVCache


def make(**kw):
    args = dict(n_layers=2, n_pages=6, n_head=2, head_dim=16, max_seq_len=64, device="cpu", batch=3, page_size=16)
    args.update(kw)
    return PagedKVCache(**args)


def test_pages_are_taken_as_sequences_grow_and_given_back():
    c = make()
    assert c.page_table.shape == (3, 4) and c.free_pages == 6 and c.cached_len == 0
    c.reserve([20, 3, 0])
    assert c.free_pages == 3 and c.counts.tolist() == [20, 3, 0] and c.totals.tolist() == [20, 3, 0]
    assert c.cached_len == 0
    c.increment()
    assert c.seq_lens == [20, 3, 0] and c.lengths.tolist() == [20, 3, 0] and c.counts.tolist() == [0, 0, 0]
    assert (c.page_table >= 0).sum(1).tolist() == [2, 1, 0]
    used = c.page_table[c.page_table >= 0].tolist()
    assert len(set(used)) == 3 and all(0 <= p < 6 for p in used)
    for _ in range(13):
        c.reserve([0, 1, 0])
        c.increment()
    assert c.seq_lens == [20, 16, 0] and c.free_pages == 3
    c.reserve(1)
    assert c.free_pages == 1 and c.totals.tolist() == [21, 17, 1]
    c.increment()
    c.release(0)
    assert c.free_pages == 3 and c.lengths.tolist() == [0, 17, 1] and (c.page_table[0] == -1).all()
    c.reset()
    assert c.free_pages == 6 and not c.lengths.any() and (c.page_table == -1).all()


def test_reserve_takes_nothing_where_it_fails():
    c = make()
    c.reserve([16, 16, 16])
    c.increment()
    before = (c.free_pages, c.page_table.clone(), c.lengths.clone())
    for bad, err in (([17, 17, 17], RuntimeError), ([49, 0, 0], ValueError), ([1, 1], ValueError), ([-1, 0, 0], ValueError)):
        with pytest.raises(err):
            c.reserve(bad)
        assert c.free_pages == before[0] and torch.equal(c.page_table, before[1]) and torch.equal(c.lengths, before[2])


def test_several_tokens_need_one_length():
    c = make()
    c.reserve([5, 9, 0])
    c.increment()
    c.reserve([2, 0, 0])
    assert c.cached_len == 5
    c.reserve([2, 2, 0])
    with pytest.raises(ValueError, match="one length"):
        c.cached_len


def test_refusals():
    for kw in (dict(page_size=24), dict(page_size=8), dict(head_dim=20)):
        with pytest.raises(ValueError):
            make(**kw)
    c = make()
    k = torch.zeros(3, 1, 2, 16, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="reserved"):
        c.write(0, k, k)
    c.reserve(2)
    with pytest.raises(RuntimeError, match="1 tokens with 2 reserved"):
        c.write(0, k, k)
    with pytest.raises(AssertionError):
        c.write(0, k[:2], k[:2])


def test_dual_numbers_and_traces_are_refused():
    """Kernels that see values alone would drop a tangent without a word, and
    leave nothing in a trace."""
    import torch.autograd.forward_ad as fw
    c = make()
    c.reserve(1)
    k = torch.ones(3, 1, 2, 16, dtype=torch.bfloat16)
    q = torch.ones(3, 2, 1, 16, dtype=torch.bfloat16)
    with fw.dual_level():
        for args in ((fw.make_dual(k, k), k), (k, fw.make_dual(k, k))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                c.write(0, *args)
        with pytest.raises(RuntimeError, match="forward-mode"):
            c.attend(0, fw.make_dual(q, q))
        # a level alone is no reason: these get to the kernels, which want a GPU
        with pytest.raises(RuntimeError, match="GPU"):
            c.write(0, k, k)
        with pytest.raises(RuntimeError, match="GPU"):
            c.attend(0, q)
    with pytest.raises(RuntimeError, match="traces"):
        torch.jit.trace(lambda q: c.attend(0, q), (q,), check_trace=False)


def test_rotary_rows_of_padding_past_the_table():
    """A padded part may end past the rotary table as long as the tokens that
    count do not: their rows are theirs, the padding's are any."""
    from src.model.chassis import cache_freqs
    table = torch.arange(128)[:, None].expand(128, 4)
    c = make(n_pages=24, max_seq_len=128)
    c.reserve([110, 110, 3])
    c.increment()
    c.reserve([10, 18, 0])
    for T, n in ((18, 18), (19, 18), (30, 18), (300, 18)):
        rows = cache_freqs(table, T, 0, c)
        assert rows.shape == (T, 4) and rows[:n, 0].tolist() == list(range(110, 110 + n))


def test_tokens_that_do_not_count_are_replaced():
    """Padding and idle sequences may hold any number: the embedding sees
    token 0 there, and the tokens that count as they are."""
    from src.model.chassis import counted_tokens
    c = make()
    far = 2 ** 40
    c.reserve([3, 0, 4])
    idx = torch.tensor([[5, 6, 7, -1, far], [-1, -1, -1, -1, -1], [1, 2, 3, 4, -100]])
    assert counted_tokens(idx, c).tolist() == [[5, 6, 7, 0, 0], [0] * 5, [1, 2, 3, 4, 0]]
    assert counted_tokens(idx[:, :3].int(), c).tolist() == [[5, 6, 7], [0] * 3, [1, 2, 3]]
    c.increment()
    c.reserve([1, 0, 1])
    assert counted_tokens(torch.tensor([[9], [far], [8]]), c).tolist() == [[9], [0], [8]]
    for other in (None, object()):
        assert counted_tokens(idx, other) is idx
    assert counted_tokens(idx[:2], c).tolist() == idx[:2].tolist()   # another batch: the cache's own check says so
