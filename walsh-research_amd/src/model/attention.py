"""Windowed attention, differentiable, and the paged key-value cache, over the
HIP kernels.

The reference's attention is causal over everything (chassis.py:441-478) and
its cache one dense tensor (:262-330); here a query may see the last
``window`` keys and the first ``sinks`` ones, and the cache may lie in pages.
"""
import math
import numbers
from typing import List, Sequence, Union

import torch
from torch.autograd.function import once_differentiable

from . import kernels
from ._common import TENSOR_TYPES, carries_tangent, first_order, plain_eager, plain_tensor


def window_attention_plain(q, k, v, window, sinks=0, lengths=None, scale=None):
    """window_attention from torch's operations, in float32 and rounded once:
    for forward-mode derivatives, transforms, traces and modes, which have to
    see each operation.  As in the kernels, what lies in rows without a key and
    past the lengths reaches nothing, gradients included."""
    B, H, Tq, D = q.shape
    G, Tk = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else float(scale)
    p = torch.arange(Tk - Tq, Tk, device=q.device)
    j = torch.arange(Tk, device=q.device)
    n = lengths[:, None] if lengths is not None else torch.full((1, 1), int(Tk), device=q.device)
    live = (p >= 0) & (p < n)
    sees = j <= p[:, None]
    if window > 0:
        sees = sees & ((j > p[:, None] - window) | (j < sinks))
    sees = (sees | ~live[:, :, None])[:, None, None]      # a row without a key: any weights, and no output
    live, there = live[:, None, :, None], (j < n)[:, None, :, None]
    # no autocast: bf16 batched products with a transposed operand have faulted the GPU
    with torch.autocast(q.device.type, enabled=False):
        qf = torch.where(live, q.float(), 0.).reshape(B, G, H // G, Tq, D)
        kf, vf = (torch.where(there, t.float(), 0.)[:, :, None] for t in (k, v))
        w = torch.softmax((torch.matmul(qf, kf.transpose(3, 4)) * scale).masked_fill(~sees, -math.inf), -1)
        o = torch.matmul(w, vf).reshape(B, H, Tq, D)
        return torch.where(live, o, 0.).to(q.dtype)


class WindowAttentionFunction(torch.autograd.Function):
    """walsh_window_attention_fwd / _bwd.  The gradients are not
    differentiable themselves."""

    @staticmethod
    def forward(ctx, q, k, v, window, sinks, lengths, scale):
        o, lse, rest = kernels.window_attention(q, k, v, window, sinks, lengths, scale, need_rest=True)
        ctx.save_for_backward(q, k, v, o, lse, lengths, rest)
        ctx.args = (window, sinks, scale)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, go):
        q, k, v, o, lse, lengths, rest = ctx.saved_tensors
        window, sinks, scale = ctx.args
        if first_order(go):
            grads = kernels.window_attention_bwd(q, k, v, o, lse, go, window, sinks, lengths, scale, rest)
        elif plain_tensor(go):
            # a mode, trace or forward derivative looks at the backward's operations
            with torch.enable_grad():
                x = [t.detach().requires_grad_(True) for t in (q, k, v)]
                grads = torch.autograd.grad(window_attention_plain(*x, window, sinks, lengths, scale), x, go)
        else:
            raise RuntimeError("window_attention: its gradient takes one plain tensor (no batched or transformed ones)")
        return tuple(g if n else None for g, n in zip(grads, ctx.needs_input_grad)) + (None,) * 4


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0,
                     lengths: torch.Tensor = None, scale: float = None) -> torch.Tensor:
    """softmax(scale q k^T + mask) v with the mask of kernels.window_attention
    (key j <= query position p, and j > p - window or j < sinks): q
    [B, H, Tq, D], k / v [B, G, Tk, D] -> [B, H, Tq, D], differentiable in
    q, k and v: once backward on the kernels; forward-mode derivatives,
    torch.func's transforms, traces and dispatch modes take
    window_attention_plain, whose [Tq, Tk] weights lie in memory."""
    if not (type(q) in TENSOR_TYPES and type(k) in TENSOR_TYPES and type(v) in TENSOR_TYPES and plain_eager()):
        kernels.check_window_attention("window_attention", q, k, v, lengths, scale)
        return window_attention_plain(q, k, v, window, sinks, lengths, scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return WindowAttentionFunction.apply(q, k, v, window, sinks, lengths, scale)
    return kernels.window_attention(q, k, v, window, sinks, lengths, scale)


def window_mask(Tq: int, Tk: int, window: int, sinks: int, device) -> torch.Tensor:
    """[Tq, Tk] truth values of the mask, for attention that takes one."""
    p = torch.arange(Tk - Tq, Tk, device=device)[:, None]
    j = torch.arange(Tk, device=device)[None, :]
    return (j <= p) & ((j > p - window) | (j < sinks))


def _plain_values(*tensors) -> None:
    """The cache's kernels see values alone: what would be lost is refused."""
    if torch.jit.is_tracing() or any(carries_tangent(t) for t in tensors):
        raise RuntimeError("PagedKVCache: no forward-mode derivatives and no traces")


class PagedKVCache:
    """Per-layer keys and values of ``batch`` sequences of their own lengths,
    in pages of ``page_size`` tokens that a sequence takes as it grows and
    gives back when it ends.

    A forward with T tokens per sequence:

        cache.reserve(counts)      # how many of the T each sequence keeps
        logits, _ = model(idx, kv_cache=cache)
        cache.increment()          # they count from now on

    T == 1 takes sequences of any lengths; T > 1 (prompts, padded on the right
    to T) needs those that keep some to stand at one length.  ``counts`` 0
    leaves a sequence as it is.  A cache holds values alone: gradients,
    forward-mode derivatives and traces through it are refused.  The tensors that the kernels read
    (``page_table`` [batch, pages], ``lengths``, ``counts``, ``totals``
    [batch], int32) keep their addresses, so a captured forward of T == 1 can
    be replayed between ``reserve(1)`` and ``increment()``."""

    def __init__(self, n_layers: int, n_pages: int, n_head: int, head_dim: int, max_seq_len: int, device,
                 dtype: torch.dtype = torch.bfloat16, batch: int = 1, page_size: int = 64):
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError(f"PagedKVCache: page_size {page_size} (a power of two from 16)")
        if head_dim not in kernels.ATTENTION_HEAD_DIMS:
            raise ValueError(f"PagedKVCache: head_dim {head_dim} (one of {kernels.ATTENTION_HEAD_DIMS})")
        self.batch, self.page_size, self.max_seq_len = batch, page_size, max_seq_len
        # one layout of both: [pages, heads, rows, head_dim], a head's rows together
        self.k_pages: List[torch.Tensor] = [torch.zeros(n_pages, n_head, page_size, head_dim, device=device, dtype=dtype)
                                            for _ in range(n_layers)]
        self.v_pages: List[torch.Tensor] = [torch.zeros_like(k) for k in self.k_pages]
        per_seq = max(1, -(-max_seq_len // page_size))
        self.page_table = torch.full((batch, per_seq), -1, dtype=torch.int32, device=device)
        self.lengths, self.counts, self.totals = (torch.zeros(batch, dtype=torch.int32, device=device) for _ in range(3))
        self.seq_lens = [0] * batch
        self._counts = [0] * batch
        self._pages: List[List[int]] = [[] for _ in range(batch)]
        self._free = list(range(n_pages))[::-1]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def cached_len(self) -> int:
        """The length at which the sequences that take tokens now stand."""
        at = {n for n, c in zip(self.seq_lens, self._counts) if c > 0}
        if len(at) > 1:
            raise ValueError(f"several tokens at once need sequences of one length, got {sorted(at)}")
        return at.pop() if at else 0

    def require_pages(self, ends: Sequence[int]) -> List[int]:
        """Pages that each sequence still lacks to be ``ends`` long; raises
        where the pool has fewer."""
        more = [max(0, -(-e // self.page_size) - len(p)) for e, p in zip(ends, self._pages)]
        if sum(more) > len(self._free):
            raise RuntimeError(f"PagedKVCache: {sum(more)} pages needed, {len(self._free)} free")
        return more

    def reserve(self, counts: Union[int, Sequence[int]]) -> None:
        """Room for the next ``counts`` tokens (one number, or one per
        sequence) of the coming forward; nothing is taken if any does not
        fit."""
        counts = [int(counts)] * self.batch if isinstance(counts, numbers.Integral) else [int(c) for c in counts]
        if len(counts) != self.batch or min(counts) < 0:
            raise ValueError(f"PagedKVCache: counts for {self.batch} sequences, got {counts}")
        ends = [n + c for n, c in zip(self.seq_lens, counts)]
        if max(ends) > self.max_seq_len:
            raise ValueError(f"PagedKVCache: {max(ends)} tokens of at most {self.max_seq_len}")
        more = self.require_pages(ends)
        if any(more):
            for pages, n in zip(self._pages, more):
                pages.extend(self._free.pop() for _ in range(n))
            self._put_table()
        if min(counts) == max(counts):
            self.counts.fill_(counts[0])
        else:
            self.counts.copy_(torch.tensor(counts, dtype=torch.int32))
        self._counts = counts
        torch.add(self.lengths, self.counts, out=self.totals)

    def increment(self) -> None:
        """The reserved tokens are in the cache; no sequence takes any until
        the next ``reserve``."""
        self.seq_lens = [n + c for n, c in zip(self.seq_lens, self._counts)]
        self._counts = [0] * self.batch
        self.lengths.copy_(self.totals)
        self.counts.zero_()

    def release(self, seq: int) -> None:
        """Ends sequence ``seq``: its pages are free, its length is 0, and it
        takes no tokens until the next ``reserve``."""
        self._free.extend(self._pages[seq][::-1])
        self._pages[seq] = []
        self.seq_lens[seq] = self._counts[seq] = 0
        for t in (self.lengths, self.counts, self.totals):
            t[seq] = 0
        self._put_table()

    def reset(self) -> None:
        for seq in range(self.batch):
            if self._pages[seq]:
                self.release(seq)

    def _put_table(self) -> None:
        width = self.page_table.shape[1]
        self.page_table.copy_(torch.tensor([p + [-1] * (width - len(p)) for p in self._pages], dtype=torch.int32))

    # ---- what a layer does

    def write(self, layer_idx: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """New k and v [batch, T, heads, head_dim]: each sequence's first
        ``counts``."""
        assert k.shape[0] == self.batch, f"{k.shape[0]} rows for a cache of {self.batch} sequences"
        if max(self._counts) == 0 or max(self._counts) > k.shape[1]:
            raise RuntimeError(f"PagedKVCache: a forward of {k.shape[1]} tokens with {max(self._counts)} reserved")
        _plain_values(k, v)
        kp, vp = self.k_pages[layer_idx], self.v_pages[layer_idx]
        kernels.paged_kv_write(k.detach().to(kp.dtype), v.detach().to(vp.dtype), kp, vp, self.page_table, self.lengths,
                               self.counts)

    def attend(self, layer_idx: int, q: torch.Tensor, window: int = 0, sinks: int = 0) -> torch.Tensor:
        """Attention of q [batch, heads, 1, head_dim], the sequences' newest
        tokens, over the cache with what was written for them."""
        _plain_values(q)
        kp = self.k_pages[layer_idx]
        return kernels.paged_decode_attention(q.detach().to(kp.dtype), kp, self.v_pages[layer_idx], self.page_table,
                                              self.totals, window, sinks)

    def rows(self, layer_idx: int, n: int):
        """The first n rows of every sequence, [batch, n, heads, head_dim] of
        k and of v (copies; zeros past a sequence's length)."""
        j = torch.arange(n, device=self.page_table.device)
        pages = self.page_table[:, j // self.page_size].clamp_min(0).long()
        there = (j < self.lengths[:, None])[:, :, None, None]
        return tuple(torch.where(there, t[layer_idx][pages, :, j % self.page_size], 0)
                     for t in (self.k_pages, self.v_pages))
