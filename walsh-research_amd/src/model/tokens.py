"""The two ends of a model, differentiable, over the HIP kernels: tokens to
(scaled) rows, rows of logits to tokens' probabilities, and dropout whose mask
is computed again in the backward instead of being stored.

The reference looks tokens up with nn.Embedding, has F.cross_entropy and
sampling behind its logits (chassis.py:533-668, mhc.py:616-772) and drops
attention weights alone.
"""
from typing import NamedTuple

import torch
from torch.nn import functional as F

from . import kernels
from ._common import TENSOR_TYPES, first_order, plain_eager, plain_tensor
from ._hip import dtype_code


def _kernel_tensors(*tensors) -> bool:
    """Whether a call may run kernels: tensors themselves (or None), and no
    transform, trace or mode that has to see each operation."""
    for t in tensors:
        if t is not None and type(t) not in TENSOR_TYPES:
            return False
    return plain_eager()


def _tracked(*tensors) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


# ------------------------------------------------------------------ probabilities

class TokenLogprobs(NamedTuple):
    """What token_logprobs gives: float32 [...], [...], [..., n] and int64 [..., n]."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprob: torch.Tensor
    top_index: torch.Tensor


def _log_softmax(logits):
    """Log probabilities in float32 (-inf all over a row of -inf), which of them
    are probabilities above 0, and which rows have nothing but -inf."""
    z = logits.float()
    nothing = (z == float("-inf")).all(-1, keepdim=True)
    logp = torch.log_softmax(torch.where(nothing, torch.zeros_like(z), z), -1)
    logp = torch.where(nothing, torch.full_like(z, float("-inf")), logp)
    # (not those that are only finite: a distance of 3e38 times a gradient is infinite)
    return logp, ~(logp < -104.0), nothing


def token_logprobs_plain(logits, tokens, top_n=0) -> TokenLogprobs:
    """token_logprobs from torch's operations, for forward-mode derivatives,
    transforms, traces and modes, which have to see each operation."""
    V = logits.shape[-1]
    counted = tokens >= 0
    logits = torch.where(counted[..., None], logits, torch.zeros_like(logits))    # what is not counted reaches nothing
    logp, some, _ = _log_softmax(logits)
    finite = torch.where(some, logp, torch.zeros_like(logp))
    entropy = -torch.where(some, finite.exp() * finite, torch.zeros_like(logp)).sum(-1)
    zero = torch.zeros_like(entropy)
    at = logp.gather(-1, tokens.clamp(0, V - 1)[..., None])[..., 0]
    logprob = torch.where(counted, torch.where(tokens < V, at, torch.full_like(at, float("nan"))), zero)
    # (descending and stable: of equal ones the lowest tokens first; NaN last)
    with torch.no_grad():
        order = torch.where(logits == logits, logits.float(), torch.full_like(logp, float("-inf")))
        index = torch.sort(order, dim=-1, descending=True, stable=True)[1][..., :top_n]
    top = torch.where(counted[..., None], logp.gather(-1, index), torch.full_like(logp[..., :top_n], float("-inf")))
    return TokenLogprobs(logprob, torch.where(counted, entropy, zero), top,
                         torch.where(counted[..., None], index, torch.full_like(index, -1)))


def _logprobs_grad_plain(logits, tokens, index, g_logprob, g_entropy, g_top):
    """The backward from torch's operations, differentiable itself."""
    V = logits.shape[-1]
    counted = (tokens >= 0)[..., None]
    logits = torch.where(counted, logits, torch.zeros_like(logits))
    logp, some, nothing = _log_softmax(logits)
    finite = torch.where(some, logp, torch.zeros_like(logp))
    p = torch.where(some, finite.exp(), torch.zeros_like(logp))
    zero = torch.zeros_like(logp[..., 0])
    g = zero if g_logprob is None else g_logprob
    G = g if g_top is None else g + g_top.sum(-1)
    grad = -p * G[..., None]
    if g_entropy is not None:
        entropy = -(p * finite).sum(-1, keepdim=True)
        grad = grad - g_entropy[..., None] * p * (finite + entropy)
    outside = tokens >= V
    grad = grad.scatter_add(-1, tokens.clamp(0, V - 1)[..., None], torch.where(outside, zero, g)[..., None])
    if g_top is not None:
        grad = grad.scatter_add(-1, index.clamp_min(0), g_top)
    grad = torch.where(outside[..., None], torch.full_like(grad, float("nan")), grad)
    return torch.where(counted & ~nothing, grad, torch.zeros_like(grad)).to(logits.dtype)


class TokenLogprobsFunction(torch.autograd.Function):
    """walsh_token_logprobs_fwd / _bwd; a backward that is itself
    differentiated, batched or looked at takes torch's operations."""

    @staticmethod
    def forward(ctx, logits, tokens, top_n):
        logprob, entropy, top, index, stats = kernels.token_logprobs(logits, tokens, top_n, need_stats=True)
        ctx.save_for_backward(logits, tokens, index, stats)
        ctx.mark_non_differentiable(index)
        ctx.set_materialize_grads(False)
        return logprob, entropy, top, index

    @staticmethod
    def backward(ctx, g_logprob, g_entropy, g_top, _):
        logits, tokens, index, stats = ctx.saved_tensors
        grads = [g for g in (g_logprob, g_entropy, g_top) if g is not None]
        if not grads:
            return None, None, None
        if first_order(grads[0]) and all(plain_tensor(g) for g in grads[1:]):
            return kernels.token_logprobs_bwd_run(logits, dtype_code(logits.dtype), tokens, index, stats, g_logprob,
                                                  g_entropy, g_top), None, None
        return _logprobs_grad_plain(logits, tokens, index, g_logprob, g_entropy, g_top), None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top_n: int = 0) -> TokenLogprobs:
    """The log probabilities of ``tokens`` [...] under softmax(logits
    [..., V]), every row's entropy, and its ``top_n`` most probable tokens with
    their log probabilities (kernels.token_logprobs says what odd rows give).
    Differentiable in the logits through all three.  A row whose token is
    negative is not counted: zeros, and no gradient."""
    if not _kernel_tensors(logits, tokens):
        kernels.check_token_logprobs("token_logprobs", logits, tokens, top_n)
        return token_logprobs_plain(logits, tokens, top_n)
    if _tracked(logits):
        return TokenLogprobs(*TokenLogprobsFunction.apply(logits, tokens, top_n))
    return TokenLogprobs(*kernels.token_logprobs(logits, tokens, top_n))


# ------------------------------------------------------------------ dropout

def kept(rows: int, C: int, drop: int, seed: torch.Tensor, stream: int) -> torch.Tensor:
    """Truth values [rows, C] of what the kernels' dropout keeps, from torch's
    operations (the generator is described in kernels.dropout's C
    declaration: include/walsh.h)."""
    low = 0xFFFFFFFF
    block = torch.arange(-(-C // 8), device=seed.device)[None].expand(rows, -1)
    row = torch.arange(rows, device=seed.device)[:, None].expand_as(block)
    c = [block, row, torch.zeros_like(block), torch.full_like(block, stream)]
    k0, k1 = seed.reshape(()) & low, (seed.reshape(()) >> 32) & low
    for _ in range(10):
        # 64-bit products wrap, their two halves stay right
        p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((q >> 32) & low) ^ c[1] ^ k0, q & low, ((p >> 32) & low) ^ c[3] ^ k1, p & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    bits = torch.stack([h for w in c for h in (w & 0xFFFF, w >> 16)], -1)
    return bits.reshape(rows, -1)[:, :C] >= drop


def _kept_factor(drop):
    return 65536.0 / (65536 - drop) if drop < 65536 else 0.0


def _kept_like(x, drop, seed, stream):
    C = x.shape[-1]
    return kept(x.numel() // C if C else 0, C, drop, seed, stream).reshape(x.shape)


def _drop_plain(x, drop, seed, stream, factor=1.0):
    """factor dropout(x) in float32."""
    x = x.float()
    if drop:
        x = torch.where(_kept_like(x, drop, seed, stream), x, torch.zeros_like(x))
    return x * (factor * _kept_factor(drop))


def counter_dropout_plain(x, p, seed, stream=0, residual=None):
    """counter_dropout from torch's operations."""
    y = _drop_plain(x, kernels.drop_threshold("counter_dropout", p), seed, stream)
    if residual is None:
        return y.to(x.dtype)
    return (y + residual.float()).to(torch.promote_types(x.dtype, residual.dtype))


class CounterDropoutFunction(torch.autograd.Function):
    """walsh_dropout, forward and (on the gradient) backward."""

    @staticmethod
    def forward(ctx, x, residual, p, seed, stream):
        drop, xt, rt = kernels.check_dropout("counter_dropout", x, p, seed, stream, residual)
        ctx.save_for_backward(seed)
        ctx.args = (p, drop, stream, x.dtype, None if residual is None else residual.dtype)
        return kernels.dropout_run(x, drop, xt, rt, seed, stream, residual)

    @staticmethod
    def backward(ctx, gy):
        seed, = ctx.saved_tensors
        p, drop, stream, dtype, rdtype = ctx.args
        gx = gr = None
        if ctx.needs_input_grad[0]:
            if first_order(gy):
                gt = dtype_code(gy.dtype)
                gx = kernels.dropout_run(gy, drop, gt, gt, seed, stream, None, dtype)
            else:
                gx = counter_dropout_plain(gy.float(), p, seed, stream).to(dtype)
        if ctx.needs_input_grad[1]:
            gr = gy.to(rdtype)
        return gx, gr, None, None, None


def counter_dropout(x: torch.Tensor, p: float, seed: torch.Tensor, stream: int = 0,
                    residual: torch.Tensor = None) -> torch.Tensor:
    """Dropout of x [..., C] (and ``residual`` of its shape added, in the wider
    of their types), differentiable in both; no mask is kept.  What is dropped
    is given by ``seed``, an int64 tensor of one element on the device,
    ``stream`` (0 to 2^32 - 1: a number for each place of a model that shares a
    seed) and the element's row and column (kernels.dropout): the same four
    give the same mask.  Probabilities are in steps of 2^-16.  The seed is read
    when the kernels run, so a captured step takes what it holds at each
    replay; it must hold the same in the forward and its backward."""
    if not _kernel_tensors(x, residual, seed):
        kernels.check_dropout("counter_dropout", x, p, seed, stream, residual)
        return counter_dropout_plain(x, p, seed, stream, residual)
    if _tracked(x, residual):
        return CounterDropoutFunction.apply(x, residual, p, seed, stream)
    return kernels.dropout(x, p, seed, stream, residual)


def fresh_seed(device) -> torch.Tensor:
    """A seed from torch's generator of the device (which torch.manual_seed
    sets, and a captured graph moves on with each replay)."""
    return torch.randint(2 ** 63 - 1, (1,), device=device)


# ------------------------------------------------------------------ embedding

def token_embedding_plain(tokens, weight, scale=1.0, padding_idx=None, out_dtype=None, p=0.0, seed=None, stream=0):
    """token_embedding from torch's operations."""
    V = weight.shape[0]
    drop = kernels.drop_threshold("token_embedding", p)
    there = ((tokens >= 0) & (tokens < V))[..., None]
    w = weight.float()
    if padding_idx is not None:
        pad = (torch.arange(V, device=weight.device) == padding_idx)[:, None]
        w = torch.where(pad, w.detach(), w)
    y = _drop_plain(F.embedding(tokens.clamp(0, V - 1), w), drop, seed, stream, scale)
    return torch.where(there, y, torch.full_like(y, float("nan"))).to(out_dtype or weight.dtype)


class TokenEmbeddingFunction(torch.autograd.Function):
    """walsh_embedding_fwd / _bwd."""

    @staticmethod
    def forward(ctx, weight, tokens, scale, padding_idx, out_dtype, p, seed, stream):
        ctx.save_for_backward(tokens, seed)
        ctx.args = (weight.shape[0], scale, padding_idx, weight.dtype, kernels.drop_threshold("token_embedding", p), stream)
        return kernels.embedding(tokens, weight, scale, out_dtype, p, seed, stream)

    @staticmethod
    def backward(ctx, gy):
        tokens, seed = ctx.saved_tensors
        V, scale, padding_idx, dtype, drop, stream = ctx.args
        if first_order(gy):
            gw = kernels.embedding_bwd_run(tokens, gy, V, scale, dtype, padding_idx, drop, dtype_code(gy.dtype),
                                           dtype_code(dtype), seed, stream)
        else:
            g = _drop_plain(gy, drop, seed, stream, scale)
            skip = (tokens < 0) | (tokens >= V)
            if padding_idx is not None:
                skip = skip | (tokens == padding_idx)
            g = torch.where(skip[..., None], torch.zeros_like(g), g).reshape(-1, gy.shape[-1])
            gw = g.new_zeros(V, gy.shape[-1]).index_add(0, tokens.clamp(0, V - 1).reshape(-1), g).to(dtype)
        return (gw,) + (None,) * 7


def token_embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, padding_idx: int = None,
                    out_dtype: torch.dtype = None, p: float = 0.0, seed: torch.Tensor = None,
                    stream: int = 0) -> torch.Tensor:
    """scale weight[tokens], with dropout of probability ``p`` (its ``seed`` and
    ``stream`` as in counter_dropout, a token a row): tokens [...] (int64),
    weight [V, C] -> [..., C] in ``out_dtype`` (None: the weight's), rounded
    once.  Differentiable in the weight; a token's gradients are added in float32
    in a fixed order that depends on the call's tokens and sizes, so equal calls
    give equal bits.  Tokens outside 0 .. V - 1 give rows of NaN and no gradient, and ``padding_idx`` none."""
    plain = not _kernel_tensors(tokens, weight, seed)
    if plain or padding_idx is not None:
        kernels.check_embedding("token_embedding", tokens, weight, p, seed, stream, out_dtype or weight.dtype, padding_idx)
    if plain:
        return token_embedding_plain(tokens, weight, scale, padding_idx, out_dtype, p, seed, stream)
    if _tracked(weight):
        return TokenEmbeddingFunction.apply(weight, tokens, scale, padding_idx, out_dtype, p, seed, stream)
    return kernels.embedding(tokens, weight, scale, out_dtype, p, seed, stream)


# ------------------------------------------------------------------ in a model

_modules = torch.nn.modules.module


def _plain_lookup(e) -> bool:
    """Whether calling the module ``e`` looks rows up and does nothing else: an
    nn.Embedding itself, without hooks, a forward of its own or options that
    change its weights or their gradient's form."""
    return (type(e) is torch.nn.Embedding and "forward" not in e.__dict__
            and e.max_norm is None and not e.sparse and not e.scale_grad_by_freq
            and not (e._forward_hooks or e._forward_pre_hooks or e._backward_hooks or e._backward_pre_hooks
                     or _modules._global_forward_hooks or _modules._global_forward_pre_hooks
                     or _modules._global_backward_hooks or _modules._global_backward_pre_hooks))


def embed_tokens(model, tokens: torch.Tensor, seed: torch.Tensor = None) -> torch.Tensor:
    """A model's token rows: its embedding as it is, or with its config's scale
    and (given a seed) dropout, in one kernel where the module is a lookup and
    no more, else on what the module gives."""
    scale = getattr(model.config, "embed_scale", 1.0)
    p = getattr(model.config, "embed_dropout", 0.0) if seed is not None else 0.0
    e = model.tok_embeddings
    if scale == 1.0 and p == 0.0:
        return e(tokens)
    if _plain_lookup(e):
        if tokens.dtype == torch.int32:          # (an nn.Embedding takes both)
            tokens = tokens.long()
        return token_embedding(tokens, e.weight, scale, e.padding_idx, p=p, seed=seed)
    y = e(tokens)
    rows = y.float() * scale
    return (counter_dropout(rows, p, seed) if p else rows).to(y.dtype)


def step_seed(model, tokens: torch.Tensor):
    """The seed of one forward of a model that trains with dropout of its
    tokens' rows or its layers' outputs, else None."""
    c = model.config
    if model.training and (getattr(c, "embed_dropout", 0.0) != 0 or getattr(c, "resid_dropout", 0.0) != 0):
        return fresh_seed(tokens.device)
    return None


def drop_output(y: torch.Tensor, p: float, seed, layer_idx: int, which: int, residual: torch.Tensor = None) -> torch.Tensor:
    """Output ``which`` (0 attention, 1 feed-forward, 2 channel modulation) of a
    layer with dropout, where the step has a seed, onto the residual stream if
    there is one.  Stream 0 is the tokens' rows', channel modulation's are from
    2^31 on."""
    if seed is None or p == 0.0:
        return y if residual is None else residual + y
    return counter_dropout(y, p, seed, (1 << 31) + layer_idx if which == 2 else 1 + 2 * layer_idx + which, residual)


def stack_steps(steps, idx: torch.Tensor, top_n: int) -> TokenLogprobs:
    """The TokenLogprobs [B, steps] of a loop's steps, each [B]."""
    if not steps:
        none = torch.empty(idx.shape[0], 0, device=idx.device, dtype=torch.float32)
        wide = none.new_empty(idx.shape[0], 0, top_n)
        return TokenLogprobs(none, none.clone(), wide, wide.long())
    return TokenLogprobs(*(torch.stack(parts, 1) for parts in zip(*steps)))


def causal_logits(model, idx: torch.Tensor) -> torch.Tensor:
    """Logits [B, T, V] of every position of idx [B, T], each from the tokens up
    to it: of one forward, or where layers mix positions (channel modulation
    takes means over all of a text's rows) of one for every beginning of the
    texts."""
    if any(getattr(layer, "use_channel_mod", False) for layer in model.layers):
        return torch.cat([model(idx[:, :n])[0] for n in range(1, idx.shape[1] + 1)], 1)
    return model.all_logits(idx)


def text_lengths(lengths, idx: torch.Tensor) -> torch.Tensor:
    """Lengths of the texts idx [B, T] on their device: B whole numbers from 1 to
    T.  (The host reads a device's, except where a transform or trace has to see each
    operation.)"""
    n = torch.as_tensor(lengths)
    if n.numel() == 0:
        n = n.long()
    if n.shape != idx.shape[:1] or n.dtype == torch.bool or n.is_floating_point() or n.is_complex():
        raise ValueError(f"score: lengths {tuple(n.shape)} ({n.dtype}) of texts {tuple(idx.shape)}")
    if plain_eager():
        values = n.tolist()
        if values and (min(values) < 1 or max(values) > idx.shape[1]):
            raise ValueError(f"score: lengths {values} of texts {tuple(idx.shape)}")
    return n.to(device=idx.device, dtype=torch.int64)


def score(model, idx: torch.Tensor, lengths=None, top_n: int = 0) -> TokenLogprobs:
    """The log probabilities of the tokens idx[:, 1:] of idx [B, T], each under
    the model's softmax behind those before it, with entropies and ``top_n``
    alternatives: [B, T - 1].  ``lengths`` (B whole numbers from 1 to T) are the
    tokens that each text has, padded on the right with anything: what lies past them
    is not counted.  Differentiable where autograd is on.  One forward, or T - 1
    of a model with channel modulation (causal_logits), whose training drops
    other things in each."""
    if idx.dim() != 2 or idx.shape[1] < 2:
        raise ValueError(f"score: texts [B, T] of at least two tokens, got {tuple(idx.shape)}")
    if idx.dtype == torch.int32:                 # (models take both)
        idx = idx.long()
    tokens = idx[:, 1:]
    if lengths is not None:
        n = text_lengths(lengths, idx)
        there = torch.arange(idx.shape[1], device=idx.device) < n[:, None]
        idx = torch.where(there, idx, 0)
        tokens = torch.where(there[:, 1:], tokens, -1)
    return token_logprobs(causal_logits(model, idx[:, :-1]), tokens, top_n)
