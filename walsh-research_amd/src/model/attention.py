"""Windowed attention: differentiable, over the HIP kernels.

The reference's attention is causal over everything (chassis.py:441-478);
here a query sees the last ``window`` keys and the first ``sinks`` ones.
"""
import torch
from torch.autograd.function import once_differentiable

from . import kernels
from ._common import first_order


class WindowAttentionFunction(torch.autograd.Function):
    """walsh_window_attention_fwd / _bwd.  The gradients are not
    differentiable themselves."""

    @staticmethod
    def forward(ctx, q, k, v, window, sinks, lengths, scale):
        o, lse = kernels.window_attention(q, k, v, window, sinks, lengths, scale, need_lse=True)
        ctx.save_for_backward(q, k, v, o, lse, lengths)
        ctx.args = (window, sinks, scale)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, go):
        if not first_order(go):
            raise RuntimeError("window_attention: its gradient takes one plain tensor (no batched or transformed ones)")
        q, k, v, o, lse, lengths = ctx.saved_tensors
        window, sinks, scale = ctx.args
        grads = kernels.window_attention_bwd(q, k, v, o, lse, go, window, sinks, lengths, scale)
        return tuple(g if n else None for g, n in zip(grads, ctx.needs_input_grad)) + (None,) * 4


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0,
                     lengths: torch.Tensor = None, scale: float = None) -> torch.Tensor:
    """softmax(scale q k^T + mask) v with the mask of kernels.window_attention
    (key j <= query position p, and j > p - window or j < sinks): q
    [B, H, Tq, D], k / v [B, G, Tk, D] -> [B, H, Tq, D], differentiable in
    q, k and v."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return WindowAttentionFunction.apply(q, k, v, window, sinks, lengths, scale)
    return kernels.window_attention(q, k, v, window, sinks, lengths, scale)
