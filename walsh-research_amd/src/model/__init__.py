"""Walsh ternary structured-linear hot path on MI355X (HIP kernels behind a C ABI).

Same public surface as the reference package ``src.model``
(src/model/__init__.py:1-2), and beside it what the reference has none of:
the windowed attention, the paged cache, tokens' probabilities, the scaled
embedding lookup and dropout without a mask.
"""
from .attention import PagedKVCache, window_attention
from .chassis import KVCache, Walsh, WalshConfig
from .mhc import SinkhornKnopp, mHCResidualStream, mHCWalsh
from .tokens import TokenLogprobs, counter_dropout, token_embedding, token_logprobs

__all__ = ["Walsh", "WalshConfig", "KVCache", "mHCWalsh", "mHCResidualStream", "SinkhornKnopp",
           "PagedKVCache", "window_attention", "TokenLogprobs", "counter_dropout", "token_embedding", "token_logprobs"]
