"""Refusals of the token operators' C entry points, on the host: each comes
before any launch, so pointers are never followed (CPU test)."""
import ctypes
import os

import pytest

P = 4096  # aligned, non-null, never read
EINVAL, ENOTSUP = -1, -2


@pytest.fixture(scope="module")
def L():
    from src.model import _hip
    if not os.path.exists(_hip.LIB_PATH):
        pytest.skip("libwalsh_hip.so not built (run __graft_entry__.build())")
    return _hip.lib()


def logprobs_fwd(L, **k):
    a = dict(logits=P, ld=100, N=4, V=100, tokens=P, n=5, logprob=P, entropy=P, top=P, top_index=P, stats=P, dtype=1)
    a.update(k)
    return L.walsh_token_logprobs_fwd(*a.values(), None)


def logprobs_bwd(L, **k):
    a = dict(logits=P, ld=100, N=4, V=100, tokens=P, n=5, top_index=P, stats=P, g_logprob=P, g_entropy=P, g_top=P,
             dlogits=P, ldd=100, dtype=1)
    a.update(k)
    return L.walsh_token_logprobs_bwd(*a.values(), None)


def dropout(L, **k):
    a = dict(x=P, ldx=64, xdtype=1, residual=P, ldr=64, rdtype=1, M=4, C=64, drop=6554, seed=P, rng_stream=0, y=P, ldy=64,
             ydtype=1)
    a.update(k)
    return L.walsh_dropout(*a.values(), None)


def embedding_fwd(L, **k):
    a = dict(tokens=P, N=4, weight=P, ldw=64, V=10, C=64, scale=ctypes.c_float(1), drop=6554, seed=P, rng_stream=0, y=P,
             ldy=64, wdtype=1, ydtype=1)
    a.update(k)
    return L.walsh_embedding_fwd(*a.values(), None)


def embedding_bwd(L, **k):
    a = dict(tokens=P, N=4, gy=P, ldg=64, V=10, C=64, scale=ctypes.c_float(1), padding_idx=-1, drop=6554, seed=P,
             rng_stream=0, dw=P, ldw=64, gdtype=1, wdtype=1, work=P, work_bytes=1 << 30)
    a.update(k)
    return L.walsh_embedding_bwd(*a.values(), None)


BAD = [(logprobs_fwd, EINVAL, k) for k in (
    dict(N=-1), dict(N=1 << 23), dict(V=0), dict(V=1 << 30, ld=1 << 30), dict(n=-1), dict(n=65), dict(n=60, V=50, ld=50),
    dict(ld=99), dict(logits=0), dict(tokens=0), dict(logprob=0), dict(entropy=0), dict(top=0), dict(top_index=0),
    dict(stats=P + 4))]
BAD += [(logprobs_fwd, ENOTSUP, dict(dtype=2))]
BAD += [(logprobs_bwd, EINVAL, k) for k in (
    dict(N=-1), dict(V=0), dict(n=65), dict(ld=99), dict(ldd=99), dict(logits=0), dict(tokens=0), dict(stats=0),
    dict(dlogits=0), dict(top_index=0), dict(stats=P + 8))]
BAD += [(logprobs_bwd, ENOTSUP, k) for k in (dict(dtype=-1), dict(N=1 << 22, V=1 << 20, ld=1 << 20, ldd=1 << 20))]
BAD += [(dropout, EINVAL, k) for k in (
    dict(drop=-1), dict(drop=65537), dict(rng_stream=-1), dict(rng_stream=1 << 32), dict(x=0), dict(y=0), dict(seed=0),
    dict(ldx=63), dict(ldy=63), dict(ldr=63))]
BAD += [(dropout, ENOTSUP, k) for k in (
    dict(M=-1), dict(C=-1), dict(M=1 << 31, C=1, ldx=1, ldy=1, ldr=1), dict(M=1 << 20, C=1 << 14), dict(C=1 << 31),
    dict(xdtype=2), dict(rdtype=2), dict(ydtype=2), dict(ydtype=0), dict(xdtype=0, ydtype=1), dict(residual=0, ydtype=0))]
BAD += [(embedding_fwd, EINVAL, k) for k in (
    dict(drop=-1), dict(drop=65537), dict(rng_stream=1 << 32), dict(tokens=0), dict(weight=0), dict(y=0), dict(seed=0),
    dict(ldw=63), dict(ldy=63))]
BAD += [(embedding_fwd, ENOTSUP, k) for k in (
    dict(N=-1), dict(V=0), dict(C=-1), dict(V=1 << 31), dict(N=1 << 26, C=1 << 10), dict(wdtype=2), dict(ydtype=-1))]
BAD += [(embedding_bwd, EINVAL, k) for k in (
    dict(drop=-1), dict(rng_stream=-1), dict(tokens=0), dict(gy=0), dict(dw=0), dict(seed=0), dict(work=0), dict(work=P + 4),
    dict(work_bytes=64), dict(ldg=63), dict(ldw=63))]
BAD += [(embedding_bwd, ENOTSUP, k) for k in (
    dict(N=-1), dict(V=0), dict(V=1 << 31), dict(V=1 << 26, C=1 << 10, ldw=1 << 10, ldg=1 << 10), dict(gdtype=2), dict(wdtype=2))]


@pytest.mark.parametrize("call,code,change", BAD, ids=lambda v: getattr(v, "__name__", str(v)))
def test_refused(L, call, code, change):
    assert call(L, **change) == code
    assert L.walsh_last_error().decode().startswith("walsh_" + {"logprobs_fwd": "token_logprobs_fwd",
                                                                "logprobs_bwd": "token_logprobs_bwd"}.get(call.__name__, call.__name__))


def test_nothing_to_do(L):
    """Empty calls are fine, whatever the pointers."""
    assert logprobs_fwd(L, N=0, logits=0, tokens=0) == 0 and logprobs_bwd(L, N=0, logits=0, dlogits=0) == 0
    assert dropout(L, M=0, x=0, y=0) == 0 and dropout(L, C=0, x=0, y=0) == 0
    assert embedding_fwd(L, N=0, tokens=0, y=0) == 0 and embedding_fwd(L, C=0, y=0) == 0
    assert embedding_bwd(L, C=0, dw=0) == 0


def test_workspace_bytes(L):
    """Row starts, sorted places and their tokens, two partial rows for every chunk."""
    f = L.walsh_embedding_bwd_workspace_bytes
    for N, V, C in ((1, 1, 1), (33, 5, 7), (8192, 50257, 512)):
        least = 4 * (V + 1) + 8 * N
        assert least <= f(N, V, C) and f(N, V, C) % 4 == 0
        assert f(N, V, C) >= f(N - 1, V, C)
    assert f(-1, 5, 5) == 0 and f(5, 0, 5) == 0
