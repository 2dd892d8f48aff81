"""The paged key-value cache on the GPU: decode attention over it against the
float64 oracle, element by element, and writing into it, exactly.

Tolerances as of the windowed attention: the output is rounded once and bf16
weights once for the product with v, h |o*| + h a_o with h half a step of the
type, a_o = P |v|; float32 scores, exponentials and sums add 2 rho a_o."""
import numpy as np
import pytest
import torch

from oracle import attention as oatt

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def make(B, H, G, D, page, lengths, dtype, seed, per_head=True):
    """A pool with scattered pages and three spare ones; NaN in every row that
    no sequence has; table entries past a sequence's pages are -1."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    P = sum(need) + 3
    order = torch.randperm(P, generator=g).int()
    table = torch.full((B, max(need + [1]) + 1), -1, dtype=torch.int32)
    shape = (P, G, page, D) if per_head else (P, page, G, D)
    pools = [torch.randn(shape, generator=g).to(dtype) for _ in range(2)]
    if not per_head:
        pools = [p.transpose(1, 2) for p in pools]
    used = torch.zeros(P, page, dtype=torch.bool)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
        for i in range(n):
            used[table[b, i], :max(0, lengths[b] - i * page)] = True
    for p in pools:
        p.transpose(1, 2)[~used] = float("nan")
    q = torch.randn(B, H, 1, D, generator=g).to(dtype)
    return q, pools[0], pools[1], table, torch.tensor(lengths, dtype=torch.int32)


def decode(q, kp, vp, table, lengths, W=0, S=0, **kw):
    from src.model import kernels
    o = kernels.paged_decode_attention(q.cuda(), kp.cuda(), vp.cuda(), table.cuda(), lengths.cuda(), W, S, **kw)
    torch.cuda.synchronize()
    return o.cpu()


def check(o, q, kp, vp, table, lengths, W, S):
    D = q.shape[-1]
    want, a = oatt.paged_decode_f64(q[:, :, 0].double().numpy(), kp.double().numpy(), vp.double().numpy(), table.numpy(),
                                    lengths.numpy(), W, S)
    reach = float((q.double().abs().amax((0, 1, 2)) * kp.double().nan_to_num().abs().amax((0, 1, 2))).sum()) * D ** -0.5
    rho = 2.0 ** -24 * (2 * D * reach + int(lengths.max()) + 64)
    h = HALF[q.dtype]
    err, tol = np.abs(o[:, :, 0].double().numpy() - want), h * np.abs(want) + (h + 2 * rho) * a
    print(f"worst error / bound {(err / np.maximum(tol, 1e-30)).max():.3f}", flush=True)
    assert np.isfinite(err).all() and (err <= tol).all()


CASES = [
    # H, G, D, page, lengths, W, S: blocks of 32 to 128 keys, chunks of several, pages that end inside a block
    (2, 2, 128, 16, [1, 17, 0, 300], 0, 0),
    (8, 2, 64, 32, [129, 64, 513], 0, 0),
    (6, 1, 32, 16, [700, 31], 0, 0),
    (40, 1, 16, 64, [200, 65], 0, 0),              # more query heads on one key head than a tile holds
    (4, 4, 128, 64, [1500], 0, 0),
    (4, 2, 64, 16, [400, 90, 100, 7], 100, 5),     # the window alone, exactly full, first tokens apart and adjacent
    (2, 2, 16, 16, [333, 1], 1, 0),
    (3, 3, 32, 128, [5000, 0], 64, 200),
    (2, 1, 128, 256, [9000], 5000, 17),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,G,D,page,lengths,W,S", CASES)
def test_paged_decode_against_oracle(H, G, D, page, lengths, W, S, dtype):
    print(f"case H={H} G={G} D={D} page={page} {lengths} W={W} S={S} {dtype}", flush=True)
    x = make(len(lengths), H, G, D, page, lengths, dtype, D + page, per_head=page != 32)
    o = decode(*x, W, S)
    check(o, *x, W, S)
    assert torch.equal(o, decode(*x, W, S))
    assert not o[x[4] == 0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,G,D,page,lengths,W,S", [
    # 3, 4, 5 and 8 query heads on a key head, lengths about a wavefront's step and a chunk
    (9, 3, 128, 16, [1, 7, 8, 9, 33], 0, 0), (6, 2, 16, 32, [63, 64, 65, 1023, 1025], 0, 0),
    (8, 2, 128, 64, [1024, 2049], 0, 0), (4, 1, 16, 64, [5000, 3], 0, 0), (4, 1, 64, 16, [90, 1700], 300, 9),
    (12, 3, 32, 16, [257, 0, 31], 0, 0), (5, 1, 64, 16, [400, 2], 0, 0), (16, 2, 128, 64, [3000, 64], 1000, 70),
])
def test_paged_decode_shared_heads(H, G, D, page, lengths, W, S, dtype):
    q, kp, vp, table, n = make(len(lengths), H, G, D, page, lengths, dtype, D + H)
    check(decode(q, kp, vp, table, n, W, S), q, kp, vp, table, n, W, S)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,n", [(1, 40), (5, 40), (1, 3000), (5, 3000)])
def test_paged_decode_of_infinite_scores_is_no_number(H, n, dtype):
    """Scores of -inf alone leave no weight, as in the formula: not a number,
    and not the zeros of an empty sequence; other sequences are as without."""
    q, kp, vp, table, lens = make(2, H, 1, 64, 16, [n, 50], dtype, 5)
    want = decode(q, kp, vp, table, lens)
    mine = table[0][table[0] >= 0].long()
    q[0] = 1.0
    kp[mine] = float("-inf")
    got = decode(q, kp, vp, table, lens)
    assert got[0].isnan().all() and torch.equal(got[1], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("H,G,D,lengths,parts", [
    # parts (float32, bf16) of a table as long: joined by 80 and 144 threads' worth of head_dim 16, by 96, 160 and 224
    # of head_dim 32, by whole wavefronts
    (2, 2, 16, [9000, 200], (18, 18)), (4, 1, 16, [17000], (34, 34)), (3, 1, 32, [2500, 64], (10, 5)),
    (2, 2, 32, [4900], (20, 10)), (6, 1, 32, [6700, 3000], (27, 14)), (2, 1, 32, [9900, 513], (39, 20)),
    (2, 1, 64, [2600], (21, 11)), (1, 1, 128, [2600], (21, 21)),
])
def test_paged_decode_joins_scores_of_one_sign(H, G, D, lengths, parts, sign, dtype):
    """Every logit below -120 or above 120: a maximum of the parts that any
    other number enters leaves no weight at all, or infinite ones."""
    from src.model import _hip
    page, B = 64, len(lengths)
    q, kp, vp, table, n = make(B, H, G, D, page, lengths, dtype, D + len(lengths))
    table = table[:, :-1]                          # exactly as many pages as the longest sequence has
    reach = (130.0 / D ** 0.5) ** 0.5
    q, kp = (reach * 1.01 + 0.02 * q.float()).to(dtype), (sign * reach * 1.01 + 0.02 * kp.float()).to(dtype)
    got = _hip.lib().walsh_paged_decode_workspace_bytes(B, H, G, table.shape[1], page, D, 0, 0, _hip.dtype_code(dtype))
    assert got == B * H * parts[dtype == torch.bfloat16] * (D + 2) * 4
    check(decode(q, kp, vp, table, n), q, kp, vp, table, n, 0, 0)


@pytest.mark.gpu
def test_paged_decode_takes_a_dense_cache_as_one_page_per_sequence():
    """[B, H, Lmax, D] storage of any length is B pages; the result equals the
    dense decode attention's up to the order of sums."""
    from src.model import kernels
    B, H, L, Lmax, D = 3, 4, 777, 1001, 64
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(B, H, Lmax, D, generator=g).bfloat16().cuda() for _ in range(2))
    q = torch.randn(B, H, 1, D, generator=g).bfloat16().cuda()
    table = torch.arange(B, dtype=torch.int32, device="cuda")[:, None]
    n = torch.full((B,), L, dtype=torch.int32, device="cuda")
    o = kernels.paged_decode_attention(q, k, v, table, n)
    check(o.cpu(), q.cpu(), k.cpu(), v.cpu(), table.cpu(), n.cpu(), 0, 0)
    d = kernels.decode_attention(q, k[:, :, :L], v[:, :, :L])
    assert (o.float() - d.float()).abs().max() <= 2.0 ** -7 * d.float().abs().max()


@pytest.mark.gpu
def test_paged_decode_bad_pages_and_lengths():
    """A length past the table, or a page number outside the pool among the
    rows that are seen: that sequence is NaN, the others are untouched, and
    nothing outside the pool is read (the kernel checks every number)."""
    q, kp, vp, table, n = make(5, 4, 2, 64, 16, [100, 50, 60, 300, 33], torch.bfloat16, 7)
    want = decode(q, kp, vp, table, n)
    bad = table.clone()
    bad[1, 2] = kp.shape[0]
    bad[3, 0] = -5
    m = n.clone()
    m[2] = table.shape[1] * 16 + 1
    o = decode(q, kp, vp, bad, m)
    assert torch.equal(o[[0, 4]], want[[0, 4]])
    assert o[[1, 2, 3]].isnan().all()
    m[2] = -3
    assert not decode(q, kp, vp, bad, m)[2].any()
    # behind the window it is not looked at
    o = decode(q, kp, vp, bad, n, 20, 0)
    assert torch.equal(o[3], decode(q, kp, vp, table, n, 20, 0)[3])


@pytest.mark.gpu
def test_paged_decode_in_a_graph_with_growing_lengths():
    """Two captured calls (each with its own workspace) replayed while table
    and lengths change, against eager calls."""
    from src.model import kernels
    q, kp, vp, table, n = (t.cuda() for t in make(3, 8, 8, 128, 64, [900, 5, 400], torch.bfloat16, 9))
    kp, vp = kp.nan_to_num(), vp.nan_to_num()
    full = torch.randint(0, kp.shape[0], table.shape, device="cuda", dtype=torch.int32)
    table.copy_(full)

    def step():
        return (kernels.paged_decode_attention(q, kp, vp, table, n),
                kernels.paged_decode_attention(q, kp, vp, table, n, 256, 4))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        n.add_(1)
        q.copy_(torch.randn_like(q))
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.gpu
def test_paged_decode_past_32_bit_offsets():
    """A page that lies more than 2^32 bytes into the pool."""
    from src.model import kernels
    G, page, D = 8, 256, 128
    P = (9 << 29) // (G * page * D * 2) + 2          # 4.5 GiB a pool
    kp = torch.empty(P, G, page, D, dtype=torch.bfloat16, device="cuda")
    vp = torch.empty_like(kp)
    g = torch.Generator(device="cuda").manual_seed(0)
    rows = torch.randn(2, 2, G, page, D, device="cuda", generator=g).bfloat16()
    kp[P - 1], kp[0], vp[P - 1], vp[0] = rows[0, 0], rows[0, 1], rows[1, 0], rows[1, 1]
    q = torch.randn(1, G, 1, D, device="cuda", generator=g).bfloat16()
    n = torch.tensor([300], dtype=torch.int32, device="cuda")
    far = kernels.paged_decode_attention(q, kp, vp, torch.tensor([[P - 1, 0]], dtype=torch.int32, device="cuda"), n)
    near = kernels.paged_decode_attention(q, rows[0].contiguous(), rows[1].contiguous(),
                                          torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), n)
    assert torch.equal(far, near) and far.isfinite().all()
    k = torch.randn(1, 2, G, D, device="cuda", generator=g).bfloat16()
    kernels.paged_kv_write(k, k, kp, vp, torch.tensor([[P - 1]], dtype=torch.int32, device="cuda"),
                           torch.tensor([7], dtype=torch.int32, device="cuda"))
    assert torch.equal(kp[P - 1][:, 7:9], k[0].transpose(0, 1)) and torch.equal(vp[P - 1][:, 7:9], k[0].transpose(0, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,G,D,page,counts", [(1, 1, 1, 16, 16, None), (4, 1, 3, 128, 64, [1, 0, 1, 1]),
                                                 (3, 70, 2, 64, 32, [70, 13, 0]), (2, 9, 5, 32, 16, None)])
def test_paged_write(B, T, G, D, page, counts, dtype):
    """Exactly the rows that are asked for, and no other."""
    from src.model import kernels
    g = torch.Generator().manual_seed(T)
    start = torch.randint(0, 40, (B,), generator=g).int()
    n = counts or [T] * B
    N = (40 + T) // page + 1
    P = B * N + 2
    table = torch.randperm(P, generator=g)[:B * N].reshape(B, N).int()
    kp, vp = (torch.randn(P, page, G, D, generator=g).to(dtype).transpose(1, 2) for _ in range(2))
    k, v = (torch.randn(B, T, G, D, generator=g).to(dtype) for _ in range(2))
    wk, wv = kp.clone(), vp.clone()
    for b in range(B):
        for t in range(n[b]):
            j = int(start[b]) + t
            wk[table[b, j // page], :, j % page] = k[b, t]
            wv[table[b, j // page], :, j % page] = v[b, t]
    dk, dv = kp.cuda(), vp.cuda()
    kernels.paged_kv_write(k.cuda(), v.cuda(), dk, dv, table.cuda(), start.cuda(),
                           None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda"))
    assert torch.equal(dk.cpu(), wk) and torch.equal(dv.cpu(), wv)
    # rows as a projection leaves them, one of heads and tokens strided
    dk, dv = kp.cuda(), vp.cuda()
    big = torch.zeros(2, B, T, G + 1, D, dtype=dtype, device="cuda")
    big[0, :, :, 1:], big[1, :, :, 1:] = k.cuda(), v.cuda()
    kernels.paged_kv_write(big[0, :, :, 1:], big[1, :, :, 1:], dk, dv, table.cuda(), start.cuda(),
                           None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda"))
    assert torch.equal(dk.cpu(), wk) and torch.equal(dv.cpu(), wv)


@pytest.mark.gpu
def test_paged_write_drops_rows_outside():
    from src.model import kernels
    kp, vp = torch.zeros(4, 2, 16, 32, device="cuda"), torch.zeros(4, 2, 16, 32, device="cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.tensor([[0, 1], [4, -1], [2, 3]], dtype=torch.int32, device="cuda")
    k = torch.ones(3, 3, 2, 32, device="cuda")
    kernels.paged_kv_write(k, k, kp, vp, table, i32(30, 14, -2))
    want = torch.zeros_like(kp)
    want[1, :, 14:] = 1       # positions 30, 31 of the first; 32 is past its table
    want[2, :, 0] = 1         # of the third only position 0
    assert torch.equal(kp, want) and torch.equal(vp, want)


def test_paged_refusals_on_the_cpu():
    from src.model import kernels
    z = torch.zeros(1, 1, 1, 16)
    i = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        kernels.paged_decode_attention(z, z, z, i, i[0])
    with pytest.raises(RuntimeError, match="GPU"):
        kernels.paged_kv_write(z, z, z, z, i, i[0])


def test_paged_entry_points_check_before_they_launch():
    """Sizes, strides and workspaces that the kernels do not take are refused
    by the library itself (no pointer is followed)."""
    import os
    from src.model import _hip
    if not os.path.exists(_hip.LIB_PATH):
        pytest.skip("library not built")
    L = _hip.lib()
    p = 4096

    def call(page=64, N=4, D=64, G=2, H=4, P=8, sr=64, q=p, scale=0.1, work=1 << 30, dtype=1, B=1):
        return L.walsh_paged_decode_attention(q, 256, 64, p, p, G * page * 64, page * 64, sr, P, page, p, N, N, p, B, H,
                                              G, D, 0, 0, scale, p, 256, 64, dtype, p, work, None)
    for kw, rc in ((dict(page=48), -2), (dict(page=8), -2), (dict(D=24), -2), (dict(H=3), -1), (dict(P=0), -1),
                   (dict(sr=60), -2), (dict(q=p + 2), -2), (dict(scale=0.0), -1), (dict(dtype=7), -2),
                   (dict(N=1 << 24, page=1 << 10), -1), (dict(N=4096, work=16), -1), (dict(B=-1), -1),
                   (dict(B=65535, H=128), -2)):
        assert call(**kw) == rc, kw
        assert L.walsh_last_error()
    assert call(B=0) == 0
    assert L.walsh_paged_kv_write(p, p, 64, 64, 32, 1, 1, 2, 64, p, p, 64, 64, 64, 1, 64, p, 1, 1, None, None, 1,
                                  None) == -1


@pytest.mark.gpu
def test_paged_refusals():
    from src.model import kernels
    q, kp, vp, table, n = (t.cuda() for t in make(2, 4, 2, 64, 16, [20, 30], torch.bfloat16, 1))
    with pytest.raises(AssertionError, match="evenly"):
        kernels.paged_decode_attention(q[:, :3], kp, vp, table, n)
    with pytest.raises(TypeError, match="pages in"):
        kernels.paged_decode_attention(q.float(), kp, vp, table, n)
    with pytest.raises(TypeError, match="int32"):
        kernels.paged_decode_attention(q, kp, vp, table.long(), n)
    with pytest.raises(AssertionError, match="table"):
        kernels.paged_decode_attention(q, kp, vp, table[:1], n)
    with pytest.raises(AssertionError, match="one layout"):
        kernels.paged_decode_attention(q, kp, vp.transpose(1, 2).contiguous().transpose(1, 2), table, n)
    with pytest.raises(RuntimeError, match="tensors on"):
        kernels.paged_decode_attention(q, kp, vp, table.cpu(), n)
    with pytest.raises(AssertionError, match="do not hold"):
        kernels.paged_kv_write(torch.zeros(2, 1, 3, 64, device="cuda").bfloat16(),
                               torch.zeros(2, 1, 3, 64, device="cuda").bfloat16(), kp, vp, table, n)
    with pytest.raises(TypeError, match="counts"):
        k = torch.zeros(2, 1, 2, 64, device="cuda").bfloat16()
        kernels.paged_kv_write(k, k, kp, vp, table, n, n.long())


@pytest.mark.gpu
@pytest.mark.parametrize("H,G,D,page,lengths,W,S", [
    (2, 2, 128, 16, [1, 17, 300], 0, 0), (8, 2, 64, 32, [129, 64, 513], 0, 0), (6, 1, 32, 16, [700, 31], 0, 0),
    (40, 1, 64, 64, [200, 65], 0, 0), (4, 4, 128, 64, [3000], 100, 5), (16, 2, 32, 64, [5000, 64], 0, 0)])
def test_paged_decode_rounds_bf16_results_once(H, G, D, page, lengths, W, S):
    """From head_dim 32 on the weights go into the product with v in two bf16
    parts, 2^-8 of 2^-8 off: what is left is the one rounding of the output,
    and the float32 sums of the tests above."""
    q, kp, vp, table, n = make(len(lengths), H, G, D, page, lengths, torch.bfloat16, D + H)
    o = decode(q, kp, vp, table, n, W, S)
    want, a = oatt.paged_decode_f64(q[:, :, 0].double().numpy(), kp.double().numpy(), vp.double().numpy(), table.numpy(),
                                    n.numpy(), W, S)
    reach = float((q.double().abs().amax((0, 1, 2)) * kp.double().nan_to_num().abs().amax((0, 1, 2))).sum()) * D ** -0.5
    rho = 2.0 ** -24 * (2 * D * reach + int(n.max()) + 64)
    err, tol = np.abs(o[:, :, 0].double().numpy() - want), 2.0 ** -8 * np.abs(want) + (2.0 ** -16 + 2 * rho) * a
    print(f"worst error / bound {(err / np.maximum(tol, 1e-30)).max():.3f}", flush=True)
    assert (err <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("H,n", [(1, 1), (1, 40), (4, 40), (4, 700), (2, 3000)])
def test_paged_decode_of_equal_values_is_that_value(H, n):
    """A mean of equal values is the value, whatever the weights' roundings:
    at head_dim 16, where bf16 weights are rounded, their sum is taken as
    rounded.  The sums are float32: 2^-24 times the number of terms, far below
    half a step of bf16."""
    q, kp, vp, table, lens = make(1, H, 1, 16, 16, [n], torch.bfloat16, n)
    row = torch.randn(16, generator=torch.Generator().manual_seed(n)).bfloat16()
    vp[:] = row
    o = decode(q, kp, vp, table, lens)
    assert torch.equal(o, row.expand_as(o))
