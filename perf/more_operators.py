"""Performance cases of the operators at the two ends of a model, tokens to
rows and rows to tokens' probabilities, and of the noise that training adds:

  logprobs    log probabilities of given tokens, the entropy of every row and
              its most probable alternatives, at inference or with gradients
  embed       a scaled embedding lookup, with dropout on its rows where a
              model trains, and the gradient of its weights
  dropout     dropout of rows whose mask is computed again in the backward,
              alone or added to a residual

A case is a dict with a ``kind`` and sizes.  The listed ones stand for real
use, each noted in ``listed``; ``draw`` gives more of the same ranges.  With
``own`` false, ``run`` computes the operators from elementary torch
operations in 32 bits; with ``own`` true it makes the framework's calls.
``exact`` restates them in float64 (the masks in whole numbers).
"""
import math
import os
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # one user's newest token with its five likeliest alternatives: latency
        dict(name="logprobs_one", kind="logprobs", train=False, N=1, V=50257, top_n=5, padded=False, masked=0,
             dtype="bf16"),
        # the newest tokens of a serving batch, twenty alternatives each, a vocabulary padded to a multiple of 64
        dict(name="logprobs_serve", kind="logprobs", train=False, N=64, V=50304, top_n=20, padded=False, masked=47,
             dtype="f32"),
        # scoring given texts: every token of 8 x 1024
        dict(name="logprobs_score", kind="logprobs", train=False, N=8192, V=50257, top_n=0, padded=False, masked=0,
             dtype="bf16"),
        # training on token probabilities and entropy, padded sequences
        dict(name="logprobs_train", kind="logprobs", train=True, N=8192, V=50257, top_n=0, padded=True, masked=0,
             dtype="bf16"),
        # distilling from a few alternatives, float32, odd sizes
        dict(name="logprobs_train_f32", kind="logprobs", train=True, N=999, V=32003, top_n=8, padded=True, masked=0,
             dtype="f32"),
        # the newest tokens of a serving batch into the n_embd-4096 model
        dict(name="embed_step", kind="embed", train=False, N=64, V=50257, C=4096, p=0.0, weight="bf16", out="bf16"),
        # a training micro-batch of the n_embd-512 model, float32 weights, noise on the rows
        dict(name="embed_train_512", kind="embed", train=True, N=8192, V=50257, C=512, p=0.1, weight="f32", out="f32"),
        # a long training batch of the n_embd-4096 model
        dict(name="embed_train_4096", kind="embed", train=True, N=16384, V=50257, C=4096, p=0.0, weight="bf16",
             out="bf16"),
        # a character model: every row of the weights is hit hundreds of times
        dict(name="embed_train_chars", kind="embed", train=True, N=16384, V=65, C=768, p=0.1, weight="f32",
             out="bf16"),
        # a layer's output onto the float32 residual stream of the n_embd-512 model
        dict(name="dropout_train_512", kind="dropout", train=True, M=8192, C=512, p=0.1, dtype="bf16", residual="f32"),
        # the same of the n_embd-4096 model, all bf16
        dict(name="dropout_train_4096", kind="dropout", train=True, M=8192, C=4096, p=0.2, dtype="bf16",
             residual="bf16"),
        # float32 rows of an odd width, no residual
        dict(name="dropout_odd_f32", kind="dropout", train=False, M=1021, C=1365, p=0.5, dtype="f32", residual=""),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("logprobs", "logprobs", "embed", "embed", "dropout"))
    if kind == "logprobs":
        dtype = rng.choice(["bf16", "bf16", "f32"])
        top_n = rng.choice([0, _log(rng, 1, 64)])
        V = _log(rng, 64, 131072)
        room = (2 ** 25 if top_n else 2 ** 28) // (1 if dtype == "bf16" else 2)
        return dict(kind=kind, train=rng.random() < 0.5, N=_log(rng, 1, max(1, min(8192, room // V))), V=V,
                    top_n=top_n, padded=rng.random() < 0.5, masked=rng.choice([0, 0, V // 50]), dtype=dtype)
    if kind == "embed":
        train = rng.random() < 0.6
        C = rng.choice([_log(rng, 16, 4096), 64 * _log(rng, 1, 64)])
        weight = rng.choice(["bf16", "f32"])
        V = _log(rng, 32, min(131072, 2 ** (27 if weight == "bf16" else 26) // C))
        return dict(kind=kind, train=train, N=_log(rng, 1, min(65536, 2 ** 25 // C)), V=V, C=C,
                    p=rng.choice([0.0, rng.uniform(0.01, 0.6)]) if train else 0.0, weight=weight,
                    out=rng.choice(["bf16", weight]))
    C = rng.choice([_log(rng, 8, 8192), 64 * _log(rng, 1, 128)])
    return dict(kind=kind, train=rng.random() < 0.6, M=_log(rng, 1, min(65536, 2 ** 25 // C)), C=C,
                p=rng.uniform(0.01, 0.9), dtype=rng.choice(["bf16", "bf16", "f32"]),
                residual=rng.choice(["", "bf16", "f32"]))


# ------------------------------------------------------------------ inputs

def _package():
    pkg = os.path.join(os.getcwd(), "walsh-research_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)


def _uncounted(case):
    """How many of a case's rows are padding."""
    return case["N"] // 5 if case["padded"] else 0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(dt, *shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dt)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = {"case": case, "own": own}
    if own:
        _package()
    k = case["kind"]
    # whole numbers of 63 bits, on the device, as a captured step keeps them
    s["seed"] = torch.randint(2 ** 63 - 1, (1,), generator=g, device="cuda")
    if k == "logprobs":
        # rows of a language model, some sure and some not; the token is a likely one
        N, V, dt = case["N"], case["V"], _DT[case["dtype"]]
        z = randn(dt, N, V)
        z *= (1.0 + 3.0 * rand(N, 1)).to(dt)
        if case["masked"]:
            z[:, V - case["masked"]:] = -math.inf
        some = (rand(N, 32) * (V - case["masked"])).long()
        s["logits"], s["tokens"] = z, some.gather(1, z.gather(1, some).argmax(1, keepdim=True))[:, 0]
        if _uncounted(case):
            s["tokens"][rand(N).argsort()[:_uncounted(case)]] = -1
        if case["train"]:
            s["g"] = [randn(torch.float32, N) / N, 0.1 * randn(torch.float32, N) / N]
            if case["top_n"]:
                s["g"].append(randn(torch.float32, N, case["top_n"]) / N)
            if own:
                z.requires_grad_(True)
    elif k == "embed":
        # tokens as frequent as words are, in no order of the vocabulary
        N, V, C = case["N"], case["V"], case["C"]
        rank = (torch.exp(rand(N) * math.log(V + 1)) - 1).long().clamp(0, V - 1)
        s["tokens"] = torch.randperm(V, generator=g, device="cuda")[rank]
        s["weight"] = 0.02 * randn(_DT[case["weight"]], V, C)
        s["scale"] = math.sqrt(C)
        if case["train"]:
            s["gy"] = randn(_DT[case["out"]], N, C)
            if own:
                s["weight"].requires_grad_(True)
    else:
        M, C = case["M"], case["C"]
        s["x"] = randn(_DT[case["dtype"]], M, C)
        s["residual"] = randn(_DT[case["residual"]], M, C) if case["residual"] else None
        if case["train"]:
            s["gy"] = randn(_out_dtype(case), M, C)
            if own:
                s["x"].requires_grad_(True)
                if case["residual"]:
                    s["residual"].requires_grad_(True)
    return s


def _out_dtype(case):
    return torch.promote_types(_DT[case["dtype"]], _DT[case["residual"] or case["dtype"]])


# ------------------------------------------------------------------ plain forms

_STREAM = 7


def _keep(case, seed, rows, C):
    """Truth values [rows, C] of what dropout keeps, and the factor of it: 16
    bits of the ten-round generator of Salmon et al. (SC 2011) for every
    element, from the key ``seed`` and the counter (column / 8, row, stream)."""
    w32 = 0xFFFFFFFF
    c = torch.arange(-(-C // 8), device="cuda")[None].expand(rows, -1)
    r = torch.arange(rows, device="cuda")[:, None].expand(-1, c.shape[1])
    x = [c, r & w32, r >> 32, torch.full_like(c, _STREAM)]
    k0, k1 = seed & w32, (seed >> 32) & w32
    for i in range(10):
        if i:
            k0, k1 = (k0 + 0x9E3779B9) & w32, (k1 + 0xBB67AE85) & w32
        # (products of 64 bits wrap; their halves are what is wanted)
        a, b = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
        x = [(b >> 32) & w32 ^ x[1] ^ k0, b & w32, (a >> 32) & w32 ^ x[3] ^ k1, a & w32]
    bits = torch.stack([h for w in x for h in (w & 0xFFFF, w >> 16)], -1).reshape(rows, -1)[:, :C]
    drop = int(round(case["p"] * 65536))
    return bits >= drop, 65536.0 / (65536 - drop)


def _logprobs_plain(s):
    case = s["case"]
    N, V, n = case["N"], case["V"], case["top_n"]
    lp, H = torch.empty(N, device="cuda"), torch.empty(N, device="cuda")
    top, idx = torch.empty(N, n, device="cuda"), torch.empty(N, n, device="cuda", dtype=torch.int64)
    dz = torch.empty_like(s["logits"].detach()) if case["train"] else None
    step = max(1, 2 ** 28 // V)
    for a in range(0, N, step):
        e = min(N, a + step)
        z = s["logits"][a:e].detach().float()
        t = s["tokens"][a:e]
        live = t >= 0
        t = t.clamp_min(0)[:, None]
        d = z - z.amax(-1, keepdim=True)
        w = torch.exp(d)
        S = w.sum(-1, keepdim=True)
        logS = torch.log(S)
        # (what is masked has no weight, whatever its distance)
        h = logS - torch.where(w > 0, w * d, torch.zeros_like(w)).sum(-1, keepdim=True) / S
        lp[a:e] = torch.where(live, (d.gather(1, t) - logS)[:, 0], torch.zeros_like(lp[a:e]))
        H[a:e] = torch.where(live, h[:, 0], torch.zeros_like(lp[a:e]))
        if n:
            i = torch.sort(z, dim=-1, descending=True, stable=True)[1][:, :n]
            top[a:e] = torch.where(live[:, None], d.gather(1, i) - logS, torch.full_like(top[a:e], -math.inf))
            idx[a:e] = torch.where(live[:, None], i, torch.full_like(i, -1))
        if case["train"]:
            g_lp, g_H = s["g"][0][a:e, None], s["g"][1][a:e, None]
            G = g_lp + (s["g"][2][a:e].sum(-1, keepdim=True) if n else 0)
            p = w / S
            g = -p * (G + torch.where(w > 0, g_H * (d - logS + h), torch.zeros_like(w)))
            g.scatter_add_(1, t, g_lp)
            if n:
                g.scatter_add_(1, i, s["g"][2][a:e])
            dz[a:e] = torch.where(live[:, None], g, torch.zeros_like(g)).to(dz.dtype)
    return [lp, H] + ([top, idx] if n else []) + ([dz] if case["train"] else [])


def _embed_plain(s):
    case = s["case"]
    out, w = _DT[case["out"]], s["weight"].detach()
    y = w[s["tokens"]].float()
    f = s["scale"]
    keep = None
    if case["p"]:
        keep, inv = _keep(case, s["seed"], case["N"], case["C"])
        f *= inv
        y = torch.where(keep, y * f, torch.zeros_like(y))
    else:
        y = y * f
    if not case["train"]:
        return [y.to(out)]
    g = s["gy"].float()
    if keep is not None:
        g = torch.where(keep, g, torch.zeros_like(g))
    dw = torch.zeros(w.shape, device="cuda").index_add_(0, s["tokens"], g) * f
    return [y.to(out), dw.to(w.dtype)]


def _dropout_plain(s):
    case = s["case"]
    keep, inv = _keep(case, s["seed"], case["M"], case["C"])
    x = s["x"].detach().float()
    y = torch.where(keep, x * inv, torch.zeros_like(x))
    if s["residual"] is not None:
        y = y + s["residual"].detach().float()
    out = [y.to(_out_dtype(case))]
    if case["train"]:
        g = s["gy"].float()
        out.append(torch.where(keep, g * inv, torch.zeros_like(g)).to(s["x"].dtype))
        if s["residual"] is not None:
            out.append(s["gy"].to(s["residual"].dtype))
    return out


# ------------------------------------------------------------------ run

def run(s):
    case = s["case"]
    k = case["kind"]
    if not s["own"]:
        return {"logprobs": _logprobs_plain, "embed": _embed_plain, "dropout": _dropout_plain}[k](s)
    from src.model import counter_dropout, token_embedding, token_logprobs
    if not case["train"]:
        with torch.no_grad():
            if k == "logprobs":
                r = token_logprobs(s["logits"], s["tokens"], case["top_n"])
                return [r.logprob, r.entropy] + ([r.top_logprob, r.top_index] if case["top_n"] else [])
            if k == "embed":
                return [token_embedding(s["tokens"], s["weight"], s["scale"], out_dtype=_DT[case["out"]])]
            return [counter_dropout(s["x"], case["p"], s["seed"], _STREAM, s["residual"])]
    if k == "logprobs":
        r = token_logprobs(s["logits"], s["tokens"], case["top_n"])
        y = [r.logprob, r.entropy] + ([r.top_logprob] if case["top_n"] else [])
        dz, = torch.autograd.grad(y, [s["logits"]], s["g"])
        return [t.detach() for t in y] + ([r.top_index] if case["top_n"] else []) + [dz]
    if k == "embed":
        y = token_embedding(s["tokens"], s["weight"], s["scale"], out_dtype=_DT[case["out"]], p=case["p"],
                            seed=s["seed"], stream=_STREAM)
        return [y.detach()] + list(torch.autograd.grad(y, [s["weight"]], s["gy"]))
    y = counter_dropout(s["x"], case["p"], s["seed"], _STREAM, s["residual"])
    x = [s["x"]] + ([s["residual"]] if s["residual"] is not None else [])
    return [y.detach()] + list(torch.autograd.grad(y, x, s["gy"]))


# ------------------------------------------------------------------ work

def _size(dtype):
    return 2 if dtype == "bf16" else 4


def work(case):
    k = case["kind"]
    if k == "logprobs":
        rows = case["N"] - _uncounted(case)
        row, e = case["V"], _size(case["dtype"])
        small = case["N"] * (16 + 12 * case["top_n"])
        if not case["train"]:
            return {"bytes": float(rows * row * e + small), "flops": float(6 * rows * row)}
        # the logits in once, their gradient out, in the rows of padding too
        return {"bytes": float((rows + case["N"]) * row * e + 2 * small), "flops": float(12 * rows * row)}
    if k == "embed":
        N, V, C = case["N"], case["V"], case["C"]
        # distinct tokens among N of which the one of rank i has a share of about 1 / ((i + 1) log(V + 1))
        logv = math.log(V + 1)
        marks = [math.exp(logv * i / 256) for i in range(257)]
        distinct = sum((b - a) * -math.expm1(-N / (math.sqrt(a * b) * logv)) for a, b in zip(marks, marks[1:]))
        w, o = C * _size(case["weight"]), C * _size(case["out"])
        n = 8 * N + N * o + distinct * w
        if not case["train"]:
            return {"bytes": float(n), "flops": float(N * C)}
        return {"bytes": float(n + N * o + V * w), "flops": float(4 * N * C)}
    n = case["M"] * case["C"]
    x, r = _size(case["dtype"]), _size(case["residual"]) if case["residual"] else 0
    y = max(x, r)
    # (the residual's gradient is the output's)
    return {"bytes": float(n * (x + r + y + (y + x if case["train"] else 0))), "flops": float(3 * n)}


# ------------------------------------------------------------------ float64 restatement

def _keep_exact(case, seed, rows, C):
    """The mask on the host, in unsigned numbers."""
    import numpy as np
    u = np.uint64
    w32, half = u(0xFFFFFFFF), u(32)
    nb = -(-C // 8)
    out = np.empty((rows, nb, 8), np.uint16)
    seed = u(seed)
    for a in range(0, rows, max(1, 2 ** 18 // nb)):
        r = np.arange(a, min(rows, a + max(1, 2 ** 18 // nb)), dtype=u)[:, None]
        c0 = np.broadcast_to(np.arange(nb, dtype=u)[None], (len(r), nb))
        c1 = np.broadcast_to(r & w32, c0.shape)
        c2 = np.broadcast_to(r >> half, c0.shape)
        c3 = np.full(c0.shape, _STREAM, u)
        k0, k1 = int(seed) & 0xFFFFFFFF, int(seed) >> 32
        for _ in range(10):
            p0, p1 = u(0xD2511F53) * c0, u(0xCD9E8D57) * c2
            c0, c1, c2, c3 = (p1 >> half) ^ c1 ^ u(k0), p1 & w32, (p0 >> half) ^ c3 ^ u(k1), p0 & w32
            k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
        for j, w in enumerate((c0, c1, c2, c3)):
            out[a:a + len(r), :, 2 * j] = w & u(0xFFFF)
            out[a:a + len(r), :, 2 * j + 1] = w >> u(16)
    drop = int(round(case["p"] * 65536))
    return torch.from_numpy(out.reshape(rows, -1)[:, :C] >= drop).cuda(), 65536.0 / (65536 - drop)


def _logprobs_exact(s):
    """Through the log probabilities of whole rows, a few rows at a time."""
    case = s["case"]
    N, V, n = case["N"], case["V"], case["top_n"]
    out = []
    for a in range(0, N, max(1, 2 ** 26 // V)):
        e = min(N, a + max(1, 2 ** 26 // V))
        z = s["logits"][a:e].detach().double()
        dead = s["tokens"][a:e] < 0
        t = s["tokens"][a:e].clamp_min(0)
        logp = torch.log_softmax(z, -1)
        p = logp.exp()
        H = torch.special.entr(p).sum(-1)
        rows = torch.arange(e - a, device="cuda")
        r = [logp[rows, t].masked_fill(dead, 0), H.masked_fill(dead, 0)]
        if n:
            # the n largest, and where the last of them has equals the first of these
            last = torch.topk(z, n, dim=-1)[0][:, -1:]
            order = torch.where(z > last, 2, torch.where(z == last, 1, 0))
            order = torch.where((order == 1) & (torch.cumsum(order == 1, -1) > n - (order == 2).sum(-1, keepdim=True)),
                                torch.zeros_like(order), order)
            i = torch.nonzero(order)[:, 1].reshape(e - a, n)
            i = i.gather(1, torch.sort(z.gather(1, i), dim=-1, descending=True, stable=True)[1])
            r += [logp.gather(1, i).masked_fill(dead[:, None], -math.inf), i.masked_fill(dead[:, None], -1)]
        if case["train"]:
            # the gradient of every log probability, then through the softmax
            g = -s["g"][1][a:e, None].double() * p * (1 + logp.masked_fill(p == 0, 0))
            g[rows, t] += s["g"][0][a:e].double()
            if n:
                g.scatter_add_(1, i, s["g"][2][a:e].double())
            r.append((g - p * g.sum(-1, keepdim=True)).masked_fill(dead[:, None], 0))
        out.append(r)
    return [torch.cat(x) for x in zip(*out)]


def _embed_exact(s):
    case = s["case"]
    y = s["weight"].detach().double()[s["tokens"]] * s["scale"]
    g = s["gy"].double() * s["scale"] if case["train"] else None
    if case["p"]:
        keep, inv = _keep_exact(case, s["seed"].item(), case["N"], case["C"])
        y = y * keep * inv
        g = g * keep * inv
    if g is None:
        return [y]
    # sums of the sorted rows as differences of running ones
    order = torch.argsort(s["tokens"], stable=True)
    run_sum = torch.cat([g.new_zeros(1, g.shape[1]), torch.cumsum(g[order], 0)])
    ends = torch.cumsum(torch.bincount(s["tokens"], minlength=case["V"]), 0)
    begins = torch.cat([ends.new_zeros(1), ends[:-1]])
    return [y, run_sum[ends] - run_sum[begins]]


def _dropout_exact(s):
    case = s["case"]
    keep, inv = _keep_exact(case, s["seed"].item(), case["M"], case["C"])
    y = s["x"].detach().double() * inv * keep
    if s["residual"] is not None:
        y += s["residual"].detach().double()
    out = [y]
    if case["train"]:
        out.append(s["gy"].double() * inv * keep)
        if s["residual"] is not None:
            out.append(s["gy"].double())
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"logprobs": _logprobs_exact, "embed": _embed_exact, "dropout": _dropout_exact}[case["kind"]](s)
