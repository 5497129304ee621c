"""Timed workloads of the operators that distilling a student model and serving
it add: the norms of queries and keys with the position rotation, the scaled
embedding with its gradient, and the distillation loss from a teacher's top
logits.

A case is a dict of plain values; the tensors come from the seed that
``prepare`` gets.  With ``own`` the framework's operators run, without it the
same mathematics in elementary torch operations.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

VOCAB = 50257
IGNORE = -100
EPS = 1e-6


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # The attention prologue of one layer of the 12-layer training step,
        # forward and backward over a packed 16k row.
        dict(name="qk_train", kind="qk", dtype="bfloat16", B=1, T=16384, H=12, Hkv=12, D=64,
             train=1),
        # Grouped heads of 128, two rows of an odd length.
        dict(name="qk_gqa_train", kind="qk", dtype="bfloat16", B=2, T=4097, H=16, Hkv=2, D=128,
             train=1),
        # A short float32 row (a model that is not cast): latency.
        dict(name="qk_f32_small", kind="qk", dtype="float32", B=1, T=513, H=8, Hkv=8, D=64,
             train=1),
        # The prologue of scoring or prefilling a context, forward only.
        dict(name="qk_score", kind="qk", dtype="bfloat16", B=1, T=2048, H=12, Hkv=12, D=64,
             train=0),
        # One generated token: its query, and its key and value into the cache.
        dict(name="qk_token", kind="append", dtype="bfloat16", B=1, M=1, H=12, Hkv=12, D=64,
             cap=4096),
        # The embedding of the training step and its weight gradient.
        dict(name="embed_train", kind="embed", dtype="bfloat16", N=16384, V=VOCAB, C=768, pad=-1,
             train=1),
        # A large batch, the longest lists of equal tokens; padded rows.
        dict(name="embed_batch", kind="embed", dtype="bfloat16", N=131072, V=VOCAB, C=768, pad=0,
             train=1),
        # A small float32 model, an odd number of tokens.
        dict(name="embed_f32_small", kind="embed", dtype="float32", N=1537, V=8192, C=512, pad=0,
             train=1),
        # One generated token's embedding.
        dict(name="embed_token", kind="embed", dtype="bfloat16", N=1, V=VOCAB, C=768, pad=-1,
             train=0),
        # The distillation step's loss and logit gradient, temperature 2, half
        # of the weight on the hard labels.
        dict(name="distill_train", kind="distill", dtype="bfloat16", N=8192, V=VOCAB, K=64, tau=2.0,
             alpha=0.5, train=1),
        # Losses of every token of a held-out row.
        dict(name="distill_eval", kind="distill", dtype="bfloat16", N=2048, V=VOCAB, K=32, tau=1.0,
             alpha=1.0, train=0),
        # A small float32 model and vocabulary.
        dict(name="distill_f32_small", kind="distill", dtype="float32", N=96, V=8192, K=16, tau=1.5,
             alpha=0.7, train=1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(12, 12, 64), (8, 8, 64), (4, 4, 128), (16, 2, 128), (16, 4, 64), (16, 16, 128), (6, 3, 64)]


def draw(rng):
    kind = rng.choice(["qk", "qk", "append", "embed", "embed", "distill", "distill"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    H, Hkv, D = rng.choice(HEADS)
    if kind == "qk":
        B = rng.choice([1, 2, 3])
        return dict(kind="qk", dtype=dtype, B=B, T=_log_int(rng, 1, 16384 // B), H=H, Hkv=Hkv, D=D,
                    train=rng.choice([0, 1, 1]))
    if kind == "append":
        return dict(kind="append", dtype=dtype, B=rng.choice([1, 2, 5, 8]), M=rng.randint(1, 8),
                    H=H, Hkv=Hkv, D=D, cap=_log_int(rng, 16, 4096))
    if kind == "embed":
        return dict(kind="embed", dtype=dtype, N=_log_int(rng, 1, 65536),
                    V=rng.choice([VOCAB, 8192, _log_int(rng, 300, VOCAB)]),
                    C=rng.choice([512, 768, 1024, 8 * rng.randint(5, 90)]), pad=rng.choice([-1, 0]),
                    train=rng.choice([0, 1, 1]))
    V = rng.choice([VOCAB, _log_int(rng, 300, VOCAB)])
    return dict(kind="distill", dtype=dtype, N=_log_int(rng, 1, 4096), V=V,
                K=_log_int(rng, 1, 256), tau=rng.choice([1.0, 2.0, round(rng.uniform(0.5, 4), 2)]),
                alpha=rng.choice([1.0, 0.5, round(rng.uniform(0.1, 0.9), 2)]),
                train=rng.choice([0, 1, 1]))


# -------------------------------------------------------------------- inputs

def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _tables(rows, D, dev):
    """cos / sin of position * 10000^(-i / (D / 2)), float32 [rows, D / 2]."""
    inv = 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))
    ang = torch.outer(torch.arange(rows, dtype=torch.float64), inv)
    return ang.cos().float().to(dev), ang.sin().float().to(dev)


def _zipf(V):
    """Token frequencies by id: 1 / (id + 2.7)."""
    p = 1.0 / (np.arange(V) + 2.7)
    return p / p.sum()


def prepare(case, seed):
    dev = _device()
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = getattr(torch, case["dtype"])

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=dev)

    s = dict(case)
    if case["kind"] in ("qk", "append"):
        B, H, Hkv, D = (case[n] for n in ("B", "H", "Hkv", "D"))
        T = case["T"] if case["kind"] == "qk" else case["M"]
        # projections whose size differs from row to row, as an unnormed
        # attention input's does
        s["qkv"] = (randn(B, T, (H + 2 * Hkv) * D) * (0.5 + 2 * rand(B, T, 1))).to(dt)
        s["qw"], s["kw"] = ((1 + 0.1 * randn(D)).to(dt) for _ in range(2))
        if case["kind"] == "append":
            cap = case["cap"]
            s["cos"], s["sin"] = _tables(cap, D, dev)
            s["kc"], s["vc"] = (randn(B, Hkv, cap, D).to(dt) for _ in range(2))
            # each sequence's new rows behind its context
            first = (rand(B, 1) * (cap - T + 1)).long().clamp_(max=cap - T)
            s["pos"] = first + torch.arange(T, device=dev)
            return s
        s["cos"], s["sin"] = _tables(T, D, dev)
        if case["train"]:
            s["grads"] = tuple(randn(B, h, T, D).to(dt) for h in (H, Hkv, Hkv))
            for n in ("qkv", "qw", "kw"):
                s[n].requires_grad_(True)
        return s
    if case["kind"] == "embed":
        N, V, C = case["N"], case["V"], case["C"]
        cdf = torch.from_numpy(np.cumsum(_zipf(V))).to(dev)
        u = torch.rand(N, generator=g, device=dev, dtype=torch.float64)
        s["tokens"] = torch.searchsorted(cdf, u).clamp_(max=V - 1)
        s["scale"] = math.sqrt(C)
        s["weight"] = (randn(V, C) * C ** -0.5).to(dt)
        if case["train"]:
            s["dy"] = randn(N, C).to(dt)
            s["weight"].requires_grad_(True)
        return s
    N, V, K = case["N"], case["V"], case["K"]
    # K distinct ids a row, the teacher's logits falling over them, the
    # student's raised at the same ids
    step = 1 + (rand(N, 1) * (V // K - 1)).long()
    at = ((rand(N, 1) * V).long().clamp_(max=V - 1) + step * torch.arange(K, device=dev)) % V
    t = 8 - 2 * torch.log1p(torch.arange(K, device=dev, dtype=torch.float32)) + 0.5 * randn(N, K)
    z = 2 * randn(N, V)
    z.scatter_(1, at, 0.7 * t + randn(N, K))
    # rows with fewer slots than K, rows without any, rows not counted
    u = rand(N, 1)
    keep = torch.where(u < 0.03, 0, torch.where(u < 0.15, (rand(N, 1) * K).long(), K))
    idx = torch.where(torch.arange(K, device=dev) < keep, at, -1)
    target = torch.where(rand(N) < 0.7, at[:, 0], (rand(N) * V).long().clamp_(max=V - 1))
    s["targets"] = torch.where((rand(N) < 1 / 16) & (torch.arange(N, device=dev) > 0), IGNORE,
                               target)
    s["idx"] = idx.int() if case["dtype"] == "bfloat16" else idx
    s["t"] = t.to(dt)
    s["z"] = z.to(dt)
    if case["train"]:
        s["z"].requires_grad_(True)
    return s


# ------------------------------------------------------- the framework's calls

def _own_qk(s):
    from tagseq2tagseq_amd.rope import qk_norm_rope
    out = qk_norm_rope(s["qkv"], s["qw"], s["kw"], s["cos"], s["sin"], s["H"],
                       num_kv_heads=s["Hkv"], eps=EPS)
    if not s["train"]:
        return out
    return out, torch.autograd.grad(out, (s["qkv"], s["qw"], s["kw"]), s["grads"])


def _own_append(s):
    from tagseq2tagseq_amd.rope import qk_norm_rope_append
    q = qk_norm_rope_append(s["qkv"], s["qw"], s["kw"], s["cos"], s["sin"], s["H"], s["pos"],
                            s["kc"], s["vc"], eps=EPS)
    return q, s["kc"], s["vc"]


def _own_embed(s):
    from tagseq2tagseq_amd.embedding import embedding
    pad = s["pad"] if s["pad"] >= 0 else None
    out = embedding(s["tokens"], s["weight"], scale=s["scale"], padding_idx=pad)
    if not s["train"]:
        return out
    return out, torch.autograd.grad(out, s["weight"], s["dy"])


def _own_distill(s):
    from tagseq2tagseq_amd.distill import distill_loss
    loss = distill_loss(s["z"], s["idx"], s["t"], s["targets"], temperature=s["tau"],
                        alpha=s["alpha"], ignore_index=IGNORE,
                        reduction="mean" if s["train"] else "none")
    if not s["train"]:
        return loss
    return loss, torch.autograd.grad(loss, s["z"])


# ------------------------------------------------------------ the plain forms

def _heads(x, H, Hkv):
    """q, k, v [B, heads, T, D] of packed rows [B, T, (H + 2 Hkv) D]."""
    x = x.view(x.shape[0], x.shape[1], H + 2 * Hkv, -1).transpose(1, 2)
    return x.split((H, Hkv, Hkv), dim=1)


def _norm_rotate(x, w, cos, sin):
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    a, b = y.chunk(2, dim=-1)
    return torch.cat((a * cos + b * sin, b * cos - a * sin), dim=-1)


def _plain_qk(s):
    dt = s["qkv"].dtype
    x, qw, kw = (s[n].detach().float().requires_grad_(bool(s["train"]))
                 for n in ("qkv", "qw", "kw"))
    q, k, v = _heads(x, s["H"], s["Hkv"])
    out = (_norm_rotate(q, qw, s["cos"], s["sin"]), _norm_rotate(k, kw, s["cos"], s["sin"]), v)
    rounded = tuple(o.detach().to(dt).contiguous() for o in out)
    if not s["train"]:
        return rounded
    got = torch.autograd.grad(out, (x, qw, kw), tuple(d.float() for d in s["grads"]))
    return rounded, tuple(d.to(dt) for d in got)


def _plain_append(s):
    dt = s["qkv"].dtype
    q, k, v = _heads(s["qkv"].float(), s["H"], s["Hkv"])
    cos, sin = s["cos"][s["pos"]][:, None], s["sin"][s["pos"]][:, None]
    row = torch.arange(s["B"], device=q.device)[:, None]
    q, k = (_norm_rotate(q, s["qw"].float(), cos, sin), _norm_rotate(k, s["kw"].float(), cos, sin))
    s["kc"][row, :, s["pos"]] = k.to(dt).transpose(1, 2)
    s["vc"][row, :, s["pos"]] = v.to(dt).transpose(1, 2)
    return q.to(dt), s["kc"], s["vc"]


def _plain_embed(s):
    w, t = s["weight"].detach(), s["tokens"]
    out = (w[t].float() * s["scale"]).to(w.dtype)
    if not s["train"]:
        return out
    dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
    dw.index_add_(0, t, s["dy"].float() * s["scale"])
    if s["pad"] >= 0:
        dw[s["pad"]] = 0
    return out, (dw.to(w.dtype),)


def _plain_softmax(x):
    """(softmax, log of the sum of exponentials) over the last dimension; a
    row of -inf alone has the softmax 0."""
    m = x.amax(-1, keepdim=True).clamp_(min=torch.finfo(x.dtype).min)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    return e / total.clamp(min=torch.finfo(x.dtype).tiny), (m + torch.log(total)).squeeze(-1)


def _plain_distill(s):
    tau, alpha = s["tau"], s["alpha"]
    z = s["z"].detach().float()
    at = s["idx"].long()
    valid = at >= 0
    at = at.clamp(min=0)
    t = s["t"].float().masked_fill(~valid, -math.inf) / tau
    p, t_lse = _plain_softmax(t)
    taught = valid.any(-1)
    log_p = (t - t_lse[:, None]).masked_fill(~valid, 0)
    soft, soft_lse = _plain_softmax(z / tau)
    kd = (p * (log_p - z.gather(1, at) / tau + soft_lse[:, None])).sum(-1)
    counted = s["targets"] != IGNORE
    target = s["targets"].clamp(min=0)
    hard, hard_lse = _plain_softmax(z)
    ce = hard_lse - z.gather(1, target[:, None])[:, 0]
    rows = (alpha * tau * tau * kd + (1 - alpha) * ce) * counted
    if not s["train"]:
        return rows
    n = counted.sum()
    d = alpha * tau * taught[:, None] * soft + (1 - alpha) * hard
    d.scatter_add_(1, at, -alpha * tau * p)
    d.scatter_add_(1, target[:, None], torch.full_like(d[:, :1], alpha - 1))
    return rows.sum() / n, ((d * (counted / n)[:, None]).to(s["z"].dtype),)


def run(state):
    """One pass: (outputs, gradients) of a training case, outputs of the others."""
    if own:
        calls = dict(qk=_own_qk, append=_own_append, embed=_own_embed, distill=_own_distill)
    else:
        calls = dict(qk=_plain_qk, append=_plain_append, embed=_plain_embed,
                     distill=_plain_distill)
    return calls[state["kind"]](state)


# -------------------------------------------------------------- in 64 bits

def _exact_heads(case, s, x, w, cos, sin):
    """Rotated normed heads of x [B, T, heads, D] as [B, heads, T, D], and what
    the gradient needs of them."""
    r = 1 / torch.sqrt((x ** 2).sum(-1, keepdim=True) / case["D"] + EPS)
    y = w * x * r
    h = case["D"] // 2
    out = torch.empty_like(y)
    out[..., :h] = y[..., :h] * cos + y[..., h:] * sin
    out[..., h:] = y[..., h:] * cos - y[..., :h] * sin
    return out.transpose(1, 2).contiguous(), r


def _exact_heads_grad(case, d, x, r, w, cos, sin):
    d = d.double().transpose(1, 2)
    h = case["D"] // 2
    dy = torch.cat((d[..., :h] * cos - d[..., h:] * sin, d[..., h:] * cos + d[..., :h] * sin), -1)
    n = x * r
    gw = dy * w
    return r * (gw - n * (gw * n).mean(-1, keepdim=True)), (dy * n).sum((0, 1, 2))


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] in ("qk", "append"):
            B, H, Hkv, D = (case[n] for n in ("B", "H", "Hkv", "D"))
            x = s["qkv"].double().reshape(B, -1, H + 2 * Hkv, D)
            q, k, v = x[:, :, :H], x[:, :, H:H + Hkv], x[:, :, H + Hkv:]
            cos, sin = s["cos"].double(), s["sin"].double()
            if case["kind"] == "append":
                cos, sin = cos[s["pos"]], sin[s["pos"]]
            cos, sin = cos[..., None, :], sin[..., None, :]
            qw, kw = s["qw"].double(), s["kw"].double()
            (qo, qr), (ko, kr) = (_exact_heads(case, s, q, qw, cos, sin),
                                  _exact_heads(case, s, k, kw, cos, sin))
            vo = v.transpose(1, 2).contiguous()
            if case["kind"] == "append":
                kc, vc = s["kc"].double(), s["vc"].double()
                for b in range(B):
                    kc[b, :, s["pos"][b]] = ko[b]
                    vc[b, :, s["pos"][b]] = vo[b]
                return qo, kc, vc
            if not case["train"]:
                return qo, ko, vo
            dq, dk, dv = s["grads"]
            dx = torch.empty_like(x)
            dx[:, :, :H], dqw = _exact_heads_grad(case, dq, q, qr, qw, cos, sin)
            dx[:, :, H:H + Hkv], dkw = _exact_heads_grad(case, dk, k, kr, kw, cos, sin)
            dx[:, :, H + Hkv:] = dv.double().transpose(1, 2)
            return (qo, ko, vo), (dx.reshape(s["qkv"].shape), dqw, dkw)
        if case["kind"] == "embed":
            out = s["weight"].double().index_select(0, s["tokens"]).mul_(s["scale"])
            if not case["train"]:
                return out
            dw = torch.zeros(case["V"], case["C"], dtype=torch.float64, device=out.device)
            seen = s["tokens"] != case["pad"]
            dw.index_add_(0, s["tokens"][seen], s["dy"].double()[seen])
            return out, (dw.mul_(s["scale"]),)
        tau, alpha = case["tau"], case["alpha"]
        z, idx = s["z"].double(), s["idx"].long()
        N = case["N"]
        P = torch.zeros(N, case["V"] + 1, dtype=torch.float64, device=z.device)
        t = torch.where(idx >= 0, s["t"].double() / tau, -math.inf)
        p = torch.where((idx >= 0).any(-1, keepdim=True), torch.softmax(t, -1), 0.0)
        P.scatter_add_(1, torch.where(idx >= 0, idx, case["V"]), p)
        P = P[:, :-1]
        neg = torch.where(p > 0, p * p.clamp(min=1e-300).log(), 0.0).sum(-1)
        log_q = torch.log_softmax(z / tau, -1)
        rows = alpha * tau ** 2 * (neg - (P * log_q).sum(-1))
        counted = s["targets"] != IGNORE
        target = torch.where(counted, s["targets"], 0)[:, None]
        grad = (log_q.exp_() * (idx >= 0).any(-1, keepdim=True)).sub_(P).mul_(alpha * tau)
        del P, log_q
        log_s = torch.log_softmax(z, -1)
        rows = torch.where(counted, rows - (1 - alpha) * log_s.gather(1, target)[:, 0], 0.0)
        if not case["train"]:
            return rows
        grad.add_(log_s.exp_(), alpha=1 - alpha)
        grad[torch.arange(N, device=z.device), target[:, 0]] -= 1 - alpha
        n = counted.sum()
        return rows.sum() / n, (torch.where(counted[:, None], grad / n, 0.0),)


# ------------------------------------------------------------------ the work

def work(case):
    e = 2 if case["dtype"] == "bfloat16" else 4
    if case["kind"] in ("qk", "append"):
        n = case["B"] * (case["T"] if case["kind"] == "qk" else case["M"])
        wide = (case["H"] + 2 * case["Hkv"]) * case["D"]
        turned = (case["H"] + case["Hkv"]) * case["D"]
        rows = case["T"] if case["kind"] == "qk" else n
        passes = 2 if case["kind"] == "append" or not case["train"] else 4
        flops = (8 if passes == 2 else 28) * n * turned
        return {"bytes": passes * n * wide * e + rows * case["D"] * 4, "flops": flops}
    if case["kind"] == "embed":
        N, V, C = case["N"], case["V"], case["C"]
        distinct = float((-np.expm1(N * np.log1p(-_zipf(V)))).sum())
        once = 8 * N + (distinct + N) * C * e
        if not case["train"]:
            return {"bytes": once, "flops": N * C}
        return {"bytes": once + (N + V) * C * e, "flops": 3 * N * C}
    N, V, K = case["N"], case["V"], case["K"]
    slots = N * K * (e + (4 if e == 2 else 8)) + 8 * N
    once = N * V * e + slots
    if not case["train"]:
        return {"bytes": once + 4 * N, "flops": 4 * N * V}
    two = case["tau"] != 1.0 and case["alpha"] != 1.0
    return {"bytes": once + N * V * e, "flops": (14 if two else 8) * N * V}
