"""Timed workloads of the operators that long contexts add: the rotary
embedding in its forms (half-split or interleaved pairs, part of the head,
any position per token), attention with a sliding window and the first tokens
of a document that stay visible, and attention over a key/value cache held in
8 bits with a scale for each block of tokens and head.

A case is a dict of plain values; the tensors come from the seed that
``prepare`` gets.  With ``own`` the framework's operators run, without it the
same mathematics in elementary torch operations.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

BLOCK = 64          # cache positions that share a scale
LARGEST = 448.0     # of the 8-bit format (4 exponent bits, 3 mantissa bits)
LN2 = math.log(2.0)
FP8 = torch.float8_e4m3fn


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # The attention prologue of one layer of the 12-layer training step,
        # forward and backward; positions count from each document's start.
        dict(name="rot_train", kind="rotary", dtype="bfloat16", B=1, T=16384, H=12, Hkv=12, D=64,
             R=64, inter=0, pos="docs", train=1),
        # Grouped heads of 128 whose first half rotates, interleaved pairs, two
        # rows of an odd length.
        dict(name="rot_gqa_train", kind="rotary", dtype="bfloat16", B=2, T=4097, H=16, Hkv=2,
             D=128, R=64, inter=1, pos="range", train=1),
        # A short float32 row (a model that is not cast): latency.
        dict(name="rot_f32_small", kind="rotary", dtype="float32", B=1, T=513, H=8, Hkv=8, D=64,
             R=32, inter=1, pos="range", train=1),
        # One generated token, its position on the device: the smallest call.
        dict(name="rot_token", kind="rotary", dtype="bfloat16", B=1, T=1, H=12, Hkv=12, D=64,
             R=64, inter=0, pos="docs", train=0),
        # One layer's attention over a packed 16k row, a window of 1024 and
        # four first tokens; the step's mask and its tables too.
        dict(name="win_train", kind="window", dtype="bfloat16", B=1, T=16384, H=12, Hkv=12, D=64,
             docs=6, links=0, window=1024, sinks=4),
        # Grouped heads of 128 over linked documents: a link's grant is read
        # whole, the window bounds what a document reads of itself.
        dict(name="win_link_train", kind="window", dtype="bfloat16", B=2, T=4001, H=16, Hkv=4,
             D=128, docs=9, links=1, window=700, sinks=1),
        # A short float32 row.
        dict(name="win_f32_small", kind="window", dtype="float32", B=1, T=1000, H=4, Hkv=4, D=64,
             docs=3, links=0, window=128, sinks=2),
        # One generated token behind a long context, window over the cache.
        dict(name="win_token", kind="decode", B=1, M=1, H=12, Hkv=12, D=64, cap=32768, docs=1,
             links=0, window=4096, sinks=4),
        # One generated token into an 8-bit cache and its attention over it.
        dict(name="kv8_token", kind="kv8", B=1, M=1, H=12, Hkv=12, D=64, cap=4096, docs=4,
             links=1, window=0, sinks=0),
        # The same behind a long context.
        dict(name="kv8_long", kind="kv8", B=1, M=1, H=12, Hkv=12, D=64, cap=32768, docs=1,
             links=0, window=0, sinks=0),
        # A batch of sequences, grouped heads, two new tokens each.
        dict(name="kv8_batch", kind="kv8", B=16, M=2, H=32, Hkv=8, D=128, cap=8192, docs=1,
             links=0, window=0, sinks=0),
        # A prompt's keys and values into the cache.
        dict(name="kv8_prompt", kind="prompt", B=1, M=16384, Hkv=12, D=64, cap=16384),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(12, 12, 64), (8, 8, 64), (4, 4, 128), (16, 2, 128), (16, 4, 64), (6, 3, 64), (1, 1, 64),
         (32, 8, 128)]


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "window", "window", "decode", "kv8", "kv8", "prompt"])
    H, Hkv, D = rng.choice(HEADS)
    if kind == "rotary":
        B = rng.choice([1, 2, 3])
        return dict(kind=kind, dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), B=B,
                    T=_log_int(rng, 1, 8192 // B), H=H, Hkv=Hkv, D=D,
                    R=rng.choice([D, D // 2, 16 * rng.randint(1, D // 16)]),
                    inter=rng.choice([0, 1]), pos=rng.choice(["docs", "range"]),
                    train=rng.choice([0, 1, 1]))
    docs, links = rng.choice([(1, 0), (rng.randint(2, 12), 0), (rng.randint(2, 12), 1)])
    window = rng.choice([0, 1, _log_int(rng, 2, 4096), _log_int(rng, 2, 4096)])
    sinks = rng.choice([0, 1, 4, rng.randint(1, 200)]) if window else 0
    if kind == "window":
        B = rng.choice([1, 1, 2])
        return dict(kind=kind, dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), B=B,
                    T=_log_int(rng, 32, 4096 // B), H=H, Hkv=Hkv, D=D, docs=docs, links=links,
                    window=max(window, 2), sinks=sinks)  # some row sees two keys
    if kind == "prompt":
        M = _log_int(rng, 1, 8192)
        return dict(kind=kind, B=rng.choice([1, 2]), M=M, Hkv=Hkv, D=D,
                    cap=M + rng.randint(0, 300))
    most = 8 if kind == "decode" else 16
    M = rng.choice([1, 1, rng.randint(1, most // (H // Hkv))])
    B = rng.choice([1, 2, 5, 8])
    return dict(kind=kind, B=B, M=M, H=H, Hkv=Hkv, D=D, cap=_log_int(rng, 16, 32768 // B),
                docs=docs, links=links, window=window, sinks=sinks)


# -------------------------------------------------------------------- inputs

def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _spans(n, docs):
    """Start of each of `docs` documents of uneven lengths that fill n
    positions (fewer where n is short)."""
    w = np.array([1.0 + 2.5 * ((7 * i + 3) % 5) / 4 for i in range(docs)])
    cut = np.floor(np.concatenate(([0.0], np.cumsum(w)[:-1])) / w.sum() * n).astype(np.int64)
    return np.unique(cut)


def _documents(n, docs):
    """Document of every position, int64 [n]."""
    return np.searchsorted(_spans(n, docs), np.arange(n), side="right") - 1


def _granted(docs):
    """Word of the documents that each document's links grant: two of the
    earlier ones."""
    return [sum(1 << j for j in {(5 * i) % i, i // 2}) if i else 0 for i in range(docs)]


def _starts(case):
    """First new token's position of each sequence of a generation case."""
    last = case["cap"] - case["M"]
    return [last - (37 * b + 11) % (last // 8 + 1) for b in range(case["B"])]


def _tables(rows, R, dev):
    """cos / sin of position / 4 * 10000^(-i / (R / 2)), float32 [rows, R / 2]:
    positions interpolated for a context four times the trained one."""
    inv = 10000.0 ** (-torch.arange(R // 2, dtype=torch.float64) / (R // 2))
    ang = torch.outer(torch.arange(rows, dtype=torch.float64) / 4, inv)
    return ang.cos().float().to(dev), ang.sin().float().to(dev)


def _signed(word):
    return word - (1 << 64) if word >> 63 else word


def _mask_inputs(s, case, n, dev):
    doc = _documents(n, case["docs"])
    s["doc"] = torch.from_numpy(doc.astype(np.int32)).to(dev)[None]
    s["qb"] = s["kb"] = None
    if case["links"]:
        grant = _granted(case["docs"])
        s["qb"] = torch.tensor([[[_signed(grant[d]) for d in doc]]], device=dev)
        s["kb"] = torch.tensor([[[_signed(1 << int(d)) for d in doc]]], device=dev)


def _encode(x, scale):
    """8-bit codes of x / scale (float32; scale a power of two)."""
    return (x / scale).to(FP8)


def _block_scale(amax):
    """Power of two s with amax / s <= 448 and amax / s > 224."""
    m, e = torch.frexp(amax)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(-120, 120)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e, -120))


def prepare(case, seed):
    dev = _device()
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = getattr(torch, case.get("dtype", "bfloat16"))

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=dev)

    s = dict(case)
    kind = case["kind"]
    if kind == "rotary":
        B, T, H, Hkv, D = (case[n] for n in ("B", "T", "H", "Hkv", "D"))
        rows = max(T, 64)
        s["cos"], s["sin"] = _tables(rows, case["R"], dev)
        s["qkv"] = (randn(B, T, (H + 2 * Hkv) * D) * (0.5 + 2 * rand(B, T, 1))).to(dt)
        s["at"] = 0
        if case["pos"] == "docs":
            if T <= 8:  # new tokens behind their contexts
                first = (rand(B, 1) * (rows - T + 1)).long().clamp_(max=rows - T)
                s["at"] = first + torch.arange(T, device=dev)
            else:
                start = _spans(T, 7)
                at = np.arange(T) - start[np.searchsorted(start, np.arange(T), side="right") - 1]
                s["at"] = torch.from_numpy(at).to(dev)
        if case["train"]:
            s["grads"] = tuple(randn(B, h, T, D).to(dt) for h in (H, Hkv, Hkv))
            s["qkv"].requires_grad_(True)
        return s
    if kind == "window":
        B, T, H, Hkv, D = (case[n] for n in ("B", "T", "H", "Hkv", "D"))
        _mask_inputs(s, case, T, dev)
        s["q"], s["k"], s["v"] = (randn(B, h, T, D).to(dt).requires_grad_(True)
                                  for h in (H, Hkv, Hkv))
        s["do"] = randn(B, H, T, D).to(dt)
        return s
    B, M, Hkv, D, cap = (case[n] for n in ("B", "M", "Hkv", "D", "cap"))
    # channels of different sizes, as keys have them
    wide = (0.3 + 2 * rand(1, Hkv, 1, D) ** 4)
    if kind in ("decode", "kv8"):
        _mask_inputs(s, case, cap, dev)
        s["q"] = (0.5 * randn(B, case["H"], M, D)).to(dt)
        pos = np.array(_starts(case))[:, None] + np.arange(M)
        doc = _documents(cap, case["docs"])
        start = _spans(cap, case["docs"])[doc]
        s["pos"], s["qdoc"], s["qstart"] = (torch.from_numpy(x.astype(np.int32)).to(dev)
                                            for x in (pos, doc[pos], start[pos]))
        s["doc"] = s["doc"].repeat(B, 1)
        if case["links"]:
            s["kb"] = s["kb"].repeat(B, 1, 1)
            s["qrow"] = s["qb"][0, :, s["pos"].long()].transpose(0, 1).contiguous()
        else:
            s["qrow"] = None
    if kind == "decode":
        s["kc"], s["vc"] = ((randn(B, Hkv, cap, D) * wide).to(dt) for _ in range(2))
        return s
    s["k"], s["v"] = ((randn(B, Hkv, M, D) * wide).to(dt) for _ in range(2))
    nb = -(-cap // BLOCK)
    if kind == "prompt":
        s["at"] = 0
        s["kc"] = torch.zeros(B, Hkv, nb, BLOCK, D, device=dev).to(FP8)
        s["vc"] = torch.zeros(B, Hkv, nb, D, BLOCK, device=dev).to(FP8)
        s["ks"], s["vs"] = (torch.zeros(B, Hkv, nb, device=dev) for _ in range(2))
        return s
    s["at"] = s["pos"][:, 0].long()
    for c, sc, turn in (("kc", "ks", False), ("vc", "vs", True)):
        x = randn(B, Hkv, nb, BLOCK, D) * wide[:, :, None]
        s[sc] = _block_scale(x.abs().amax((-1, -2)))
        x = _encode(x, s[sc][..., None, None])
        s[c] = x.view(torch.uint8).transpose(-1, -2).contiguous().view(FP8) if turn else x
    return s


# ------------------------------------------------------- the framework's calls

def _own_rotary(s):
    from tagseq2tagseq_amd.rope import qkv_rotary
    out = qkv_rotary(s["qkv"], s["cos"], s["sin"], s["H"], num_kv_heads=s["Hkv"], pos=s["at"],
                     interleaved=bool(s["inter"]))
    if not s["train"]:
        return out
    return out, torch.autograd.grad(out, s["qkv"], s["grads"])


def _own_window(s):
    from tagseq2tagseq_amd.attention import flex_attention
    from tagseq2tagseq_amd.block_mask import build_block_mask
    bm = build_block_mask(s["doc"], s["qb"], s["kb"], window=s["window"], sinks=s["sinks"])
    out = flex_attention(s["q"], s["k"], s["v"], block_mask=bm, enable_gqa=True)
    return out, torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["do"])


def _own_decode(s):
    from tagseq2tagseq_amd.decode import attn_decode
    return attn_decode(s["q"], s["kc"], s["vc"], s["cap"], s["doc"], s["kb"], s["pos"], s["qdoc"],
                       s["qrow"], window=s["window"] or None, sinks=s["sinks"],
                       q_start=s["qstart"] if s["sinks"] else None)


def _own_prompt(s):
    from tagseq2tagseq_amd.kv8 import kv8_append
    kv8_append(s["k"], s["v"], s["at"], s["kc"], s["vc"], s["ks"], s["vs"])
    return s["kc"], s["vc"], s["ks"], s["vs"]


def _own_kv8(s):
    from tagseq2tagseq_amd.kv8 import attn_decode_kv8, kv8_append
    kv8_append(s["k"], s["v"], s["at"], s["kc"], s["vc"], s["ks"], s["vs"])
    o, lse2 = attn_decode_kv8(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["cap"], s["doc"],
                              s["kb"], s["pos"], s["qdoc"], s["qrow"],
                              window=s["window"] or None, sinks=s["sinks"],
                              q_start=s["qstart"] if s["sinks"] else None)
    return o, lse2, s["kc"], s["vc"], s["ks"], s["vs"]


# ------------------------------------------------------------ the plain forms

def _turn(x, cos, sin, R, inter, back=False):
    """Heads x [..., D] with the first R dimensions rotated (back: by the
    angles' negatives)."""
    if back:
        sin = -sin
    r, rest = x[..., :R], x[..., R:]
    if inter:
        a, b = r[..., 0::2], r[..., 1::2]
        return torch.cat((torch.stack((a * cos + b * sin, b * cos - a * sin), -1).flatten(-2),
                          rest), -1)
    a, b = r[..., :R // 2], r[..., R // 2:]
    return torch.cat((a * cos + b * sin, b * cos - a * sin, rest), -1)


def _plain_rotary(s):
    dt, (H, Hkv, R, inter) = s["qkv"].dtype, (s[n] for n in ("H", "Hkv", "R", "inter"))
    B, T = s["qkv"].shape[:2]
    x = s["qkv"].detach().float().view(B, T, H + 2 * Hkv, -1).transpose(1, 2)
    at = s["at"] if torch.is_tensor(s["at"]) else torch.arange(T, device=x.device) + s["at"]
    cos, sin = s["cos"][at], s["sin"][at]
    if at.dim() == 2:
        cos, sin = cos[:, None], sin[:, None]
    q, k, v = x.split((H, Hkv, Hkv), dim=1)
    out = tuple(t.to(dt).contiguous() for t in (_turn(q, cos, sin, R, inter),
                                                _turn(k, cos, sin, R, inter), v))
    if not s["train"]:
        return out
    dq, dk, dv = (d.float() for d in s["grads"])
    d = torch.cat((_turn(dq, cos, sin, R, inter, True), _turn(dk, cos, sin, R, inter, True), dv), 1)
    return out, (d.transpose(1, 2).reshape(B, T, -1).to(dt),)


def _visible(q_pos, q_doc, q_start, q_bits, j, k_doc, k_bits, window, sinks):
    """Truth of (query row, key position) pairs: q_* [B, Tq], k_* [B, n], bits
    with a dimension of words in front of the last."""
    far = q_pos[:, :, None] - j
    near = q_doc[:, :, None] == k_doc[:, None, :]
    if window:
        seen = far < window
        if sinks:
            at = j - q_start[:, :, None]
            seen |= (at >= 0) & (at < sinks)
        near &= seen
    if q_bits is not None:
        near |= ((q_bits[:, :, :, None] & k_bits[:, :, None, :]) != 0).any(1)
    return near & (far >= 0)


def _plain_window(s):
    dt, (B, T, H, Hkv, D) = s["q"].dtype, (s[n] for n in ("B", "T", "H", "Hkv", "D"))
    q, k, v, do = (s[n].detach().float() for n in ("q", "k", "v", "do"))
    k, v = (x.repeat_interleave(H // Hkv, 1) for x in (k, v))
    at = torch.arange(T, device=q.device)
    doc = s["doc"]
    new = torch.ones_like(doc, dtype=torch.bool)
    new[:, 1:] = doc[:, 1:] != doc[:, :-1]
    start = torch.where(new, at, 0).cummax(-1).values
    ok = _visible(at[None], doc, start, s["qb"], at, doc, s["kb"], s["window"], s["sinks"])[:, None]
    p = (q @ k.transpose(2, 3).contiguous()).mul_(D ** -0.5).masked_fill_(~ok, -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    p /= p.sum(-1, keepdim=True)
    out = p @ v
    dv = p.transpose(2, 3) @ do
    ds = do @ v.transpose(2, 3).contiguous()
    ds -= (do * out).sum(-1, keepdim=True)
    ds *= p
    del p
    ds *= D ** -0.5
    dq = ds @ k
    dk = ds.transpose(2, 3) @ q
    dk, dv = (x.view(B, Hkv, H // Hkv, T, D).sum(2) for x in (dk, dv))
    return out.to(dt), tuple(x.to(dt) for x in (dq, dk, dv))


def _plain_attend(s, k, v):
    """(o, lse2) of the new rows over k, v [B, Hkv, n, D] in float32."""
    B, H, M, D = s["q"].shape
    n, G = k.shape[2], H // k.shape[1]
    ok = _visible(s["pos"], s["qdoc"], s["qstart"], s["qrow"], torch.arange(n, device=k.device),
                  s["doc"][:, :n], None if s["kb"] is None else s["kb"][:, :, :n], s["window"],
                  s["sinks"])
    q = s["q"].float().view(B, -1, G * M, D)
    p = (q @ k.transpose(2, 3).contiguous()).view(B, H, M, n) * D ** -0.5
    p = p.masked_fill_(~ok[:, None], -math.inf)
    m = p.amax(-1, keepdim=True).clamp_(min=torch.finfo(p.dtype).min)
    p = torch.exp(p - m)
    total = p.sum(-1, keepdim=True)
    o = (p.view(B, -1, G * M, n) @ v).view(B, H, M, D) / total.clamp(min=1e-30)
    return o.to(s["q"].dtype), ((m + torch.log(total)) / LN2).squeeze(-1)


def _plain_decode(s):
    return _plain_attend(s, s["kc"].float(), s["vc"].float())


def _store(x, at, codes, scale, turn):
    """M new tokens x [B, Hkv, M, D] at positions at[b] .. at[b] + M - 1 of
    codes [B, Hkv, nb, 64, D] ([.., D, 64] with turn).  A block's scale grows to
    what its new tokens need; the tokens before them in the block are
    written again under it."""
    B, Hkv, M, D = x.shape
    blocks = (M + BLOCK - 2) // BLOCK + 1
    blk = at[:, None] // BLOCK + torch.arange(blocks, device=x.device)
    slot = (blk * BLOCK)[..., None] + torch.arange(BLOCK, device=x.device) - at[:, None, None]
    touched = ((slot >= 0) & (slot < M)).any(-1)
    b, i = touched.nonzero(as_tuple=True)
    blk, slot = blk[b, i], slot[b, i]                          # [n], [n, 64]
    raw = codes.view(torch.uint8)[b, :, blk]
    raw = raw.transpose(-1, -2) if turn else raw               # [n, Hkv, 64, D]
    fresh = ((slot >= 0) & (slot < M))[:, None, :, None]
    kept = (slot < 0)[:, None, :, None]
    new = x.float()[b[:, None], :, slot.clamp(0, M - 1)].transpose(1, 2)
    was = torch.where(kept.any(-2).squeeze(-1), scale[b, :, blk], 0)
    now = torch.maximum(was, _block_scale((new.abs() * fresh).amax((-1, -2))))
    old = raw.contiguous().view(FP8).float() * (was / now)[..., None, None]
    put = torch.where(fresh, new / now[..., None, None], old).to(FP8).view(torch.uint8)
    put = torch.where(fresh | kept, put, raw)
    codes.view(torch.uint8)[b, :, blk] = put.transpose(-1, -2) if turn else put
    scale[b, :, blk] = now


def _plain_prompt(s):
    at = s["at"] if torch.is_tensor(s["at"]) else torch.full((s["B"],), s["at"],
                                                             device=s["k"].device)
    _store(s["k"], at, s["kc"], s["ks"], False)
    _store(s["v"], at, s["vc"], s["vs"], True)
    return s["kc"], s["vc"], s["ks"], s["vs"]


def _plain_kv8(s):
    _plain_prompt(s)
    k = (s["kc"].float() * s["ks"][..., None, None]).flatten(2, 3)[:, :, :s["cap"]]
    v = (s["vc"].float() * s["vs"][..., None, None]).transpose(3, 4).flatten(2, 3)[:, :, :s["cap"]]
    return *_plain_attend(s, k, v), s["kc"], s["vc"], s["ks"], s["vs"]


def run(state):
    """One pass: (outputs, gradients) of a training case, outputs of the others
    (a cache's codes as the 8-bit numbers that they are)."""
    if own:
        calls = dict(rotary=_own_rotary, window=_own_window, decode=_own_decode, kv8=_own_kv8,
                     prompt=_own_prompt)
    else:
        calls = dict(rotary=_plain_rotary, window=_plain_window, decode=_plain_decode,
                     kv8=_plain_kv8, prompt=_plain_prompt)
    return calls[state["kind"]](state)


# -------------------------------------------------------------- in 64 bits

def _exact_rotary(case, s):
    B, T, H, Hkv, D, R = (case[n] for n in ("B", "T", "H", "Hkv", "D", "R"))
    at = s["at"] if torch.is_tensor(s["at"]) else torch.arange(T, device=s["qkv"].device)
    at = at.expand(B, T)
    first = torch.arange(0, R, 2) if case["inter"] else torch.arange(R // 2)
    second = first + (1 if case["inter"] else R // 2)
    # every pair (x, y) as the complex number x + iy, turned by -angle
    turn = torch.complex(s["cos"].double(), -s["sin"].double())[at][:, :, None]

    def rotate(x, by):
        z = torch.complex(x[..., first], x[..., second]) * by
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    x = s["qkv"].detach().double().reshape(B, T, H + 2 * Hkv, D)
    y = torch.cat((rotate(x[:, :, :H + Hkv], turn), x[:, :, H + Hkv:]), 2).transpose(1, 2)
    out = tuple(t.contiguous() for t in (y[:, :H], y[:, H:H + Hkv], y[:, H + Hkv:]))
    if not case["train"]:
        return out
    d = torch.cat([t.double().transpose(1, 2) for t in s["grads"]], 2)
    d = torch.cat((rotate(d[:, :, :H + Hkv], turn.conj()), d[:, :, H + Hkv:]), 2)
    return out, (d.reshape(B, T, -1),)


def _exact_row_mask(case, n, q_pos):
    """[len(q_pos), n] truth, row by row from the documents' spans."""
    first = _spans(n, case["docs"])
    last = np.append(first[1:], n)
    grant = _granted(case["docs"])
    ok = np.zeros((len(q_pos), n), dtype=bool)
    for r, p in enumerate(q_pos):
        d = int(np.nonzero(first <= p)[0][-1])
        lo = first[d]
        if case["window"]:
            ok[r, max(lo, p - case["window"] + 1):p + 1] = True
            ok[r, lo:min(lo + case["sinks"], p + 1)] = True
        else:
            ok[r, lo:p + 1] = True
        if case["links"]:
            for e in range(d):
                if grant[d] >> e & 1:
                    ok[r, first[e]:last[e]] = True
    return ok


def _exact_window(case, s):
    B, T, H, Hkv, D = (case[n] for n in ("B", "T", "H", "Hkv", "D"))
    ok = torch.from_numpy(_exact_row_mask(case, T, range(T))).to(s["q"].device)
    q, k, v, do = (s[n].detach().double() for n in ("q", "k", "v", "do"))
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    for b in range(B):
        for h in range(H):
            e = h * Hkv // H
            w = q[b, h] @ k[b, e].t().contiguous() / math.sqrt(D)
            w = torch.softmax(w.masked_fill_(~ok, -math.inf), -1)
            out[b, h] = w @ v[b, e]
            dv[b, e] += w.t() @ do[b, h]
            g = do[b, h] @ v[b, e].t().contiguous()
            g = w * (g - (w * g).sum(-1, keepdim=True)) / math.sqrt(D)
            dq[b, h] = g @ k[b, e]
            dk[b, e] += g.t() @ q[b, h]
    return out, (dq, dk, dv)


def _exact_rows(case, s, k, v):
    """(o, lse2) over k, v [B, Hkv, n, D] of doubles."""
    B, M, H, Hkv, D = (case[n] for n in ("B", "M", "H", "Hkv", "D"))
    o = torch.zeros(B, H, M, D, dtype=torch.float64, device=k.device)
    lse2 = torch.full((B, H, M), -math.inf, dtype=torch.float64, device=k.device)
    for b, first in enumerate(_starts(case)):
        ok = _exact_row_mask(case, case["cap"], range(first, first + M))
        for t in range(M):
            j = torch.from_numpy(np.nonzero(ok[t])[0]).to(k.device)
            kj, vj = (x[b].index_select(1, j) for x in (k, v))
            kj, vj = (x.repeat_interleave(H // Hkv, 0) for x in (kj, vj))
            w = (kj * s["q"][b, :, t, None].double()).sum(-1) / math.sqrt(D)
            lse2[b, :, t] = torch.logsumexp(w, -1) / LN2
            o[b, :, t] = (torch.softmax(w, -1)[..., None] * vj).sum(1)
    return o, lse2


def _exact_code(x):
    """The number of 3 mantissa bits nearest to x, ties to the even one
    (exponents from -6; |x| <= 448)."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -20))).clamp(min=-6)
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _exact_store(case, s, x, codes, scale, turn):
    """(numbers that the codes stand for before their scale, laid out as they
    are; scales) after the append."""
    M = case["M"]
    c = codes.float().double()
    c = c.transpose(-1, -2).clone() if turn else c
    sc = scale.double().clone()
    for b, first in enumerate([0] * case["B"] if case["kind"] == "prompt" else _starts(case)):
        for blk in range(first // BLOCK, (first + M - 1) // BLOCK + 1):
            lo, hi = max(first, blk * BLOCK), min(first + M, (blk + 1) * BLOCK)
            new = x[b, :, lo - first:hi - first].double()
            top = new.abs().amax((-1, -2))
            need = torch.where(top > 0, torch.exp2(torch.ceil(torch.log2(top / LARGEST))), 0.0)
            need = need.clamp(min=2.0 ** -120)
            n = lo - blk * BLOCK
            now = torch.maximum(sc[b, :, blk], need) if n else need
            if n:
                c[b, :, blk, :n] = _exact_code(c[b, :, blk, :n] *
                                               (sc[b, :, blk] / now)[:, None, None])
            c[b, :, blk, n:n + hi - lo] = _exact_code(new / now[:, None, None])
            sc[b, :, blk] = now
    return c, sc


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "rotary":
            return _exact_rotary(case, s)
        if case["kind"] == "window":
            return _exact_window(case, s)
        if case["kind"] == "decode":
            return _exact_rows(case, s, s["kc"].double(), s["vc"].double())
        kc, ks = _exact_store(case, s, s["k"], s["kc"], s["ks"], False)
        vc, vs = _exact_store(case, s, s["v"], s["vc"], s["vs"], True)
        state = kc, vc.transpose(-1, -2).contiguous(), ks, vs
        if case["kind"] == "prompt":
            return state
        k, v = ((c * sc[..., None, None]).flatten(2, 3) for c, sc in ((kc, ks), (vc, vs)))
        return *_exact_rows(case, s, k, v), *state


# ------------------------------------------------------------------ the work

def _pairs(case, n, q_pos):
    """(visible pairs, positions that some row sees) of the rows q_pos."""
    first = _spans(n, case["docs"])
    last = np.append(first[1:], n)
    grant = _granted(case["docs"])
    pairs, seen = 0, np.zeros(n + 1, dtype=np.int64)
    for p in q_pos:
        d = int(np.searchsorted(first, p, side="right")) - 1
        lo = int(first[d])
        parts = [(lo, p + 1)]
        if case["window"]:
            near = max(lo, p - case["window"] + 1)
            parts = [(near, p + 1), (lo, min(lo + case["sinks"], near))]
        if case["links"]:
            parts += [(int(first[e]), int(last[e])) for e in range(d) if grant[d] >> e & 1]
        for a, z in parts:
            if z > a:
                pairs += z - a
                seen[a] += 1
                seen[z] -= 1
    return pairs, int((np.cumsum(seen) > 0).sum())


def work(case):
    kind = case["kind"]
    e = 4 if case.get("dtype") == "float32" else 2
    if kind == "rotary":
        B, T, H, Hkv, D, R = (case[n] for n in ("B", "T", "H", "Hkv", "D", "R"))
        passes = 4 if case["train"] else 2
        rows = B * T if case["pos"] == "docs" and T <= 8 else T
        return {"bytes": passes * B * T * (H + 2 * Hkv) * D * e + rows * R * 4,
                "flops": passes // 2 * 3 * B * T * (H + Hkv) * R}
    if kind == "window":
        B, T, H, Hkv, D = (case[n] for n in ("B", "T", "H", "Hkv", "D"))
        pairs, _ = _pairs(case, T, range(T))
        # read q, k, v, dO; written out, dq, dk, dv
        return {"bytes": (4 * H + 4 * Hkv) * B * T * D * e + 4 * T, "flops": 14 * B * H * pairs * D}
    B, M, Hkv, D, cap = (case[n] for n in ("B", "M", "Hkv", "D", "cap"))
    if kind == "prompt":
        blocks = -(-M // BLOCK)
        return {"bytes": B * Hkv * (2 * M * D * 3 + 8 * blocks), "flops": 4 * B * Hkv * M * D}
    pairs = seen = 0
    for p in _starts(case):
        a, z = _pairs(case, cap, range(p, p + M))
        pairs, seen = pairs + a, seen + z
    H = case["H"]
    rows = B * H * M
    if kind == "decode":
        return {"bytes": seen * (4 * Hkv * D + 4) + rows * (4 * D + 4), "flops": 4 * H * pairs * D}
    new = B * Hkv * M * D
    return {"bytes": seen * (2 * Hkv * D + 4) + seen * Hkv * 8 // BLOCK + 6 * new +
            rows * (4 * D + 4), "flops": 4 * H * pairs * D}
