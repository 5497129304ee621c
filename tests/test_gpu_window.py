"""GPU checks of the sliding window with sinks: the mask's tables and bitmaps
against the dense mask, the attention over them, and the decode step, against
plain implementations in 64 bits.
"""
import math

import numpy as np
import pytest
import torch

from oracle import mask_oracle as mo
from tagseq2tagseq_amd import synth
from tagseq2tagseq_amd.attention import flex_attention
from tagseq2tagseq_amd.block_mask import build_block_mask, doc_starts, mask_inputs
from tagseq2tagseq_amd.decode import attn_decode
from tagseq2tagseq_amd.mask_creators import (CrossDocLinkMaskCreator, SlidingWindowMaskCreator,
                                             create_causal_block_mask,
                                             create_doc_causal_block_mask,
                                             create_doc_link_block_mask,
                                             make_mask_creator_callable)
from tagseq2tagseq_amd.model import TS2TSModel
from tagseq2tagseq_amd.modules import TS2TSTrainingModule
from tagseq2tagseq_amd.rope import RotaryForm
from tests.helpers import TABLES, random_row, to_dev_words

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
U = 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32


def _starts(doc):
    s = np.zeros(len(doc), dtype=np.int32)
    for t in range(1, len(doc)):
        s[t] = s[t - 1] if doc[t] == doc[t - 1] else t
    return s


def _dense(doc, qb, kb, window, sinks, rows=None):
    """[rows, T] truth of the mask, from its definition."""
    T = len(doc)
    q = np.arange(T)[:, None] if rows is None else np.asarray(rows)[:, None]
    k = np.arange(T)[None]
    ok = doc[q[:, 0]][:, None] == doc[None]
    if window is not None:
        at = k - _starts(doc)[q[:, 0]][:, None]
        ok &= (q - k < window) | ((at >= 0) & (at < sinks))
    if qb is not None:
        for w in range(qb.shape[0]):
            ok |= (qb[w][q[:, 0]][:, None] & kb[w][None]) != 0
    return ok & (q >= k)


def _row(T, seed, words, max_doc):
    return random_row(T, np.random.default_rng(seed), words=words, uncovered=True, max_doc=max_doc)


def _build(rows, window, sinks):
    doc = torch.stack([torch.from_numpy(r[0]) for r in rows]).to(DEV)
    qb = kb = None
    if rows[0][1] is not None:
        qb = torch.stack([to_dev_words(r[1], DEV) for r in rows])
        kb = torch.stack([to_dev_words(r[2], DEV) for r in rows])
    return build_block_mask(doc, qb, kb, window=window, sinks=sinks)


def _check_tables(bm, rows, window, sinks):
    for b, (doc, qb, kb) in enumerate(rows):
        T = len(doc)
        nt = (T + 127) // 128
        dense = np.zeros((nt * 128, nt * 128), dtype=bool)
        dense[:T, :T] = _dense(doc, qb, kb, window, sinks)
        tiles = dense.reshape(nt, 128, nt, 128).transpose(0, 2, 1, 3)
        counts = tiles.sum((2, 3))
        ref = mo.block_mask_tables(doc, qb, kb, counts=counts)
        np.testing.assert_array_equal(bm.tile_class[b].cpu().numpy(),
                                      (counts > 0) + 1 * (counts == 128 * 128))
        for name in TABLES:
            np.testing.assert_array_equal(getattr(bm, name)[b, 0].cpu().numpy(), ref[name], name)
        off = bm.kv_bits_off[b].cpu().numpy()
        bits = bm.tile_bits.cpu().numpy().view("<u4")
        pack = lambda m: np.packbits(m, axis=1, bitorder="little").view("<u4").reshape(128, 4)  # noqa
        for r, c in zip(*np.nonzero((counts > 0) & (counts < 128 * 128))):
            np.testing.assert_array_equal(bits[off[r] + c, 0], pack(tiles[r, c]), f"rows {r} {c}")
            np.testing.assert_array_equal(bits[off[r] + c, 1], pack(tiles[r, c].T.copy()),
                                          f"columns {r} {c}")


@pytest.mark.parametrize("T", [1, 255, 256, 257, 1000, 4096, 4353, 20001])
def test_doc_starts(T):
    rng = np.random.default_rng(T)
    rows = [np.full(T, 3, dtype=np.int32), np.arange(T, dtype=np.int32) // 2,
            np.repeat(rng.integers(0, 3, T), 1 + rng.integers(0, 9000, T))[:T].astype(np.int32)]
    got = doc_starts(torch.from_numpy(np.stack(rows)).to(DEV)).cpu().numpy()
    for g, doc in zip(got, rows):
        np.testing.assert_array_equal(g, _starts(doc))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (5, 0), (64, 1), (127, 130), (128, 0),
                                          (129, 4), (300, 7), (4000, 2)])
@pytest.mark.parametrize("T,words,max_doc", [(1, 0, 5), (130, 0, 400), (700, 0, 900),
                                             (600, 1, 60), (1025, 3, 500), (400, 8, 3)])
def test_tables_and_bitmaps(T, words, max_doc, window, sinks):
    rows = [_row(T, 17 * T + i, words, max_doc) for i in range(2)]
    bm = _build(rows, window, sinks)
    assert (bm.window, bm.sinks) == (window, sinks) and (bm.doc_start is not None) == bool(sinks)
    _check_tables(bm, rows, window, sinks)


def test_documents_that_come_back():
    """One id in two runs: the window spans both, sinks are the own run's."""
    doc = np.repeat(np.array([4, 9, 4, 4, 2, 9], dtype=np.int32), [100, 3, 40, 90, 1, 200])
    for window, sinks in ((50, 3), (150, 0), (2, 60)):
        _check_tables(_build([(doc, None, None)], window, sinks), [(doc, None, None)], window, sinks)


@pytest.mark.parametrize("window", [1000, 2 ** 31 - 1, 2 ** 40])
def test_a_window_past_the_row_is_none(window):
    rows = [_row(1000, 5, 2, 300)]
    a, b = _build(rows, window, 2 ** 33), _build(rows, None, 0)
    for x, y in zip([a.tile_class, *a.tables()[:11]], [b.tile_class, *b.tables()[:11]]):
        assert torch.equal(x, y)
    _check_tables(a, rows, None, 0)


def test_mask_mod_and_torch_block_mask():
    rows = [_row(300, 8, 1, 200)]
    bm = _build(rows, 40, 3)
    dense = torch.from_numpy(_dense(*rows[0], 40, 3)).to(DEV)
    i = torch.arange(300, device=DEV)
    got = bm.mask_mod()(torch.zeros((), dtype=torch.long, device=DEV), 0, i[:, None], i[None])
    assert torch.equal(got, dense)
    assert torch.equal(bm.to_block_mask().kv_num_blocks, bm.kv_num_blocks)


# ---- attention

def _attention_ref(q, k, v, do, dense, r):
    """(o, dq, dk, dv) in 64 bits and what each may be off by.

    r is half a step of the operands' type where the kernels round to it (p and
    ds before their second products, o before it is stored and before the
    backward takes sum(o do) of it, every result), 0 for float32.  a bounds the
    fp32 arithmetic relative to sums of absolute values: a score is a chain of
    D products, S = max sum |q k| / sqrt(D) of them, twice in p; sums over T
    terms in chains of at most T / 16 + 32."""
    G, D = q.shape[1] // k.shape[1], q.shape[-1]
    q, k, v, do = (t.detach().double() for t in (q, k, v, do))
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    t = lambda x: x.transpose(2, 3).contiguous()  # noqa: E731
    c = D ** -0.5
    S = float((q.abs() @ t(k.abs())).max()) * c
    a = (2 * (D + 8) * max(S, 1.0) + q.shape[2] / 16 + 32) * U
    p = torch.softmax((q @ t(k) * c).masked_fill(~dense[:, None], -math.inf), -1)
    o = p @ v
    o_big = p @ v.abs()
    o_tol = (r + a) * o_big + r * o.abs()
    ds = p * (do @ t(v) - (do * o).sum(-1, keepdim=True))
    delta = ((o_tol + a * o_big) * do.abs()).sum(-1, keepdim=True)
    ds_tol = p * (delta + a * (do.abs() @ t(v.abs()))) + (r + a) * ds.abs()
    fold = lambda x: x.view(x.shape[0], -1, G, *x.shape[2:]).sum(2)  # noqa: E731
    dq, dk, dv = c * (ds @ k), c * fold(t(ds) @ q), fold(t(p) @ do)
    tols = (o_tol, c * (ds_tol @ k.abs()), c * fold(t(ds_tol) @ q.abs()),
            (r + a) * fold(t(p) @ do.abs()))
    # (second order: 1% more)
    return [(x, 1.01 * e + (r + a) * x.abs() + 1e-30) for x, e in zip((o, dq, dk, dv), tols)]


@pytest.mark.parametrize("dtype,B,T,H,Hkv,D,words,window,sinks", [
    (BF, 1, 1, 2, 2, 64, 0, 1, 0), (BF, 1, 129, 2, 1, 128, 0, 1, 1), (BF, 2, 700, 4, 2, 64, 1, 64, 3),
    (BF, 1, 1300, 4, 4, 64, 0, 200, 0), (BF, 1, 1025, 2, 2, 128, 2, 257, 130),
    (BF, 1, 900, 16, 4, 64, 0, 16, 0),
    (F32, 1, 300, 2, 2, 64, 0, 30, 2), (F32, 2, 515, 4, 2, 128, 1, 128, 1),
])
def test_attention_forward_and_backward(dtype, B, T, H, Hkv, D, words, window, sinks):
    rows = [_row(T, 3 * T + i, words, 500) for i in range(B)]
    bm = _build(rows, window, sinks)
    dense = torch.stack([torch.from_numpy(_dense(*r, window, sinks)) for r in rows]).to(DEV)
    g = torch.Generator().manual_seed(T)
    q, k, v, do = (torch.randn(B, h, T, D, generator=g).to(dtype).to(DEV)
                   for h in (H, Hkv, Hkv, H))
    for t in (q, k, v):
        t.requires_grad_(True)
    out = flex_attention(q, k, v, block_mask=bm, enable_gqa=True)
    got = (out, *torch.autograd.grad(out, (q, k, v), do))
    refs = _attention_ref(q, k, v, do, dense, 2.0 ** -8 if dtype == BF else 0.0)
    for name, x, (ref, tol) in zip(("o", "dq", "dk", "dv"), got, refs):
        worst = float(((x.detach().double() - ref).abs() / tol).max())
        assert worst <= 1, f"{name}: {worst:.3g} of the tolerance"


def test_gradient_against_differences():
    rows = [_row(150, 1, 1, 80)]
    bm = _build(rows, 20, 2)
    g = torch.Generator().manual_seed(0)
    q, k, v, do = (torch.randn(1, 2, 150, 64, generator=g).to(DEV) for _ in range(4))
    for t in (q, k, v):
        t.requires_grad_(True)
    grads = torch.autograd.grad(flex_attention(q, k, v, block_mask=bm), (q, k, v), do)
    with torch.no_grad():
        for i, d in enumerate(grads):
            step = torch.randn(d.shape, generator=g).to(DEV)
            h = 2.0 ** -6
            hi, lo = ([t + s * h * step if j == i else t for j, t in enumerate((q, k, v))]
                      for s in (1, -1))
            f = lambda x: (flex_attention(*x, block_mask=bm).double() * do.double()).sum()  # noqa
            slope = float((f(hi) - f(lo)) / (2 * h))
            want = float((d.double() * step.double()).sum())
            # central differences: h^2 / 6 of a third derivative that is about
            # the first one's size; fp32 sums of 2e4 terms over 2 h
            assert abs(slope - want) < 2e-3 * float((d.norm() * step.norm()).double())


def test_values_in_masked_places_do_not_matter():
    """NaN and infinities behind the window stay there."""
    T, window = 400, 30
    doc = np.zeros(T, dtype=np.int32)
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(1, 1, T, 64, generator=g).to(BF).to(DEV) for _ in range(3))
    pos = torch.tensor([[T - 1]], dtype=torch.int32, device=DEV)
    zero = torch.zeros_like(pos)
    args = (torch.zeros(1, T, dtype=torch.int32, device=DEV), None, pos, zero, None)
    want = attn_decode(q[:, :, -1:], k, v, T, *args, window=window, sinks=2, q_start=zero)
    for bad in (float("nan"), float("inf")):
        k2, v2 = k.clone(), v.clone()
        k2[:, :, 2:T - window] = bad
        v2[:, :, 2:T - window] = bad
        got = attn_decode(q[:, :, -1:], k2, v2, T, *args, window=window, sinks=2, q_start=zero)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert _dense(doc, None, None, window, 2, [T - 1]).sum() == window + 2


# ---- decode

def _rows_ref(q, k, v, ok):
    """o, lse2 and sum p |v| of rows q [H, D] over k, v [H, n, D] in 64 bits."""
    s = (k.double() @ q.double()[..., None]).squeeze(-1) * q.shape[-1] ** -0.5
    s = s.masked_fill(~ok, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(ok, torch.exp(s - torch.where(lse.isinf(), 0, lse)[:, None]), 0.0)
    return ((p[..., None] * v.double()).sum(-2), lse / math.log(2.0),
            (p[..., None] * v.double().abs()).sum(-2))


def check_rows(o, lse2, q, k, v, ok, p_rounding):
    """Against _rows_ref for every row.  Scores: a chain of D products and their
    scaling in fp32, under (D + 4) U of sum |q k| / sqrt(D) -- 20 for these
    inputs -- in units of e; p within twice that and 2^-21 of the exponential;
    a sum of n terms within (n / 64 + 16) U of itself; p rounded for the second
    product where p_rounding says so; o rounded once (2^-8)."""
    B, H, M, D = q.shape
    n = k.shape[2]
    e = 20 * (D + 4) * U
    part = 2 * e + 2.0 ** -21 + (n / 64 + 16) * U
    for b in range(B):
        for t in range(M):
            kk, vv = (x[b].repeat_interleave(H // x.shape[1], 0) for x in (k, v))
            ref, lse, size = _rows_ref(q[b, :, t], kk, vv, ok[b, t])
            err = (o[b, :, t].double() - ref).abs()
            tol = 2.0 ** -8 * ref.abs() + (2 * part + p_rounding) * 1.01 * size + 1e-30
            assert bool((err <= tol).all()), float((err / tol).max())
            got = lse2[b, :, t].double()
            assert torch.equal(got.isinf(), lse.isinf())
            fin = ~lse.isinf()
            assert bool(((got - lse)[fin].abs() <= 1.5 * part + 2.0 ** -22 * lse[fin].abs()).all())


@pytest.mark.parametrize("words", [0, 2])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (100, 4), (256, 0), (300, 300), (9000, 9)])
@pytest.mark.parametrize("B,H,Hkv,M,D,T", [(1, 2, 2, 1, 64, 1500), (2, 4, 2, 3, 128, 700),
                                           (1, 8, 1, 1, 64, 33), (1, 1, 1, 8, 64, 2100)])
def test_decode_rows(B, H, Hkv, M, D, T, window, sinks, words):
    rows = [_row(T, 7 * T + i, words, 600) for i in range(B)]
    g = torch.Generator().manual_seed(T + window)
    cap = T + 5
    q = torch.randn(B, H, M, D, generator=g).to(BF).to(DEV)
    k, v = (torch.randn(B, Hkv, cap, D, generator=g).to(BF).to(DEV) for _ in range(2))
    k[:, :, T:] = float("nan")
    v[:, :, T:] = float("nan")
    pos = np.sort(np.random.default_rng(T).integers(0, T, (B, M)), 1)
    dev = lambda x, t: torch.from_numpy(np.ascontiguousarray(x)).to(DEV).to(t)  # noqa: E731
    key_doc = torch.full((B, cap), -9, dtype=torch.int32, device=DEV)
    key_doc[:, :T] = dev(np.stack([r[0] for r in rows]), torch.int32)
    kb = qb = None
    if words:
        kb = torch.zeros(B, words, cap, dtype=torch.int64, device=DEV)
        kb[:, :, :T] = torch.stack([to_dev_words(r[2], DEV) for r in rows])
        qb = torch.stack([to_dev_words(r[1][:, p], DEV) for r, p in zip(rows, pos)])
    q_doc = dev(np.stack([r[0][p] for r, p in zip(rows, pos)]), torch.int32)
    start = dev(np.stack([_starts(r[0])[p] for r, p in zip(rows, pos)]), torch.int32)
    o, lse2 = attn_decode(q, k, v, T, key_doc, kb, dev(pos, torch.int32), q_doc, qb,
                          window=window, sinks=sinks, q_start=start if sinks else None)
    ok = torch.from_numpy(np.stack([_dense(*r, window, sinks, p)
                                    for r, p in zip(rows, pos)])).to(DEV)
    check_rows(o, lse2, q, k[:, :, :T], v[:, :, :T], ok, 0.0)


def test_decode_rows_without_a_key():
    T = 700
    k = torch.randn(1, 1, T, 64, device=DEV).to(BF)
    q = torch.randn(1, 1, 2, 64, device=DEV).to(BF)
    i32 = lambda *x: torch.tensor([x], dtype=torch.int32, device=DEV)  # noqa: E731
    doc = torch.zeros(1, T, dtype=torch.int32, device=DEV)
    # a document without keys; a position before the cache
    o, lse2 = attn_decode(q, k, k, T, doc, None, i32(T - 1, -1), i32(5, 0), None, window=3, sinks=2,
                          q_start=i32(0, 0))
    assert not o.any() and torch.isneginf(lse2).all()
    o, lse2 = attn_decode(q, k, k, 0, doc, None, i32(5, 6), i32(0, 0), None, window=3)
    assert not o.any() and torch.isneginf(lse2).all()


@pytest.mark.parametrize("kw,error,match", [
    (dict(window=0), ValueError, "at least 1"), (dict(window=-3), ValueError, "at least 1"),
    (dict(window=2.5), ValueError, "at least 1"), (dict(sinks=3), ValueError, "without a window"),
    (dict(window=4, sinks=-1), ValueError, "number of tokens"),
    (dict(window=4, sinks=2), ValueError, "goes with sinks"),
    (dict(window=4, q_start=(1, "cpu")), ValueError, "goes with sinks"),
    (dict(window=4, sinks=1, q_start=(2, "cuda")), ValueError, "q_start must be"),
    (dict(window=4, sinks=1, q_start=(1, "cpu")), RuntimeError, "q's device"),
])
def test_decode_refuses(kw, error, match):
    if "q_start" in kw:
        n, dev = kw["q_start"]
        kw = {**kw, "q_start": torch.zeros(1, n, dtype=torch.int32, device=dev)}
    k = torch.zeros(1, 1, 9, 64, dtype=BF, device=DEV)
    one = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    doc = torch.zeros(1, 9, dtype=torch.int32, device=DEV)
    with pytest.raises(error, match=match):
        attn_decode(k[:, :, :1], k, k, 9, doc, None, one, one, None, **kw)


# ---- creators and models

def test_creators_take_a_window():
    row = synth.linked_lognormal_docs(900, 60.0, 1.0, 300, 0.3, seed=2)
    tokens = torch.zeros(1, 900, dtype=torch.long, device=DEV)
    doc = mo.document_ids(900, row.spans)
    qb, kb = mo.doc_link_token_bits(row.doc_index, row.link_rows)
    for bm in (create_doc_link_block_mask(tokens, row.spans, row.link_rows, window=33, sinks=2),
               SlidingWindowMaskCreator(create_doc_link_block_mask, 33, 2)(
                   tokens, row.spans, doc_links=row.link_rows)):
        _check_tables(bm, [(doc, qb, kb)], 33, 2)
    bm = make_mask_creator_callable("doc_causal", window=50)(tokens=tokens, doc_spans=row.spans)
    _check_tables(bm, [(doc, None, None)], 50, 0)
    bm = create_causal_block_mask(tokens, [], window=7, sinks=1)
    _check_tables(bm, [(np.zeros(900, dtype=np.int32), None, None)], 7, 1)

    class Detector:
        def detect_links(self, ids):
            return []

        def index_doc_span(self, span):
            return str(span.doc_id)

    bm = SlidingWindowMaskCreator(CrossDocLinkMaskCreator(Detector()), 50, 1)(
        tokens, row.spans, inputs_only=True)
    assert (bm.window, bm.sinks) == (50, 1) and bm.words == 1
    assert torch.equal(bm.doc_start[0].cpu(), torch.from_numpy(_starts(doc)))
    with pytest.raises(TypeError, match="does not take window"):
        SlidingWindowMaskCreator(lambda tokens, spans, **kw: create_causal_block_mask(tokens, spans),
                                 5)(tokens, [])
    with pytest.raises(ValueError, match="without a window"):
        mask_inputs(torch.zeros(5, dtype=torch.int32, device=DEV), sinks=1)


def _spans(n):
    cut = [0, 37, 38, 120, 300]
    return [synth.DocSpan(i, a, min(b, n)) for i, (a, b) in enumerate(zip(cut, cut[1:] + [10 ** 6]))
            if a < n]


def logits_agree(got, want, what):
    """Two evaluations of a row through four layers in other groupings of the
    same operations.  Each rounds a row to bf16 some 38 times (nine a layer,
    norm and logits), by 2^-9.8 of its norm (half a step of 2^-8 at most,
    uniform over it, values spread over a binade), independently: sqrt(2 * 38)
    2^-9.8 = 1% of the logits' norm.  Twice that is the bound."""
    got, want = got.float(), want.float()
    off = float((got - want).norm() / want.norm())
    assert off < 2e-2, f"{what}: {off:.3g} of the logits' norm"


@pytest.mark.parametrize("kv_bits,rotary,qk_norm,fuse", [
    (16, None, False, True), (16, None, False, False), (16, None, True, True),
    (16, RotaryForm(fraction=0.5, interleaved=True), False, True),
    (16, RotaryForm(scaling="by_parts", factor=4.0, original_len=64), False, True),
])
def test_generation_with_a_window(kv_bits, rotary, qk_norm, fuse):
    """Cached rows and the whole sequence's agree to bf16 rounding, token by
    token, over the graph and after an edit of the context."""
    torch.manual_seed(0)
    creator = make_mask_creator_callable("doc_causal", window=40, sinks=3)
    m = TS2TSModel.from_config(vocab_size=211, num_layers=4, model_dim=128, num_heads=2,
                               max_seq_len=512, dropout=0.0, drop_path_rate=0.0,
                               block_mask_creator=creator, qk_norm=qk_norm, rotary=rotary)
    m.to(DEV, torch.bfloat16).eval()
    m.fuse_rows, m.kv_bits = fuse, kv_bits
    g = torch.Generator().manual_seed(1)
    tokens = torch.randint(0, 211, (1, 420), generator=g).to(DEV)
    for T in [390, 391, 392, 393, 400, 401, 402]:
        got = m.forward_inference_last(tokens[:, :T], _spans(T))
        want = m.forward_inference(tokens[:, :T], _spans(T))[:, -1:]
        logits_agree(got, want, f"T={T}")
    tokens[0, 385] = 5
    for T in (403, 404):
        got = m.forward_inference_last(tokens[:, :T], _spans(T))
        want = m.forward_inference(tokens[:, :T], _spans(T))[:, -1:]
        logits_agree(got, want, f"edited, T={T}")
    # (a mask without the window would be noticed)
    m.block_mask_creator = make_mask_creator_callable("doc_causal")
    other = m.forward_inference(tokens[:, :404], _spans(404))[:, -1:]
    with pytest.raises(AssertionError, match="without"):
        logits_agree(other, want, "without")


def test_another_window_drops_the_cache():
    torch.manual_seed(0)
    m = TS2TSModel.from_config(vocab_size=97, num_layers=2, model_dim=128, num_heads=2,
                               max_seq_len=256, dropout=0.0, drop_path_rate=0.0,
                               block_mask_creator=make_mask_creator_callable("causal", window=16))
    m.to(DEV, torch.bfloat16).eval()
    tokens = torch.randint(0, 97, (1, 200), device=DEV)
    m.forward_inference_last(tokens[:, :150], [])
    for w, s in ((17, 0), (17, 1), (None, 0)):
        m.block_mask_creator = make_mask_creator_callable("causal", window=w, sinks=s)
        got = m.forward_inference_last(tokens[:, :151], [])
        fresh = m.kv_cache
        m.reset_cache()
        assert torch.equal(got, m.forward_inference_last(tokens[:, :151], []))
        m.kv_cache = fresh


@pytest.mark.parametrize("rotary", [None, RotaryForm(fraction=0.5, interleaved=True,
                                                     scaling="linear", factor=2.0)])
def test_training_step_of_a_windowed_model(rotary):
    """Loss and gradients are finite, every parameter has one, and a token that
    no window reaches has no influence."""
    torch.manual_seed(0)
    mod = TS2TSTrainingModule.from_config(
        vocab_size=101, num_layers=2, model_dim=128, num_heads=2, max_seq_len=512, dropout=0.0,
        drop_path_rate=0.0, block_mask_creator=make_mask_creator_callable("causal", window=8),
        rotary=rotary).to(DEV, torch.bfloat16)
    tokens = torch.randint(0, 101, (1, 301), device=DEV)
    loss = mod(dict(tokens=tokens))
    loss.backward()
    assert torch.isfinite(loss)
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all())
               for p in mod.parameters())
    with torch.no_grad():
        x = mod.backbone(mod.embedding(tokens[:, :300]),
                         mod.block_mask_creator(tokens=tokens[:, :300]))
        tokens[0, 100] = (tokens[0, 100] + 1) % 101
        y = mod.backbone(mod.embedding(tokens[:, :300]),
                         mod.block_mask_creator(tokens=tokens[:, :300]))
    same = (x == y).all(-1)[0]  # two layers of window 8 reach 14 tokens on
    assert bool(same[:100].all()) and bool(same[115:].all()) and not bool(same[100:115].any())


def test_decode_captured_and_replayed():
    T, cap = 900, 1000
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(1, 2, cap, 64, generator=g).to(BF).to(DEV) for _ in range(2))
    q = torch.randn(1, 2, 1, 64, generator=g).to(BF).to(DEV)
    doc = torch.zeros(1, cap, dtype=torch.int32, device=DEV)
    pos, zero = (torch.full((1, 1), x, dtype=torch.int32, device=DEV) for x in (T, 0))

    def step():
        return attn_decode(q, k, v, cap, doc, None, pos, zero, None, window=300, sinks=4,
                           q_start=zero)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for p in (900, 3, 640, 999):
        pos.fill_(p)
        q.copy_(torch.randn_like(q))
        graph.replay()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("B,T,H,Hkv,words", [(1, 4200, 8, 1, 0), (2, 2500, 8, 2, 2), (1, 100, 2, 1, 0),
                                             (1, 2304, 4, 4, 1)])
def test_columns_shared_by_work_groups(B, T, H, Hkv, words):
    """Long columns of few heads of 128: dk and dv summed from several
    work-groups' parts, within the same bounds and the same bits again."""
    from tagseq2tagseq_amd import _lib
    assert _lib.lib().t2t_attn_bwd_uneven_workspace(B, Hkv, T, 128, 0) > 0
    rows = [_row(T, 5 * T + i, words, 3000) for i in range(B)]
    window, sinks = 150, 5
    bm = _build(rows, window, sinks)
    items = (bm.q_num_blocks + bm.full_q_num_blocks) * (H // Hkv)
    assert H == Hkv or T < 1000 or int(items.max()) > 32
    dense = torch.stack([torch.from_numpy(_dense(*r, window, sinks)) for r in rows]).to(DEV)
    g = torch.Generator().manual_seed(T)
    q, k, v, do = (torch.randn(B, h, T, 128, generator=g).to(BF).to(DEV)
                   for h in (H, Hkv, Hkv, H))
    for t in (q, k, v):
        t.requires_grad_(True)
    out = flex_attention(q, k, v, block_mask=bm, enable_gqa=True)
    got = (out, *torch.autograd.grad(out, (q, k, v), do, retain_graph=True))
    again = torch.autograd.grad(out, (q, k, v), do)
    assert all(torch.equal(a, b) for a, b in zip(got[1:], again))
    for name, x, (ref, tol) in zip(("o", "dq", "dk", "dv"), got,
                                   _attention_ref(q, k, v, do, dense, 2.0 ** -8)):
        worst = float(((x.detach().double() - ref).abs() / tol).max())
        assert worst <= 1, f"{name}: {worst:.3g} of the tolerance"


# A rounding to bf16 is off by 2^-7 / m / sqrt(12) (root of the mean square)
# relative to a value of mantissa m, over mantissas spread as 1 / m
# 2^-7 sqrt(3 / (8 ln 2) / 12) = 1.66e-3.  dS is rounded once, and what it is
# summed to once; P of 9 bits adds a quarter of one: 2.38e-3 in all, and 5 % for
# the sample.
ONE_ROUNDING = 2.0 ** -7 * math.sqrt(3 / (8 * math.log(2)) / 12)
TWO_ROUNDINGS = 1.05 * ONE_ROUNDING * math.sqrt(2 + 1 / 16)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(4, 0), (40, 0), (300, 4)])
def test_gradients_round_twice(D, window, sinks):
    T, H = 1500, 4
    rows = [_row(T, 3, 0, 400)]
    bm = _build(rows, window, sinks)
    dense = torch.from_numpy(_dense(*rows[0], window, sinks))[None].to(DEV)
    g = torch.Generator().manual_seed(D + window)
    q, k, v, do = (torch.randn(1, H, T, D, generator=g).to(BF).to(DEV) for _ in range(4))
    for t in (q, k, v):
        t.requires_grad_(True)
    out = flex_attention(q, k, v, block_mask=bm)
    got = torch.autograd.grad(out, (q, k, v), do, retain_graph=True)
    want = [r for r, _ in _attention_ref(q, k, v, do, dense, 2.0 ** -8)][1:]
    for name, a, b in zip(("dq", "dk", "dv"), got, want):
        off = float((a.double() - b).norm() / b.norm())
        assert off <= TWO_ROUNDINGS, f"{name}: {off:.3g}"

    class Seen(torch.overrides.TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    with Seen():  # (a call that more than autograd watches)
        out2 = flex_attention(q, k, v, block_mask=bm)
    assert torch.equal(out, out2)
    assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(out2, (q, k, v), do)))


def _recorded(dtype, D=64, T=700, window=90, sinks=3, seed=0):
    rows = [_row(T, seed, 1, 300)]
    bm = _build(rows, window, sinks)
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn(1, 2, T, D, generator=g).to(dtype).to(DEV) for _ in range(4))
    return bm, [t.requires_grad_(True) for t in (q, k, v)], do


@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_recomputed_and_offloaded_regions(dtype):
    """Where a checkpoint or hooks take what the call's graph saves."""
    from torch.utils.checkpoint import checkpoint
    bm, x, do = _recorded(dtype)

    def call(q, k, v):
        return flex_attention(q, k, v, block_mask=bm)
    out = call(*x)
    want = torch.autograd.grad(out, x, do)
    got = [checkpoint(call, *x, use_reentrant=False), checkpoint(call, *x, use_reentrant=True)]
    with torch.autograd.graph.save_on_cpu():
        got.append(call(*x))
    for o in got:
        assert torch.equal(o, out)
        o.backward(do)
        for t, w in zip(x, want):
            assert torch.equal(t.grad, w)
            t.grad = None


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (torch.float32, 64)])
def test_training_captured_and_replayed(dtype, D):
    """The mask, forward and backward in one graph, replayed with other inputs
    beside eager calls."""
    T, H, window, sinks = 900, 2, 120, 4
    doc = torch.from_numpy(_row(T, 1, 0, 300)[0]).to(DEV).int()[None]
    g = torch.Generator().manual_seed(1)
    x = [torch.randn(1, H, T, D, generator=g).to(dtype).to(DEV).requires_grad_(True)
         for _ in range(3)]
    do = torch.randn(1, H, T, D, generator=g).to(dtype).to(DEV)

    def step(leaves):
        bm = build_block_mask(doc, window=window, sinks=sinks)
        out = flex_attention(*leaves, block_mask=bm)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(x)
    for i in range(4):
        with torch.no_grad():
            for t in (*x, do):
                t.copy_(torch.randn(t.shape, generator=g).to(dtype).to(DEV))
            doc.copy_(torch.from_numpy(_row(T, 2 + i, 0, 300)[0]).to(DEV).int()[None])
        graph.replay()
        torch.cuda.synchronize()
        own = [t.detach().clone().requires_grad_(True) for t in x]
        for a, b in zip(outs, step(own)):
            assert torch.equal(a, b)


def test_training_on_other_streams_and_threads():
    import threading
    bm, x, do = _recorded(BF, D=128, T=2500, window=400)
    want = torch.autograd.grad(flex_attention(*x, block_mask=bm), x, do)
    torch.cuda.synchronize()
    bad = []

    def work():
        own = [t.detach().clone().requires_grad_(True) for t in x]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(10):
                got = torch.autograd.grad(flex_attention(*own, block_mask=bm), own, do)
            s.synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want)):
                bad.append(1)
    threads = [threading.Thread(target=work) for _ in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


@pytest.mark.parametrize("window,sinks", [(40, 0), (300, 130)])
@pytest.mark.parametrize("D", [64, 128])
def test_decode_rows_far_apart(D, window, sinks):
    """Rows whose windows lie apart read a hull of more pieces than rows next to
    one another: up to the whole cache, in whole and in half chunks."""
    cap, M = 5000, 4
    g = torch.Generator().manual_seed(window)
    k, v = (torch.randn(2, 2, cap, D, generator=g).to(BF).to(DEV) for _ in range(2))
    q = torch.randn(2, 2, M, D, generator=g).to(BF).to(DEV)
    doc = torch.zeros(2, cap, dtype=torch.int32, device=DEV)
    at = torch.arange(cap, device=DEV)
    for row in ([0, 1, 2, 3], [0, 1700, 3333, 4999], [4999, 20, 4000, 4100], [2550, 2600, 4999, 5200]):
        pos = torch.tensor([row, row[::-1]], dtype=torch.int32, device=DEV)
        start = torch.clamp(pos - 900, min=0)
        far = pos[..., None].long() - at
        since = at - start[..., None].long()
        ok = (far >= 0) & ((far < window) | ((since >= 0) & (since < sinks)))
        o, lse2 = attn_decode(q, k, v, cap, doc, None, pos, torch.zeros_like(pos), None,
                              window=window, sinks=sinks, q_start=start if sinks else None)
        check_rows(o, lse2, q, k, v, ok, 0.0)


# (position, document's start) of rows whose windows hold no key of the cache, and
# whose sinks lie behind the other rows' windows
PAST_THE_CACHE = [[(100, 0), (5200, 4300)], [(10, 0), (10000, 4000)], [(9000, 2000), (2, 0)]]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(40, 4), (4, 4), (300, 130)])
def test_decode_rows_past_the_cache_keep_their_sinks(D, window, sinks):
    cap = 5000
    g = torch.Generator().manual_seed(window)
    k, v = (torch.randn(1, 2, cap, D, generator=g).to(BF).to(DEV) for _ in range(2))
    q = torch.randn(1, 2, 2, D, generator=g).to(BF).to(DEV)
    doc = torch.zeros(1, cap, dtype=torch.int32, device=DEV)
    at = torch.arange(cap, device=DEV)
    for rows in PAST_THE_CACHE:
        pos, start = (torch.tensor([x], dtype=torch.int32, device=DEV) for x in zip(*rows))
        far, since = (x[..., None].long() - at for x in (pos, start))
        ok = (far >= 0) & ((far < window) | ((since <= 0) & (-since < sinks)))
        assert bool(ok.any(-1).all())
        o, lse2 = attn_decode(q, k, v, cap, doc, None, pos, torch.zeros_like(pos), None,
                              window=window, sinks=sinks, q_start=start)
        check_rows(o, lse2, q, k, v, ok, 0.0)


@pytest.mark.parametrize("B,T,H,Hkv,words,pieces", [(1, 4230, 8, 8, 0, 2), (1, 2304, 8, 4, 1, 2),
                                                    (1, 2304, 8, 2, 0, 3), (2, 2200, 8, 1, 1, 4)])
def test_every_number_of_shares(B, T, H, Hkv, words, pieces):
    """Columns of more than 32 items, shared by two to four work-groups."""
    from tagseq2tagseq_amd import _lib
    assert _lib.lib().t2t_attn_bwd_uneven_pieces(B, H, Hkv, T, 128, 0) == pieces
    # one document: its sinks' column is read by the whole row
    rows = [_row(T, 5 * T + i, words, 3000) for i in range(B)]
    rows = [(np.zeros(T, dtype=np.int32), *r[1:]) for r in rows]
    window, sinks = 150, 5
    bm = _build(rows, window, sinks)
    items = (bm.q_num_blocks + bm.full_q_num_blocks) * (H // Hkv)
    assert int(items.max()) > 32 * (pieces - 1)
    dense = torch.stack([torch.from_numpy(_dense(*r, window, sinks)) for r in rows]).to(DEV)
    g = torch.Generator().manual_seed(T)
    q, k, v, do = (torch.randn(B, h, T, 128, generator=g).to(BF).to(DEV)
                   for h in (H, Hkv, Hkv, H))
    for t in (q, k, v):
        t.requires_grad_(True)
    out = flex_attention(q, k, v, block_mask=bm, enable_gqa=True)
    got = (out, *torch.autograd.grad(out, (q, k, v), do, retain_graph=True))
    again = torch.autograd.grad(out, (q, k, v), do)
    assert all(torch.equal(a, b) for a, b in zip(got[1:], again))
    for name, x, (ref, tol) in zip(("o", "dq", "dk", "dv"), got,
                                   _attention_ref(q, k, v, do, dense, 2.0 ** -8)):
        worst = float(((x.detach().double() - ref).abs() / tol).max())
        assert worst <= 1, f"{name}: {worst:.3g} of the tolerance"


def test_columns_that_cannot_be_long_take_no_workspace():
    """4 x 4 heads of 128 over 4096 tokens: 32 items a column at most."""
    B, H, T = 4, 4, 4096
    bm = build_block_mask(torch.zeros(B, T, dtype=torch.int32, device=DEV), window=500, sinks=4)
    q, k, v, do = (torch.randn(B, H, T, 128, device=DEV).to(BF) for _ in range(4))
    for t in (q, k, v):
        t.requires_grad_(True)
    out = flex_attention(q, k, v, block_mask=bm)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    grads = torch.autograd.grad(out, (q, k, v), do)
    results = sum(t.numel() * t.element_size() for t in grads) + B * H * T * 4
    assert torch.cuda.max_memory_allocated() - before < results + (8 << 20)


def test_scores_past_the_steps_of_their_sums():
    """Scores of 2^25 to 2^26 in log2 units, where the log-sum-exp of a row, a
    float, has steps of 4.

    Documents of two tokens with one key twice: the second token's P is 1/2 for
    both, and its log-sum-exp is one more than the score.  Off by at most half a
    step each in the score's rounding and in the sum's, 4 in all, P is 2^-5 .. 2^3
    to the kernel, and at most 1 where it knows that: dK of the first token,
    c P (dP - Delta) q, is 2^-4 to 2 of its value, but for the roundings of q k
    (none: all its terms are one power of two's multiple), P, dS and dK (2^-8
    each at most) and of Delta (16 bits of O)."""
    n, D = 256, 64
    T = 2 * n
    doc = (torch.arange(T, device=DEV) // 2).int()
    bm = build_block_mask(doc, window=2)
    g = torch.Generator().manual_seed(0)
    q, k = torch.zeros(1, 1, T, D), torch.zeros(1, 1, T, D)
    a = 2.0 ** torch.linspace(10.6, 11.3, n)  # (8 a 2^11 log2(e) of scores)
    q[0, 0, 1::2] = a[:, None]
    k[0, 0] = 2048.0
    v, do = torch.randn(1, 1, T, D, generator=g), torch.randn(1, 1, T, D, generator=g)
    q, k, v, do = (t.to(BF).to(DEV) for t in (q, k, v, do))
    score = (q.double() * k.double()).sum(-1)[0, 0, 1::2] / 8 / math.log(2.0)
    assert 2 ** 25 < float(score.min()) and float(score.max()) < 2 ** 26
    for t in (q, k, v):
        t.requires_grad_(True)
    _, dk, _ = torch.autograd.grad(flex_attention(q, k, v, block_mask=bm), (q, k, v), do)
    v64, do64 = v.detach().double()[0, 0].view(n, 2, D), do.double()[0, 0].view(n, 2, D)[:, 1]
    diff = ((v64[:, 0] - v64[:, 1]) / 2 * do64).sum(-1)  # dP - Delta of the first token
    clear = diff.abs() > 2.0 ** -6 * (v64.abs().amax(1) * do64.abs()).sum(-1)
    want = (diff / 2 / 8)[:, None] * q.detach().double()[0, 0, 1::2]
    ratio = (dk.double()[0, 0, 0::2] / want)[clear]
    assert int(clear.sum()) > n / 2
    assert 2.0 ** -4 * 0.95 < float(ratio.min()) and float(ratio.max()) < 2 * 1.05


@pytest.mark.parametrize("dtype,D,H,Hkv,T", [(BF, 64, 4, 2, 700), (BF, 128, 8, 1, 1300),
                                             (F32, 64, 2, 2, 300)])
def test_compiled_windowed_attention_is_the_eager_one(dtype, D, H, Hkv, T):
    """Outputs and gradients bit for bit, and without a graph to record."""
    from tagseq2tagseq_amd.attention import windowed_attention
    bm = _build([_row(T, T, 1, 300)], 90, 3)
    g = torch.Generator().manual_seed(T)
    q, k, v, do = (torch.randn(1, h, T, D, generator=g).to(dtype).to(DEV)
                   for h in (H, Hkv, Hkv, H))

    def fn(q, k, v):
        return flex_attention(q, k, v, block_mask=bm, enable_gqa=True)
    results = []
    for f in (fn, torch.compile(fn, backend="aot_eager", fullgraph=True)):
        x = [t.clone().requires_grad_(True) for t in (q, k, v)]
        out = f(*x)
        results.append([out.detach(), *torch.autograd.grad(out, x, do)])
        with torch.no_grad():
            results[-1].append(f(q, k, v))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    x = [t.clone().requires_grad_(True) for t in (q, k, v)]
    torch.library.opcheck(windowed_attention, (*x, bm.tables(), D ** -0.5))


def _windowed_loss(p, tokens, spans, layers, H, form, window, sinks):
    """Mean cross-entropy of the whole model in 64 bits, from parameters p."""
    ids, target = tokens[0, :-1], tokens[0, 1:]
    n, C = ids.shape[0], p["embedding.weight"].shape[1]
    D = C // H
    R = int(form.fraction * D)
    doc = torch.full((n,), -1, dtype=torch.int64)
    for s in spans:
        doc[s.start:min(s.end, n)] = s.doc_id
    mask = torch.from_numpy(_dense(doc.numpy(), None, None, window, sinks)).to(DEV)
    w = (form.base ** (-torch.arange(R // 2, dtype=torch.float64, device=DEV) * 2 / R)
         / form.factor)  # (positions divided)
    ang = torch.arange(n, dtype=torch.float64, device=DEV)[:, None] * w
    cos, sin = ang.cos(), ang.sin()

    def turn(x):  # interleaved pairs by the negative angle
        a, b = x[..., :R:2], x[..., 1:R:2]
        y = torch.stack((a * cos + b * sin, b * cos - a * sin), -1).flatten(-2)
        return torch.cat((y, x[..., R:]), -1)

    def rms(x, w):
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w

    x = p["embedding.weight"][ids]
    skips, n_skip = [], layers // 2
    for i in range(layers):
        at = f"backbone.layers.{i}."
        if i >= n_skip and skips:
            x = x + p["backbone.skip_weights"][i - n_skip] * skips.pop()
        h = rms(x, p[at + "ln_1.weight"]) @ p[at + "attn.qkv.weight"].t()
        a, b, v = h.view(n, 3, H, D).permute(1, 2, 0, 3)
        s = (turn(a) @ turn(b).transpose(-1, -2) / math.sqrt(D)).masked_fill(~mask, -math.inf)
        y = (torch.softmax(s, -1) @ v).transpose(0, 1).reshape(n, C)
        x = x + y @ p[at + "attn.proj.weight"].t()
        g, u = (rms(x, p[at + "ln_2.weight"]) @ p[at + "mlp.gate_up.weight"].t()).chunk(2, -1)
        x = x + (torch.nn.functional.silu(g) * u) @ p[at + "mlp.down.weight"].t()
        if i < n_skip:
            skips.append(x)
    z = rms(x, p["norm.weight"]) @ p["embedding.weight"].t()
    return torch.nn.functional.cross_entropy(z, target)


@pytest.mark.parametrize("dtype,bound", [(BF, 3e-2), (F32, 1e-4)])
@pytest.mark.parametrize("window,sinks", [(8, 0), (20, 3)])
def test_gradients_of_a_windowed_model(dtype, bound, window, sinks):
    """A training step with a rotary form and a window with sinks against the
    model in 64 bits.  Some 12 stored activations a layer and 2 layers, each
    rounded by 2^-9.8 of itself in the mean square and independent: sqrt(24)
    2^-9.8 = 0.6 % at the logits, 0.8 % behind a backward with as many; the bound
    is over three times that.  float32 has 2^-16 of it; 1e-4 is its attention's."""
    torch.manual_seed(0)
    form = RotaryForm(fraction=0.5, interleaved=True, base=500.0, scaling="linear", factor=2.0)
    m = TS2TSTrainingModule.from_config(
        vocab_size=211, num_layers=2, model_dim=256, num_heads=4, max_seq_len=512, dropout=0.0,
        drop_path_rate=0.0, rotary=form,
        block_mask_creator=make_mask_creator_callable("doc_causal", window=window, sinks=sinks))
    m = m.to(DEV, dtype)
    tokens = torch.randint(0, 211, (1, 251), generator=torch.Generator().manual_seed(1)).to(DEV)
    spans = _spans(250)
    loss = m(dict(tokens=tokens, doc_spans=spans))
    loss.backward()
    named = m.state_dict()
    p = {n: named[n].double().requires_grad_(True) for n, _ in m.named_parameters()}
    ref = _windowed_loss(p, tokens, spans, 2, 4, form, window, sinks)
    assert abs(float(loss.detach()) - float(ref.detach())) <= bound * float(ref.detach())
    for (name, prm), want in zip(m.named_parameters(), torch.autograd.grad(ref, [*p.values()])):
        off = float((prm.grad.double() - want).norm() / want.norm())
        assert off <= bound, f"{name}: {off:.3g}"
