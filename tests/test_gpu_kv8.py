"""GPU checks of the 8-bit key/value cache: the append bit for bit against its
definition, the attention over it against a plain implementation in 64 bits,
and the model's generation with it.
"""
import math

import numpy as np
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from tagseq2tagseq_amd import kv8
from tagseq2tagseq_amd.kv8 import BLOCK, KV8Cache, attn_decode_kv8, kv8_append
from tagseq2tagseq_amd.mask_creators import make_mask_creator_callable
from tagseq2tagseq_amd.model import TS2TSModel
from tagseq2tagseq_amd.rope import RotaryForm
from tests.helpers import random_row, to_dev_words
from tests.test_gpu_window import (ONE_ROUNDING, PAST_THE_CACHE, _dense, _spans, _starts, check_rows,
                                   logits_agree)

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
BF, F32 = torch.bfloat16, torch.float32


# ---- append

def _scale(amax):
    """Smallest power of two under which amax is at most 448, from 2^-120 to 2^120."""
    if amax == 0:
        return 2.0 ** -120
    m, e = math.frexp(amax)
    return 2.0 ** min(max(e - 9 + (m > 0.875), -120), 120)


class Model:
    """The cache as its definition has it: codes as numbers, on the CPU."""

    def __init__(self, cache):
        self.cap = cache.capacity
        self.k = cache.k_codes.cpu().float()
        self.v = cache.v_codes.cpu().float().transpose(3, 4).contiguous()
        self.ks, self.vs = cache.k_scale.cpu().clone(), cache.v_scale.cpu().clone()

    def append(self, k, v, pos):
        B, Hkv, M, D = k.shape
        k, v = k.cpu().double(), v.cpu().double()
        bad = ~(k.isfinite().all(-1) & v.isfinite().all(-1))
        for b in range(B):
            p = int(pos[b % len(pos)])
            if M == 0 or p < 0 or p > self.cap - M:
                continue
            for x, codes, scale, fill in ((k, self.k, self.ks, math.nan), (v, self.v, self.vs, 0.0)):
                for h in range(Hkv):
                    for blk in range(p // BLOCK, (p + M - 1) // BLOCK + 1):
                        lo, hi = max(p, blk * BLOCK), min(p + M, (blk + 1) * BLOCK)
                        new = x[b, h, lo - p:hi - p].clone()
                        off = bad[b, h, lo - p:hi - p]
                        new[off] = 0
                        n = lo - blk * BLOCK
                        now = _scale(float(new.abs().max()))
                        if n:
                            was = float(scale[b, h, blk])
                            now = max(now, was)
                            codes[b, h, blk, :n] = self._round(codes[b, h, blk, :n].double() *
                                                               (was / now))
                        new = self._round(new / now)
                        new[off] = fill
                        codes[b, h, blk, n:n + hi - lo] = new
                        scale[b, h, blk] = now

    @staticmethod
    def _round(x):
        """To 3 mantissa bits, ties to even, exponents from -6 (exact in float64)."""
        e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30))).clamp(min=-6)
        step = torch.exp2(e - 3)
        return (torch.round(x / step) * step).float()

    def check(self, cache):
        same = lambda a, b: bool(((a == b) | (a.isnan() & b.isnan())).all())  # noqa: E731
        assert torch.equal(cache.k_scale.cpu(), self.ks), "key scales"
        assert torch.equal(cache.v_scale.cpu(), self.vs), "value scales"
        assert same(cache.k_codes.cpu().float(), self.k), "key codes"
        assert same(cache.v_codes.cpu().float().transpose(3, 4), self.v), "value codes"


def _rows(B, Hkv, M, D, dt, g, size=1.0):
    wide = torch.exp2(torch.randint(-4, 5, (1, Hkv, 1, D), generator=g).float()) * size
    return tuple((torch.randn(B, Hkv, M, D, generator=g) * wide).to(dt).to(DEV) for _ in range(2))


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("B,Hkv,D,cap,steps", [
    (1, 1, 64, 1, [(0, 1)]),
    (1, 2, 64, 200, [(0, 64), (64, 64), (128, 72)]),
    (2, 3, 128, 300, [(0, 5), (5, 1), (6, 57), (63, 1), (64, 1), (65, 200), (265, 35)]),
    (1, 2, 128, 130, [(0, 130), (100, 3), (64, 1), (3, 1), (3, 127), (129, 1)]),
    (1, 12, 64, 700, [(0, 700), (0, 700), (699, 1), (1, 640)]),
])
def test_append_bit_for_bit(B, Hkv, D, cap, steps, dt):
    g = torch.Generator().manual_seed(cap)
    cache = KV8Cache(B, Hkv, cap, D, DEV)
    model = Model(cache)
    for i, (pos, M) in enumerate(steps):
        # sizes that grow and shrink, so that scales do
        k, v = _rows(B, Hkv, M, D, dt, g, 2.0 ** [0, 6, -9, 3, 12, -20, 1][i % 7])
        at = (pos if i % 2 == 0 else
              torch.full((1 + (i // 2) % 2 * (B - 1),), pos, dtype=torch.int64, device=DEV))
        cache.append(k, v, at)
        model.append(k, v, [pos])
        model.check(cache)


def test_append_at_each_sequences_position():
    B, Hkv, D, cap, M = 5, 2, 64, 150, 70
    g = torch.Generator().manual_seed(0)
    cache = KV8Cache(B, Hkv, cap, D, DEV)
    model = Model(cache)
    k, v = _rows(B, Hkv, cap, D, BF, g)
    cache.append(k, v, 0)
    model.append(k, v, [0])
    for pos in ([0, 80, 17, 63, 64], [-1, 81, 2 ** 40, -2 ** 62, 80], [1, 2, 3, 4, 5]):
        k, v = _rows(B, Hkv, M, D, BF, g, 4.0)
        cache.append(k, v, torch.tensor(pos, device=DEV))
        model.append(k, v, pos)
        model.check(cache)


def test_values_that_are_hard_to_hold():
    """Zeros, ties, the largest and smallest numbers, and tokens that are not
    finite."""
    D, cap = 64, 192
    cache = KV8Cache(1, 1, cap, D, DEV)
    model = Model(cache)
    k = torch.zeros(1, 1, 192, D)
    v = torch.zeros(1, 1, 192, D)
    k[0, 0, :64] = torch.linspace(-1, 1, 64 * D).view(64, D)
    k[0, 0, 1, :8] = torch.tensor([17., 19., 21., 23., 448., -448., 2.0 ** -9, 2.0 ** -10])
    k[0, 0, 2, :4] = torch.tensor([449., 447., 464., 480.])
    v[0, 0, 64:128] = 3e38
    v[0, 0, 65] = 1e-38
    k[0, 0, 128:] = 2.0 ** -130
    k[0, 0, 10, 5] = math.nan
    k[0, 0, 70, 0] = math.inf
    v[0, 0, 71, 63] = -math.inf
    v[0, 0, 140, 7] = math.nan
    k, v = k.to(DEV), v.to(DEV)
    cache.append(k, v, 0)
    model.append(k, v, [0])
    model.check(cache)
    assert bool(cache.k_codes[0, 0, 1, 6].float().isnan().all())
    # a block that holds NaN is written again under a larger scale
    big = torch.full((1, 1, 1, D), 3e5, device=DEV)
    cache.append(big, big, 20)
    model.append(big, big, [20])
    model.check(cache)


def test_strided_heads():
    B, Hkv, M, D, cap = 2, 3, 40, 64, 100
    g = torch.Generator().manual_seed(0)
    k, v = _rows(B, Hkv, M, D, BF, g)
    want = KV8Cache(B, Hkv, cap, D, DEV)
    want.append(k, v, 30)
    packed = torch.zeros(B, M, 3 * Hkv, D, dtype=BF, device=DEV)
    packed[:, :, Hkv:2 * Hkv], packed[:, :, 2 * Hkv:] = k.transpose(1, 2), v.transpose(1, 2)
    odd = torch.zeros(B, Hkv, M, D + 1, dtype=BF, device=DEV)
    odd[..., 1:] = k
    turned = v.permute(3, 2, 1, 0).contiguous().permute(3, 2, 1, 0)
    for kk, vv in ((packed[:, :, Hkv:2 * Hkv].transpose(1, 2), packed[:, :, 2 * Hkv:].transpose(1, 2)),
                   (odd[..., 1:], turned)):
        got = KV8Cache(B, Hkv, cap, D, DEV)
        got.append(kk, vv, 30)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8))
                   for a, b in zip(got.buffers(), want.buffers()))
    one = k[:, :, :1].expand(-1, -1, M, -1)
    got, want = KV8Cache(B, Hkv, cap, D, DEV), KV8Cache(B, Hkv, cap, D, DEV)
    got.append(one, one, 0)
    want.append(one.contiguous(), one.contiguous(), 0)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8))
               for a, b in zip(got.buffers(), want.buffers()))


def test_append_moves_the_caches_versions():
    cache = KV8Cache(1, 1, 64, 64, DEV)
    k = torch.ones(1, 1, 1, 64, device=DEV)
    before = [t._version for t in cache.buffers()]
    cache.append(k, k, 3)
    assert all(t._version > b for t, b in zip(cache.buffers(), before))


def test_nothing_to_append():
    cache = KV8Cache(2, 1, 64, 64, DEV)
    none = torch.zeros(2, 1, 0, 64, device=DEV)
    cache.append(none, none, 64)
    cache.append(none, none, torch.zeros(2, dtype=torch.int64, device=DEV))
    assert not cache.k_scale.any()


# ---- attention

def _attend_case(B, H, Hkv, M, D, T, words, window, sinks, cap=None, seed=0, max_doc=600):
    g = torch.Generator().manual_seed(seed + T + H)
    cap = cap or T + 5
    cache = KV8Cache(B, Hkv, cap, D, DEV)
    k, v = (0.5 * t for t in _rows(B, Hkv, cap, D, F32, g, 0.25))
    cache.append(k, v, 0)
    rows = [random_row(T, np.random.default_rng(7 * T + i), words=words, uncovered=True,
                       max_doc=max_doc) for i in range(B)]
    q = (0.5 * torch.randn(B, H, M, D, generator=g)).to(BF).to(DEV)
    pos = np.sort(np.random.default_rng(T).integers(0, T, (B, M)), 1)
    pos[:, -1] = T - 1
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(DEV).int()  # noqa: E731
    key_doc = torch.full((B, cap), -9, dtype=torch.int32, device=DEV)
    key_doc[:, :T] = dev(np.stack([r[0] for r in rows]))
    kb = qb = None
    if words:
        kb = torch.zeros(B, words, cap, dtype=torch.int64, device=DEV)
        kb[:, :, :T] = torch.stack([to_dev_words(r[2], DEV) for r in rows])
        qb = torch.stack([to_dev_words(r[1][:, p], DEV) for r, p in zip(rows, pos)])
    q_doc = dev(np.stack([r[0][p] for r, p in zip(rows, pos)]))
    start = dev(np.stack([_starts(r[0])[p] for r, p in zip(rows, pos)]))
    mask = (key_doc, kb, dev(pos), q_doc, qb)
    limits = dict(window=window, sinks=sinks, q_start=start if sinks else None)
    ok = torch.from_numpy(np.stack([_dense(*r, window, sinks, p)
                                    for r, p in zip(rows, pos)])).to(DEV)
    return cache, q, mask, limits, ok


@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (70, 3), (300, 200)])
@pytest.mark.parametrize("B,H,Hkv,M,D,T,words", [
    (1, 1, 1, 1, 64, 1, 0), (1, 2, 2, 1, 64, 63, 0), (2, 2, 1, 1, 128, 64, 1),
    (1, 12, 12, 1, 64, 1500, 0), (2, 4, 2, 3, 128, 700, 2), (1, 8, 1, 2, 64, 333, 0),
    (1, 16, 1, 1, 128, 257, 8), (1, 1, 1, 16, 64, 2100, 1), (3, 6, 3, 5, 64, 129, 0),
    (1, 3, 1, 5, 128, 5000, 0), (1, 2, 1, 2, 64, 4097, 0), (2, 4, 4, 1, 64, 4096, 1),
    (1, 9, 1, 1, 64, 20000, 0), (1, 2, 2, 1, 64, 1024, 0), (1, 2, 2, 1, 64, 1025, 1),
    (2, 2, 2, 1, 128, 512, 1), (2, 12, 1, 1, 64, 900, 0), (1, 2, 2, 1, 128, 513, 0), (1, 4, 2, 1, 128, 2049, 1), (40, 4, 4, 1, 64, 9000, 0),
])
def test_attention_rows(B, H, Hkv, M, D, T, words, window, sinks):
    cache, q, mask, limits, ok = _attend_case(B, H, Hkv, M, D, T, words, window, sinks)
    o, lse2 = cache.attend(q, T, *mask, **limits)
    k, v = (t[:, :, :T] for t in cache.values(F32))
    check_rows(o, lse2, q, k, v, ok, 2.0 ** -8)  # p in bf16
    # the whole capacity: the positions behind are of no document
    again = cache.attend(q, cache.capacity, *mask, **limits)
    check_rows(*again, q, k, v, ok, 2.0 ** -8)


def kv8_chunks(B, Hkv, n, D):
    """0 where no row is split."""
    from tagseq2tagseq_amd import _lib
    return _lib.lib().t2t_kv8_attend_workspace(B, Hkv, Hkv, 1, n, D)


@pytest.mark.parametrize("T,D", [(300, 64), (200, 64), (1000, 64), (4300, 64), (512, 128),
                                 (2100, 128)])
def test_many_sequences_in_one_chunk_each(T, D):
    """Enough sequences that no row is split."""
    B = 130 if T <= 1000 else 33
    cache, q, mask, limits, ok = _attend_case(B, 64, 32, 2, D, T, 0, None, 0, max_doc=200)
    assert kv8_chunks(B, 32, T, D) == 0
    o, lse2 = cache.attend(q, T, *mask, **limits)
    few = slice(0, 5)
    check_rows(o[few], lse2[few], q[few], *(t[few, :, :T] for t in cache.values(F32)), ok[few],
               2.0 ** -8)


def test_rows_without_a_key():
    cache, q, mask, _, _ = _attend_case(1, 2, 1, 3, 64, 400, 0, None, 0)
    doc, _, pos, q_doc, _ = mask
    q_doc = torch.tensor([[77, int(doc[0, 5]), 77]], dtype=torch.int32, device=DEV)
    pos = torch.tensor([[399, -1, 2]], dtype=torch.int32, device=DEV)
    for n in (400, 0):
        o, lse2 = cache.attend(q, n, doc, None, pos, q_doc, None)
        assert not o.any() and torch.isneginf(lse2).all()


def test_tokens_that_are_not_finite():
    """They make the rows that read them NaN, and no other."""
    cache = KV8Cache(1, 1, 300, 64, DEV)
    k, v = (torch.randn(1, 1, 300, 64, device=DEV) for _ in range(2))
    clean = KV8Cache(1, 1, 300, 64, DEV)
    clean.append(k, v, 0)
    k2, v2 = k.clone(), v.clone()
    k2[0, 0, 50, 3], v2[0, 0, 250, 9] = math.nan, math.inf
    cache.append(k2, v2, 0)
    q = torch.randn(1, 1, 3, 64, device=DEV).to(BF)
    doc = torch.zeros(1, 300, dtype=torch.int32, device=DEV)
    pos = torch.tensor([[40, 120, 290]], dtype=torch.int32, device=DEV)
    for window, bad in ((None, [False, True, True]), (20, [False] * 3), (60, [False, False, True])):
        o, lse2 = cache.attend(q, 300, doc, None, pos, torch.zeros_like(pos), None, window=window)
        assert o[0, 0].isnan().all(-1).tolist() == bad and lse2[0, 0].isnan().tolist() == bad
        want, _ = clean.attend(q, 300, doc, None, pos, torch.zeros_like(pos), None, window=window)
        for t in range(3):
            if not bad[t]:  # (their block's scale is the clean one's: both near 1)
                assert torch.equal(o[0, 0, t], want[0, 0, t])


@pytest.mark.parametrize("n", [1, 17, 64, 100, 130])
def test_what_was_never_stored_is_not_looked_at(n):
    """NaN codes and scales around the tokens, as fresh memory may hold them,
    and around the positions that a row's window leaves."""
    g = torch.Generator().manual_seed(n)
    clean, junk = KV8Cache(2, 2, 300, 64, DEV), KV8Cache(2, 2, 300, 64, DEV)
    for t in junk.buffers():
        t.view(torch.uint8).fill_(0xff)
    k, v = _rows(2, 2, n, 64, BF, g)
    for c in (clean, junk):
        c.append(k, v, 0)
    q = torch.randn(2, 2, 3, 64, generator=g).to(BF).to(DEV)
    doc = torch.zeros(1, 300, dtype=torch.int32, device=DEV)
    doc[:, n // 2:] = 1  # (two documents, the second to the end)
    pos = torch.tensor([[n // 3, n - 1, n - 1]], dtype=torch.int32, device=DEV)
    q_doc = doc[:, pos[0].long()]
    for window in (None, 5):
        want = clean.attend(q, n, doc, None, pos, q_doc, None, window=window)
        assert want[0].isfinite().all()
        for keys in (n, 300):
            got = junk.attend(q, keys, doc, None, pos, q_doc, None, window=window)
            ref = clean.attend(q, keys, doc, None, pos, q_doc, None, window=window)
            assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_strided_queries_and_masks_of_one_row():
    cache, q, mask, _, _ = _attend_case(2, 4, 2, 2, 64, 300, 0, None, 0)
    doc, _, pos, q_doc, _ = mask
    one = (doc[:1].contiguous(), None, pos[:1].contiguous(), q_doc[:1].contiguous(), None)
    want = cache.attend(q, 300, *(t if t is None else t.repeat(2, 1) for t in one))
    odd = torch.zeros(2, 2, 4, 65, dtype=BF, device=DEV)
    odd[..., 1:] = q.transpose(1, 2)
    for x in (q, q.transpose(1, 2).contiguous().transpose(1, 2), odd[..., 1:].transpose(1, 2)):
        got = cache.attend(x, 300, *one)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_past_32_bits():
    """Two sequences of codes whose second starts behind 2^32 bytes."""
    Hkv, D = 66, 128
    cap = (1 << 32) // (Hkv * D) // 64 * 64 + 64
    cache = KV8Cache(2, Hkv, cap, D, DEV)
    assert cache.k_codes[0].numel() > 1 << 32
    n = cap - 100
    k, v = (torch.randn(2, Hkv, 100, D, device=DEV) for _ in range(2))
    cache.append(k, v, n)
    near = KV8Cache(2, Hkv, 228, D, DEV)  # the same offsets inside the block
    near.append(k, v, n % 64 + 64)
    q = torch.randn(2, Hkv, 1, D, device=DEV).to(BF)
    doc = torch.zeros(1, cap, dtype=torch.int32, device=DEV)
    zero = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    o, lse2 = cache.attend(q, cap, doc, None, zero + cap - 1, zero, None, window=100)
    k8, v8 = (t[:, :, n % 64 + 64:n % 64 + 164] for t in near.values(F32))
    check_rows(o[:, :4], lse2[:, :4], q[:, :4], k8[:, :4], v8[:, :4],
               torch.ones(2, 1, 100, dtype=torch.bool, device=DEV), 2.0 ** -8)
    check_rows(o[:, -3:], lse2[:, -3:], q[:, -3:], k8[:, -3:], v8[:, -3:],
               torch.ones(2, 1, 100, dtype=torch.bool, device=DEV), 2.0 ** -8)


def test_captured_and_replayed():
    """Two graphs of append and attention, replayed in turn with eager work
    between, against the eager calls."""
    cap = 400
    g = torch.Generator().manual_seed(0)
    caches = [KV8Cache(1, 2, cap, 64, DEV) for _ in range(2)]
    eager = [KV8Cache(1, 2, cap, 64, DEV) for _ in range(2)]
    k, v = _rows(1, 2, 300, 64, BF, g)
    for c in caches + eager:
        c.append(k, v, 0)
    q = torch.randn(1, 2, 1, 64, generator=g).to(BF).to(DEV)
    kn, vn = (t[:, :, :1].contiguous() for t in (k, v))
    at = torch.full((1,), 300, dtype=torch.int64, device=DEV)
    doc = torch.zeros(1, cap, dtype=torch.int32, device=DEV)
    zero = torch.zeros(1, 1, dtype=torch.int32, device=DEV)

    def step(c):
        c.append(kn, vn, at)
        return c.attend(q, cap, doc, None, at.int().view(1, 1), zero, None)

    graphs, outs = [], []
    for c in caches:
        step(c)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(c))
        graphs.append(graph)
    for c in eager:
        step(c)  # (a warm-up appends, too)
    for i in range(5):
        at.fill_(300 + i)
        for t in (q, kn, vn):
            t.copy_(torch.randn_like(t) * 2.0 ** i)
        for j in (0, 1):
            graphs[j].replay()
        torch.cuda.synchronize()
        for j in (0, 1):
            for a, b in zip(outs[j], step(eager[j])):
                assert torch.equal(a, b)
            for a, b in zip(caches[j].buffers(), eager[j].buffers()):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_another_stream_and_two_threads():
    import threading
    cache, q, mask, limits, _ = _attend_case(1, 4, 2, 1, 64, 3000, 0, 200, 4)
    want = cache.attend(q, 3000, *mask, **limits)
    torch.cuda.synchronize()
    bad = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = cache.attend(q, 3000, *mask, **limits)
            s.synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want)):
                bad.append(1)
    threads = [threading.Thread(target=work) for _ in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_traced_calls():
    cache, q, mask, limits, _ = _attend_case(1, 4, 2, 1, 64, 200, 0, 50, 2)
    want = cache.attend(q, 200, *mask, **limits)
    doc, kb, pos, q_doc, qb = mask
    args = (q, *cache.buffers(), 200, doc, kb, pos, q_doc, qb, 0.125, 50, 2, limits["q_start"])
    assert all(torch.equal(a, b) for a, b in zip(kv8.kv8_attend_op(*args), want))
    fx = make_fx(lambda x, p: cache.attend(x, 200, doc, kb, p, q_doc, qb, **limits))(q, pos)
    assert all(torch.equal(a, b) for a, b in zip(fx(q, pos), want))
    k = torch.randn(1, 2, 3, 64, device=DEV)
    one, two = KV8Cache(1, 2, 100, 64, DEV), KV8Cache(1, 2, 100, 64, DEV)
    one.append(k, k, 7)
    kv8.kv8_append_op(k, k, None, 7, *two.buffers(), 100)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8))
               for a, b in zip(one.buffers(), two.buffers()))


def test_no_gradient():
    cache = KV8Cache(1, 1, 64, 64, DEV)
    k = torch.zeros(1, 1, 1, 64, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        cache.append(k, k.detach(), 0)
    with torch.no_grad():
        cache.append(k, k, 0)
    one = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    q = torch.zeros(1, 1, 1, 64, dtype=BF, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        cache.attend(q, 1, one, None, one, one, None)


def _zeros(*shape, dtype=F32, device="cuda"):
    return lambda: torch.zeros(*shape, dtype=dtype, device=device)


@pytest.mark.parametrize("change,error,match", [
    (dict(k=_zeros(1, 2, 3, 64, device="cpu")), RuntimeError, "GPU tensors"),
    (dict(k=_zeros(1, 2, 3, 128)), ValueError, r"must be \[B, Hkv, M, D\]"),
    (dict(k=_zeros(1, 2, 3, 64, dtype=torch.float16)), NotImplementedError, "Half"),
    (dict(k=_zeros(1, 2, 3, 64, dtype=BF)), ValueError, "differ in dtype"),
    (dict(pos=-1), ValueError, "exceed capacity"), (dict(pos=98), ValueError, "exceed capacity"),
    (dict(pos=_zeros(1, dtype=torch.int32)), ValueError, "int64"),
    (dict(pos=_zeros(3, dtype=torch.int64)), ValueError, "one position"),
    (dict(pos=_zeros(1, dtype=torch.int64, device="cpu")), ValueError, "int64 tensor on"),
    (dict(capacity=129), ValueError, "exceeds"), (dict(capacity=-1), ValueError, "negative"),
    (dict(capacity=2), ValueError, "exceed capacity"),
])
def test_append_refuses(change, error, match):
    cache = KV8Cache(1, 2, 100, 64, DEV)
    a = dict(k=_zeros(1, 2, 3, 64), v=_zeros(1, 2, 3, 64), pos=0, capacity=100)
    a = {n: x() if callable(x) else x for n, x in {**a, **change}.items()}
    cap = a.pop("capacity")
    with pytest.raises(error, match=match):
        kv8_append(*a.values(), *cache.buffers(), capacity=cap)
    assert not cache.k_scale.any()


def test_attention_refuses():
    cache, q, (doc, _, pos, q_doc, _), _, _ = _attend_case(1, 4, 2, 1, 64, 200, 0, None, 0)
    ok = dict(q=q, k=cache.k_codes, v=cache.v_codes, ks=cache.k_scale, vs=cache.v_scale, n=200,
              doc=doc, kb=None, pos=pos, q_doc=q_doc, qb=None)
    words = torch.zeros(1, 1, doc.shape[1], dtype=torch.int64, device=DEV)
    for change, error, match in [
            (dict(n=-1), ValueError, "exceeds"), (dict(n=10 ** 6), ValueError, "exceeds"),
            (dict(q=q.float()), NotImplementedError, "q dtype"),
            (dict(q=q[:, :3]), ValueError, "multiple of Hkv"),
            (dict(q=q.expand(-1, -1, 9, -1)), NotImplementedError, "exceeds 16"),
            (dict(k=cache.k_codes.view(torch.uint8)), ValueError, "float8_e4m3fn"),
            (dict(k=cache.v_codes), RuntimeError, "are one"),
            (dict(vs=cache.v_scale[:, :, :1]), ValueError, "scales"),
            (dict(ks=cache.k_scale.transpose(0, 1)), ValueError, "scales"),
            (dict(k=cache.k_codes.transpose(3, 4).contiguous().transpose(3, 4)), ValueError,
             "contiguous"),
            (dict(doc=doc.long()), ValueError, "key_doc"), (dict(doc=doc.cpu()), RuntimeError, "GPU"),
            (dict(pos=pos.expand(1, 1).repeat(1, 2)), ValueError, "q_pos"),
            (dict(kb=words), ValueError, "go together"),
            (dict(kb=words, qb=torch.zeros(1, 1, 2, dtype=torch.int64, device=DEV)), ValueError,
             "q_bits"),
            (dict(scale=0.0), ValueError, "scale"), (dict(scale=math.nan), ValueError, "scale"),
            (dict(window=0), ValueError, "at least 1"), (dict(sinks=1), ValueError, "without"),
            (dict(window=3, sinks=1), ValueError, "goes with sinks")]:
        a = {**ok, **change}
        kw = {n: a.pop(n) for n in ("scale", "window", "sinks") if n in a}
        with pytest.raises(error, match=match):
            attn_decode_kv8(*a.values(), **kw)


# ---- the model's generation

def _model(window=None, sinks=0, **kw):
    torch.manual_seed(0)
    creator = make_mask_creator_callable("doc_causal", window=window, sinks=sinks)
    m = TS2TSModel.from_config(
        vocab_size=211, num_layers=4, model_dim=128, num_heads=2, max_seq_len=450, dropout=0.0,
        drop_path_rate=0.0, block_mask_creator=creator, **kw)
    m.to(DEV, torch.bfloat16).eval()
    m.kv_bits = 8
    return m


def _cached_rows_ref(m, tokens, spans, T):
    """Logits of the last row from the model's own cache, its attention in 64
    bits: every layer's projections as the model has them."""
    cache = m.kv_cache
    bm = m.block_mask_creator(tokens=tokens[:, :T], doc_spans=spans)
    i = torch.arange(T, device=DEV)
    ok = bm.mask_mod()(torch.zeros((), dtype=torch.long, device=DEV), 0, i[-1:, None], i[None])
    bb, skips = m.backbone, []
    x = m._embed(tokens[:, T - 1:T])
    n_skip = len(bb.skip_weights)
    for j, layer in enumerate(bb.layers):
        if j >= n_skip and skips:
            x = x + bb.skip_weights[j - n_skip] * skips.pop()
        q, _, _ = layer.attn.heads(layer.attn.qkv(layer.ln_1(x)), T - 1)
        k, v = (t[:, :, :T].double() for t in cache.layers8[j].values(F32))
        s = (q.double() @ k.transpose(2, 3).contiguous()) * 64 ** -0.5
        y = (torch.softmax(s.masked_fill(~ok, -math.inf), -1) @ v).to(BF)
        x = m._layer_tail(layer, y.transpose(1, 2).reshape(1, 1, -1), x, False)
        if j < n_skip:
            skips.append(x)
    return torch.nn.functional.linear(m.norm(x), m.lm_head_weight)


@pytest.mark.parametrize("fuse", [True, False])
@pytest.mark.parametrize("window,sinks,kw", [
    (None, 0, {}), (50, 0, {}), (None, 0, dict(qk_norm=True)), (50, 3, dict(qk_norm=True)),
    # everything that long contexts add at once
    (40, 4, dict(rotary=RotaryForm(fraction=0.5, interleaved=True, scaling="by_parts", factor=4.0,
                                   original_len=128))),
])
@torch.no_grad()
def test_generation(window, sinks, kw, fuse):
    m = _model(window=window, sinks=sinks, **kw)
    m.fuse_rows = fuse
    tokens = torch.randint(0, 211, (1, 450), generator=torch.Generator().manual_seed(1)).to(DEV)
    for T in [390, 391, 392, 393, 400, 401, 449, 450]:  # whole, token by token, a few rows
        got = m.forward_inference_last(tokens[:, :T], _spans(T)).float()
        logits_agree(got, _cached_rows_ref(m, tokens, _spans(T), T), f"T={T}")
    assert m.kv_cache.bits == 8 and m.kv_cache.length == 450


@torch.no_grad()
def test_graph_and_eager_steps_agree_and_bits_switch():
    tokens = torch.randint(0, 211, (1, 420), generator=torch.Generator().manual_seed(2)).to(DEV)
    runs = []
    for graphs in (True, False):
        m = _model()
        m.use_graphs = graphs
        runs.append([m.forward_inference_last(tokens[:, :T], _spans(T)) for T in range(395, 410)])
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    m.kv_bits = 16
    a = m.forward_inference_last(tokens[:, :410], _spans(410))
    assert m.kv_cache.bits == 16
    m.reset_cache()
    assert torch.equal(a, m.forward_inference_last(tokens[:, :410], _spans(410)))
    m.kv_bits = 4
    with pytest.raises(ValueError, match="16 or 8"):
        m.forward_inference_last(tokens[:, :411], _spans(411))


@torch.no_grad()
def test_an_edited_context_is_recomputed():
    m = _model()
    tokens = torch.randint(0, 211, (1, 420), generator=torch.Generator().manual_seed(3)).to(DEV)
    for T in (395, 396):
        m.forward_inference_last(tokens[:, :T], _spans(T))
    tokens[0, 390] = 7
    for T in (397, 398):
        got = m.forward_inference_last(tokens[:, :T], _spans(T)).float()
        logits_agree(got, _cached_rows_ref(m, tokens, _spans(T), T), f"T={T}")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(40, 4), (4, 4), (300, 130)])
def test_rows_past_the_cache_keep_their_sinks(D, window, sinks):
    cap = 5000
    g = torch.Generator().manual_seed(window)
    cache = KV8Cache(1, 2, cap, D, DEV)
    cache.append(*_rows(1, 2, cap, D, BF, g, 0.25), 0)
    k, v = cache.values(F32)
    q = (0.5 * torch.randn(1, 2, 2, D, generator=g)).to(BF).to(DEV)
    doc = torch.zeros(1, cap, dtype=torch.int32, device=DEV)
    at = torch.arange(cap, device=DEV)
    for rows in PAST_THE_CACHE:
        pos, start = (torch.tensor([x], dtype=torch.int32, device=DEV) for x in zip(*rows))
        far, since = (x[..., None].long() - at for x in (pos, start))
        ok = (far >= 0) & ((far < window) | ((since <= 0) & (-since < sinks)))
        o, lse2 = cache.attend(q, cap, doc, None, pos, torch.zeros_like(pos), None,
                               window=window, sinks=sinks, q_start=start)
        check_rows(o, lse2, q, k, v, ok, 2.0 ** -16)  # (p in two bf16 numbers)


@pytest.mark.parametrize("bits,launches", [(8, [1, 1, 2, 3]), (16, [1, 2, 3, 5])])
@torch.no_grad()
def test_new_rows_go_through_as_many_at_once_as_the_cache_takes(bits, launches, monkeypatch):
    from tagseq2tagseq_amd.model import KVCache
    m = _model(window=50, sinks=2)
    m.kv_bits = bits
    seen = []
    attend = KVCache.attend
    monkeypatch.setattr(KVCache, "attend",
                        lambda self, i, q, *a, **kw: (seen.append(q.shape[2]),
                                                      attend(self, i, q, *a, **kw))[1])
    tokens = torch.randint(0, 211, (1, 450), generator=torch.Generator().manual_seed(4)).to(DEV)
    m.forward_inference_last(tokens[:, :300], _spans(300))
    T = 300
    for n, count in zip((2, 16, 17, 40), launches):
        seen.clear()
        T += n
        m.forward_inference_last(tokens[:, :T], _spans(T))
        assert len(seen) == 4 * count and sum(seen) == 4 * n


@pytest.mark.parametrize("pos", [5, 70, 127])
def test_a_sequence_that_begins_inside_a_block(pos):
    """Positions before the first token were never stored: their codes may be
    anything, their scales are zeros."""
    g = torch.Generator().manual_seed(pos)
    clean, junk = KV8Cache(1, 2, 300, 64, DEV), KV8Cache(1, 2, 300, 64, DEV)
    for t in junk.buffers()[:2]:
        t.view(torch.uint8).fill_(0xff)
    doc = torch.full((1, 300), 7, dtype=torch.int32, device=DEV)
    doc[:, pos:] = 0
    at = torch.tensor([[pos + 39]], dtype=torch.int32, device=DEV)
    q = torch.randn(1, 2, 1, 64, generator=g).to(BF).to(DEV)
    steps = [_rows(1, 2, n, 64, BF, g, 2.0 ** i) for i, n in enumerate((1, 30, 9))]
    outs = []
    for c in (clean, junk):
        p = pos
        for k, v in steps:  # (each under a larger scale)
            c.append(k, v, p)
            p += k.shape[2]
        outs.append(c.attend(q, p, doc, None, at, torch.zeros_like(at), None))
    assert outs[0][0].isfinite().all()
    assert all(torch.equal(a, b) for a, b in zip(*outs))


# A rounding to bf16 is off by 1.66e-3 in the mean square (test_gpu_window); o is
# rounded once, and by how much is known: the distance to the nearest bf16 number
# changes by no more than its argument, so that with x the sum before the rounding
# |o - want| <= |x - want| + |bf16(x) - x| <= 2 |x - want| + |bf16(want) - want|.
# (The mean of 1.66e-3 would not do: the channels' sizes differ by 2^8, and the
# few hundred values of the largest ones, which are the norm, are off by 1.5e-3 to
# 2e-3.)  p in two bf16 numbers adds 2^-8 of a rounding more, fp32 sums less than
# 1e-5; p in one would add as much again as a rounding of o (an o of independent
# values is as long as its terms' squares' sum).
@pytest.mark.parametrize("window,sinks", [(3, 0), (40, 2), (None, 0)])
@pytest.mark.parametrize("B,H,Hkv,M,D,T", [
    (2, 4, 4, 1, 64, 700), (1, 4, 1, 2, 128, 500), (1, 8, 1, 2, 64, 900), (2, 6, 2, 5, 128, 300),
    (8, 8, 4, 1, 64, 5000), (8, 6, 2, 3, 128, 5000),
])
def test_rows_round_once(B, H, Hkv, M, D, T, window, sinks):
    """Up to eight rows a kv head and more, in one pass and in chunks."""
    cache, q, mask, limits, ok = _attend_case(B, H, Hkv, M, D, T, 0, window, sinks)
    o, _ = cache.attend(q, T, *mask, **limits)
    k, v = (t[:, :, :T].repeat_interleave(H // Hkv, 1).double() for t in cache.values(F32))
    s = (q.double() @ k.transpose(2, 3).contiguous()) * D ** -0.5
    want = torch.softmax(s.masked_fill(~ok[:, None], -math.inf), -1) @ v
    off = float((o.double() - want).norm() / want.norm())
    once = float((want.to(BF).double() - want).norm() / want.norm())
    assert off <= once + 0.05 * ONE_ROUNDING, f"{off:.3g}, one rounding {once:.3g}"
