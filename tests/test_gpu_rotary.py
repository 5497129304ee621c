"""GPU checks of the prologue with any rotary form (t2t_qkv_rotary and its
gradient) against a plain implementation in 64 bits.

Tolerance: a rotated value is a c + b s in fp32 (a product, a fused
multiply-add: 2 roundings of U = 2^-24 of |a c| + |b s|), then half a step of
its type; a copied value is exact.
"""
import dataclasses

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from tagseq2tagseq_amd import rope
from tagseq2tagseq_amd.attention import FlexSelfAttention
from tagseq2tagseq_amd.mask_creators import make_mask_creator_callable
from tagseq2tagseq_amd.model import TS2TSModel
from tagseq2tagseq_amd.rope import RotaryForm, qkv_rope, qkv_rotary, rope_tables, rotary_tables

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
U = 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32

# (B, T, H, Hkv, D, R, interleaved, dtype, positions)
SHAPES = [
    (1, 1, 1, 1, 16, 16, False, BF, "int"),
    (1, 1, 12, 12, 64, 64, False, BF, "each"),
    (2, 129, 6, 3, 64, 32, True, BF, "row"),
    (1, 77, 4, 2, 48, 48, False, BF, "each"),     # three lanes a head row
    (1, 33, 4, 2, 80, 16, True, F32, "int"),      # five, one of them turns
    (3, 5, 2, 2, 512, 512, True, BF, "each"),
    (2, 33, 16, 2, 128, 64, False, BF, "row"),
    (1, 301, 8, 8, 64, 64, True, F32, "each"),
    (2, 19, 5, 1, 80, 80, False, F32, "row"),
    (1, 2500, 12, 12, 64, 64, False, BF, "row"),
    (1, 3, 1001, 7, 16, 16, True, BF, "int"),
    (2, 2, 3, 700, 32, 32, False, F32, "each"),
    (1, 70, 1, 1, 64, 48, False, BF, "each"),     # several tokens a wave
]
IDS = ["B%d T%d H%d/%d D%d R%d %s %s %s" % (*s[:6], "inter" if s[6] else "half", str(s[7])[6:], s[8])
       for s in SHAPES]


def _case(B, T, H, Hkv, D, R, inter, dt, at, seed=0):
    g = torch.Generator().manual_seed(seed + 31 * T + D)
    qkv = torch.randn(B, T, (H + 2 * Hkv) * D, generator=g).to(dt).to(DEV)
    rows = T + 9
    cos, sin = rotary_tables(R, rows, DEV, scaling="by_parts", factor=4.0, original_len=64)
    if at == "int":
        pos, full = 7, torch.arange(7, 7 + T).expand(B, T)
    elif at == "row":
        pos = full = torch.randint(0, rows, (T,), generator=g)
        full = full.expand(B, T)
    else:
        pos = full = torch.randint(0, rows, (B, T), generator=g)
    if torch.is_tensor(pos):
        pos = pos.to(DEV)
    grads = tuple(torch.randn(B, h, T, D, generator=g).to(dt).to(DEV) for h in (H, Hkv, Hkv))
    return qkv, cos, sin, pos, full.to(DEV), grads


def _turn(x, c, s, R, inter):
    """(rows [B, T, h, D] with R dimensions rotated, what roundings are relative to)."""
    a, b = ((x[..., 0:R:2], x[..., 1:R:2]) if inter else (x[..., :R // 2], x[..., R // 2:R]))
    lo, hi = a * c + b * s, b * c - a * s
    big = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    join = ((lambda u, v: torch.stack((u, v), -1).flatten(-2)) if inter else
            (lambda u, v: torch.cat((u, v), -1)))
    rest = x[..., R:]
    return torch.cat((join(lo, hi), rest), -1), torch.cat((join(*big), 0 * rest), -1)


def _within(got, ref, size, what):
    err = (got.double() - ref).abs()
    tol = torch.finfo(got.dtype).eps / 2 * (ref.abs() + 2 * U * size) + 2 * U * size + 1e-37
    assert bool((err <= tol).all()), f"{what}: {float((err / tol).max()):.3g} of the tolerance"


def _check(out, dqkv, qkv, cos, sin, full, grads, H, Hkv, R, inter, known=None):
    B, T = qkv.shape[:2]
    c, s = (t.double()[full][:, :, None] for t in (cos, sin))
    x = qkv.detach().double().view(B, T, H + 2 * Hkv, -1)
    for name, got, part in (("q", out[0], x[:, :, :H]), ("k", out[1], x[:, :, H:H + Hkv])):
        ref, size = _turn(part, c, s, R, inter)
        if known is not None:
            ref, size = ref * known, size * known
        assert got.shape == (B, part.shape[2], T, x.shape[-1]) and got.is_contiguous()
        _within(got, ref.transpose(1, 2), size.transpose(1, 2), name)
    assert torch.equal(out[2].double(), x[:, :, H + Hkv:].transpose(1, 2))
    if dqkv is None:
        return
    d = [t.double().transpose(1, 2) for t in grads]
    dx = dqkv.view(B, T, H + 2 * Hkv, -1)
    for name, got, part in (("dq", dx[:, :, :H], d[0]), ("dk", dx[:, :, H:H + Hkv], d[1])):
        ref, size = _turn(part, c, -s, R, inter)
        if known is not None:
            ref, size = ref * known, size * known
        _within(got, ref, size, name)
    assert torch.equal(dx[:, :, H + Hkv:].double(), d[2])


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_forward_and_gradient(shape):
    B, T, H, Hkv, D, R, inter, dt, at = shape
    qkv, cos, sin, pos, full, grads = _case(*shape)
    qkv.requires_grad_(True)
    out = qkv_rotary(qkv, cos, sin, H, Hkv, pos, inter)
    d, = torch.autograd.grad(out, qkv, grads)
    assert d.shape == qkv.shape and d.dtype == dt
    _check(out, d, qkv, cos, sin, full, grads, H, Hkv, R, inter)
    with torch.no_grad():
        again = qkv_rotary(qkv, cos, sin, H, Hkv, pos, inter)
    assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_gradient_against_differences():
    qkv, cos, sin, pos, _, grads = _case(1, 5, 2, 1, 32, 16, True, F32, "each")
    qkv.requires_grad_(True)
    d, = torch.autograd.grad(qkv_rotary(qkv, cos, sin, 2, 1, pos, True), qkv, grads)

    def value(x):
        return sum((o.double() * g.double()).sum() for o, g in
                   zip(qkv_rotary(x, cos, sin, 2, 1, pos, True), grads))
    with torch.no_grad():
        g = torch.Generator().manual_seed(3)
        for _ in range(4):
            step = torch.randn(qkv.shape, generator=g).to(DEV)
            # linear: the difference is exact but for fp32 roundings of |o| ~ 10 in 160 terms
            slope = (value(qkv + step) - value(qkv - step)) / 2
            assert abs(float(slope - (d.double() * step.double()).sum())) < 1e-4


def test_whole_halves_are_qkv_rope_bitwise():
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn(2, 65, 3 * 128, generator=g).to(BF).to(DEV)
    cos, sin = rope_tables(64, 80, DEV)
    for a, b in zip(qkv_rotary(qkv, cos, sin, 2, pos=3), qkv_rope(qkv, cos, sin, 2, 3)):
        assert torch.equal(a, b)


def test_positions_without_a_table_row():
    qkv, cos, sin, _, _, grads = _case(1, 6, 2, 1, 64, 32, False, BF, "int")
    pos = torch.tensor([0, -1, cos.shape[0], 2 ** 40, -2 ** 62, 3], device=DEV)
    known = ((pos >= 0) & (pos < cos.shape[0]))
    qkv.requires_grad_(True)
    out = qkv_rotary(qkv, cos, sin, 2, 1, pos)
    d, = torch.autograd.grad(out, qkv, grads)
    full = torch.where(known, pos, 0)[None]
    _check(out, d, qkv, cos, sin, full, grads, 2, 1, 32, False,
           known=known.double()[None, :, None, None])
    nan = torch.full_like(qkv.detach(), float("nan"))
    q, k, v = qkv_rotary(nan, cos, sin, 2, 1, pos)
    assert bool((q[:, :, 1:5] == 0).all() and (k[:, :, 1:5] == 0).all())
    assert bool(q[:, :, 0].isnan().all() and v.isnan().all())


def test_strided_rows_and_gradients():
    B, T, H, Hkv, D, R = 2, 21, 4, 2, 64, 64
    qkv, cos, sin, pos, full, grads = _case(B, T, H, Hkv, D, R, True, BF, "each")
    W = (H + 2 * Hkv) * D
    wide = torch.zeros(B, T, 2 * W + 8, dtype=BF, device=DEV)
    layouts = [wide[:, :, 8:8 + W], wide[:, :, 1:1 + W],  # the second off 16-byte boundaries
               torch.zeros(T, B, W, dtype=BF, device=DEV).transpose(0, 1),
               torch.zeros(W, B, T, dtype=BF, device=DEV).permute(1, 2, 0)]
    odd = tuple(g.transpose(1, 2).contiguous().transpose(1, 2) for g in grads[:2]) + (
        grads[2][:, :, :1].expand(-1, -1, T, -1),)  # one gradient row for every token
    want = None
    for x in layouts:
        x.copy_(qkv)
        x = x.detach().requires_grad_(True)
        out = qkv_rotary(x, cos, sin, H, Hkv, pos, True)
        d, = torch.autograd.grad(out, x, odd)
        _check(out, d, x, cos, sin, full, odd, H, Hkv, R, True)
        want = d if want is None else want
        assert torch.equal(d, want)


def test_part_of_the_outputs():
    """Outputs that nothing uses have zero gradients."""
    qkv, cos, sin, pos, full, grads = _case(1, 9, 2, 2, 64, 64, False, BF, "row")
    qkv.requires_grad_(True)
    _, k, _ = qkv_rotary(qkv, cos, sin, 2, 2, pos)
    d, = torch.autograd.grad(k, qkv, grads[1])
    zero = torch.zeros_like(grads[0]), grads[1], torch.zeros_like(grads[2])
    _check(qkv_rotary(qkv, cos, sin, 2, 2, pos), d, qkv, cos, sin, full, zero, 2, 2, 64, False)


def test_nothing_to_do():
    cos, sin = rotary_tables(64, 4, DEV)
    for B, T in ((0, 3), (2, 0)):
        x = torch.zeros(B, T, 256, dtype=BF, device=DEV, requires_grad=True)
        for pos in (0, torch.zeros(T, dtype=torch.int64, device=DEV)):
            out = qkv_rotary(x, cos, sin, 2, 1, pos)
            assert [tuple(o.shape) for o in out] == [(B, 2, T, 64), (B, 1, T, 64), (B, 1, T, 64)]
            d, = torch.autograd.grad(out, x, tuple(torch.zeros_like(o) for o in out))
            assert d.shape == x.shape


@pytest.mark.parametrize("train", [False, True])
def test_captured_and_replayed(train):
    qkv, cos, sin, pos, full, grads = _case(1, 40, 4, 2, 64, 32, True, BF, "row")
    out = d = None

    def step():
        if not train:
            with torch.no_grad():
                return qkv_rotary(qkv, cos, sin, 4, 2, pos, True), None
        o = qkv_rotary(qkv, cos, sin, 4, 2, pos, True)
        return o, torch.autograd.grad(o, qkv, grads)[0]

    qkv.requires_grad_(train)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, d = step()
    for i in range(3):
        with torch.no_grad():
            qkv.copy_(torch.randn_like(qkv))
            pos.copy_(torch.randint_like(pos, 0, cos.shape[0]))
        graph.replay()
        torch.cuda.synchronize()
        _check(out, d, qkv, cos, sin, pos.expand(1, -1), grads, 4, 2, 32, True)


def test_another_stream_and_two_threads():
    import threading
    qkv, cos, sin, pos, full, grads = _case(1, 500, 4, 2, 64, 64, False, BF, "row")
    want = qkv_rotary(qkv, cos, sin, 4, 2, pos)
    torch.cuda.synchronize()
    bad = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = qkv_rotary(qkv, cos, sin, 4, 2, pos)
            s.synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want)):
                bad.append(1)
    threads = [threading.Thread(target=work) for _ in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_watched_calls_agree():
    qkv, cos, sin, pos, _, grads = _case(1, 9, 2, 1, 64, 32, True, BF, "each")
    want = qkv_rotary(qkv, cos, sin, 2, 1, pos, True)
    fx = make_fx(lambda x, p: qkv_rotary(x, cos, sin, 2, 1, p, True))(qkv, pos)
    for a, b in zip(fx(qkv, pos), want):
        assert torch.equal(a, b)
    x = qkv.clone().requires_grad_(True)
    eager, = torch.autograd.grad(qkv_rotary(x, cos, sin, 2, 1, pos, True), x, grads)
    op = rope.qkv_rotary_op(x, cos, sin, 2, 1, pos, 0, True)
    assert torch.equal(torch.autograd.grad(op, x, grads)[0], eager)
    torch.library.opcheck(rope.qkv_rotary_op, (x, cos, sin, 2, 1, pos, 0, True))


@pytest.mark.parametrize("op", [False, True])
def test_second_order(op):
    """The gradient is linear in the incoming one, so its own gradient is the
    forward map."""
    qkv, cos, sin, pos, _, grads = _case(2, 7, 2, 1, 64, 32, True, F32, "each")
    qkv.requires_grad_(True)
    g = tuple(t.clone().requires_grad_(True) for t in grads)
    out = (rope.qkv_rotary_op(qkv, cos, sin, 2, 1, pos, 0, True) if op else
           qkv_rotary(qkv, cos, sin, 2, 1, pos, True))
    d, = torch.autograd.grad(out, qkv, g, create_graph=True)
    w = torch.randn_like(d).requires_grad_(True)
    back = torch.autograd.grad(d, g, w, create_graph=True)
    for a, b in zip(back, qkv_rotary(w.detach(), cos, sin, 2, 1, pos, True)):
        assert torch.equal(a, b)
    third, = torch.autograd.grad(back, w, grads)  # and that one's the gradient again
    assert torch.equal(third, d)


def test_positions_changed_before_the_backward_are_noticed():
    qkv, cos, sin, pos, _, grads = _case(1, 5, 1, 1, 64, 64, False, BF, "row")
    qkv.requires_grad_(True)
    out = qkv_rotary(qkv, cos, sin, 1, 1, pos)
    pos.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, qkv, grads)


@pytest.mark.parametrize("form", [
    None, RotaryForm(base=10001.0), RotaryForm(fraction=0.5, interleaved=True, base=10001.0)])
def test_training_behind_an_evaluation_in_inference_mode(form):
    """Tables made under inference mode serve the backward that saves them."""
    T = 333  # (no other test's: the first call here makes them)
    torch.manual_seed(0)
    mod = FlexSelfAttention(128, 2, T, rotary=form).to(DEV, BF)
    x = torch.randn(1, T, 384, device=DEV).to(BF)
    with torch.inference_mode():
        want = mod.heads(x)
    x.requires_grad_(True)
    out = mod.heads(x)
    grads = [torch.randn_like(t) for t in out]
    got, = torch.autograd.grad(out, x, grads)
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    if form is not None:
        cos, sin = mod.rotary.tables(DEV)
        again = qkv_rotary(x, cos, sin, 2, interleaved=form.interleaved)
        assert torch.equal(torch.autograd.grad(again, x, grads)[0], got)


@pytest.mark.parametrize("positive", [False, True])
@pytest.mark.parametrize("interleaved,fraction", [(False, 1.0), (False, 0.5), (True, 1.0),
                                                  (True, 0.25)])
def test_modules_turn_either_way(positive, interleaved, fraction):
    """The rotation by -angle, or by the published one's +angle: (a + i b) e^(i p w)
    with angles of 64 bits, at a range of positions and at those of a tensor."""
    T, D, H = 150, 64, 2
    R = int(fraction * D)
    form = RotaryForm(fraction=fraction, interleaved=interleaved, base=700.0, positive=positive)
    mod = FlexSelfAttention(H * D, H, T, rotary=form).to(DEV, BF)
    g = torch.Generator().manual_seed(R)
    qkv = torch.randn(1, T, 3 * H * D, generator=g).to(BF).to(DEV)
    rows = qkv.double().view(1, T, 3, H, D).permute(2, 0, 3, 1, 4)
    w = 700.0 ** (-torch.arange(R // 2, dtype=torch.float64, device=DEV) * 2 / R)

    def published(x, at):
        r = x[..., :R]
        a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else r.chunk(2, -1)
        ang = torch.outer(at.double(), w) * (1 if positive else -1)
        z = torch.complex(a, b) * torch.polar(torch.ones_like(ang), ang)
        turned = (torch.stack([z.real, z.imag], -1).flatten(-2) if interleaved else
                  torch.cat([z.real, z.imag], -1))
        return torch.cat([turned, x[..., R:]], -1)
    order = torch.randperm(T, generator=g).to(DEV)
    for pos, at in ((0, torch.arange(T, device=DEV)), (order, order)):
        q, k, v = mod.heads(qkv, pos)
        assert torch.equal(v.double(), rows[2])
        for x, y in ((q, rows[0]), (k, rows[1])):
            want = published(y, at)
            # |a c| + |b s| <= sqrt(2) |(a, b)|; tables and arithmetic 3 roundings of
            # U of that (whole halves at base 700: rope.rotary_tables' too)
            size = y.abs().amax(-1, keepdim=True) * 2
            assert bool(((x.double() - want).abs() <= 2.0 ** -8 * want.abs() + 4 * U * size).all())


@pytest.mark.parametrize("kv_bits", [16, 8])
@pytest.mark.parametrize("kw", [dict(rotary=RotaryForm(positive=True)),
                                dict(rotary=RotaryForm(positive=True), qk_norm=True),
                                dict(rotary=RotaryForm(positive=True, interleaved=True,
                                                       fraction=0.5))])
@torch.no_grad()
def test_generation_turns_as_the_whole_sequence_does(kw, kv_bits):
    """Cached rows of the published direction: new tokens and a few rows at once
    (8 bits: near the whole sequence's, whose keys are not rounded)."""
    torch.manual_seed(0)
    m = TS2TSModel.from_config(
        vocab_size=97, num_layers=2, model_dim=128, num_heads=2, max_seq_len=256, dropout=0.0,
        drop_path_rate=0.0, block_mask_creator=make_mask_creator_callable("causal"), **kw)
    m.to(DEV, BF).eval()
    m.kv_bits = kv_bits
    tokens = torch.randint(0, 97, (1, 200), generator=torch.Generator().manual_seed(1)).to(DEV)
    # bf16: as logits_agree's, two layers; e4m3 keys and values: 2^-4 / sqrt(12) of
    # a value at most in the mean square, averaged over heads and keys: under 2 %
    # of a layer's attention rows, which are part of the row they are added to
    bound = 2e-2 if kv_bits == 16 else 6e-2
    for T in (150, 151, 152, 160, 161):
        got = m.forward_inference_last(tokens[:, :T], []).float()
        want = m.forward_inference(tokens[:, :T], [])[:, -1:].float()
        assert float((got - want).norm() / want.norm()) < bound
    other = TS2TSModel.from_config(
        vocab_size=97, num_layers=2, model_dim=128, num_heads=2, max_seq_len=256, dropout=0.0,
        drop_path_rate=0.0, block_mask_creator=make_mask_creator_callable("causal"),
        **{**kw, "rotary": dataclasses.replace(kw["rotary"], positive=False)}).to(DEV, BF).eval()
    for a, b in zip(other.backbone.parameters(), m.backbone.parameters()):
        a.copy_(b)
    x = m._embed(tokens[:, :160])
    bm = make_mask_creator_callable("causal")(tokens=tokens[:, :160])
    assert not torch.allclose(other.backbone(x, bm), m.backbone(x, bm), atol=1e-3)
