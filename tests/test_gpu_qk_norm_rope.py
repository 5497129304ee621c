"""GPU checks of the prologue with per-head norms (t2t_qk_norm_rope, its
gradient and its cache-append form) against a plain implementation in 64 bits.

Tolerances count roundings.  A result is rounded once to its type: half a step,
eps / 2 of the value.  Before that stands fp32 arithmetic, U = 2^-24 a step:
  forward   o = y1 c + y2 s, y = x r w.  r: a sum of D squares in chains of at
            most 16 + 5 additions, a division, an addition, the square root
            (half of the sum's error) and 1 / sqrt itself: under 16 U.  y adds
            two products, o two roundings: under 24 U of |y1 c| + |y2 s|.
  backward  dy (2 roundings), g = dy w, the mean of g n (a chain of 21 and the
            products), r twice: under 64 U of r |g| + r |n| mean |g n|, with |g|
            taken from |d1 c| + |d2 s|.
  dw        a sum of N terms that each have 24 U; the chain is the terms a lane
            sums, 6 + 4 combinations, and at most (1024 + 15) / 16 + 16 group
            sums: under (200 + N / 4096) U of the sum of |terms|.
"""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from tagseq2tagseq_amd.rope import qk_norm_rope, qk_norm_rope_append, rope_tables

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
U = 2.0 ** -24
EPS = 1e-6
BF, F32 = torch.bfloat16, torch.float32

# (B, T, H, Hkv, D, rows dtype, weight dtype, pos0)
SHAPES = [
    (1, 1, 1, 1, 16, BF, BF, 0),
    (1, 1, 12, 12, 64, BF, F32, 5),
    (2, 129, 6, 3, 64, BF, BF, 0),
    (1, 77, 4, 2, 48, BF, BF, 3),      # three lanes of a group of four
    (3, 5, 2, 2, 512, BF, F32, 0),
    (2, 33, 16, 2, 128, BF, BF, 1),
    (1, 301, 8, 8, 64, F32, F32, 0),
    (2, 19, 5, 1, 80, F32, BF, 2),
    (1, 2500, 12, 12, 64, BF, BF, 0),  # several rounds a work-group
    (1, 3, 1001, 7, 16, BF, BF, 0),
    (2, 2, 3, 700, 32, F32, F32, 0),
]
IDS = ["B%d T%d H%d/%d D%d %s %s" % (*s[:5], str(s[5])[6:], str(s[6])[6:]) for s in SHAPES]


def _inputs(B, T, H, Hkv, D, dt, wdt, pos0, seed=0):
    g = torch.Generator().manual_seed(seed + 31 * T + D)
    qkv = (torch.randn(B, T, (H + 2 * Hkv) * D, generator=g) *
           (0.1 + 3 * torch.rand(B, T, 1, generator=g))).to(dt).to(DEV)
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).to(wdt).to(DEV) for _ in range(2))
    cos, sin = rope_tables(D, pos0 + T + 2, DEV)
    return qkv, qw, kw, cos, sin


def _split(x, H, Hkv):
    x = x.reshape(x.shape[0], x.shape[1], H + 2 * Hkv, -1).transpose(1, 2)
    return x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]


def _halves(x):
    return x[..., :x.shape[-1] // 2], x[..., x.shape[-1] // 2:]


def _forward_ref(x, w, cos, sin):
    """float64 [B, h, T, D] rows: the result, and |y1 c| + |y2 s|."""
    y = w * x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    a, b = _halves(y)
    out = torch.cat((a * cos + b * sin, b * cos - a * sin), -1)
    size = torch.cat(((a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs()), -1)
    return out, size


def _backward_ref(d, x, w, cos, sin):
    """dx, what its roundings are relative to, the dw terms and theirs."""
    D = x.shape[-1]
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    a, b = _halves(d)
    dy = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    size = torch.cat(((a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs()), -1)
    n = x * r
    dx = r * (dy * w - n * (dy * w * n).mean(-1, keepdim=True))
    big = r * (size * w.abs() + n.abs() * (size * w.abs() * n.abs()).mean(-1, keepdim=True))
    return dx, big, (dy * n).reshape(-1, D), (size * n.abs()).reshape(-1, D)


def _within(got, ref, size, steps, what):
    err = (got.double() - ref).abs()
    tol = torch.finfo(got.dtype).eps / 2 * ref.abs() + steps * U * size + 1e-37
    assert bool((err <= tol).all()), f"{what}: {float((err / tol).max()):.3g} of the tolerance"


def _check_forward(out, qkv, qw, kw, cos, sin, H, Hkv, pos0):
    T = qkv.shape[1]
    c, s = (t[pos0:pos0 + T].double() for t in (cos, sin))
    parts = _split(qkv.double(), H, Hkv)
    for name, got, x, w in (("q", out[0], parts[0], qw), ("k", out[1], parts[1], kw)):
        ref, size = _forward_ref(x, w.double(), c, s)
        assert got.shape == ref.shape and got.is_contiguous() and got.dtype == qkv.dtype
        _within(got, ref, size, 24, name)
    assert torch.equal(out[2].double(), parts[2])


def _check_backward(got, grads, qkv, qw, kw, cos, sin, H, Hkv, pos0):
    T, D = qkv.shape[1], cos.shape[1] * 2
    c, s = (t[pos0:pos0 + T].double() for t in (cos, sin))
    parts, dparts = _split(qkv.double(), H, Hkv), _split(got[0], H, Hkv)
    assert got[0].shape == qkv.shape and got[0].dtype == qkv.dtype
    for i, (name, w) in enumerate((("q", qw), ("k", kw))):
        dx, size, terms, tsize = _backward_ref(grads[i].double(), parts[i], w.double(), c, s)
        _within(dparts[i], dx, size, 64, "d" + name)
        assert got[1 + i].shape == (D,) and got[1 + i].dtype == w.dtype
        _within(got[1 + i], terms.sum(0), tsize.sum(0), 200 + terms.shape[0] / 4096,
                f"d{name}_weight")
    assert torch.equal(dparts[2].double(), grads[2].double())


def _grads(out, seed=1):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(o.shape, generator=g).to(o.dtype).to(DEV) for o in out)


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_forward_and_backward(shape):
    B, T, H, Hkv, D, dt, wdt, pos0 = shape
    qkv, qw, kw, cos, sin = _inputs(*shape)
    for t in (qkv, qw, kw):
        t.requires_grad_(True)
    out = qk_norm_rope(qkv, qw, kw, cos, sin, H, num_kv_heads=Hkv, pos0=pos0, eps=EPS)
    grads = _grads(out)
    got = torch.autograd.grad(out, (qkv, qw, kw), grads)
    plain = [t.detach() for t in (qkv, qw, kw)]
    _check_forward(tuple(o.detach() for o in out), *plain, cos, sin, H, Hkv, pos0)
    _check_backward(got, grads, *plain, cos, sin, H, Hkv, pos0)


def test_same_bits_without_autograd_and_again():
    qkv, qw, kw, cos, sin = _inputs(2, 333, 6, 2, 64, BF, BF, 0)
    a = qk_norm_rope(qkv, qw, kw, cos, sin, 6, num_kv_heads=2)
    leaves = [t.clone().requires_grad_(True) for t in (qkv, qw, kw)]
    b = qk_norm_rope(*leaves, cos, sin, 6, num_kv_heads=2)
    for x, y in zip(a, b):
        assert torch.equal(x, y.detach())
    grads = _grads(a)
    one = torch.autograd.grad(b, leaves, grads, retain_graph=True)
    two = torch.autograd.grad(b, leaves, grads)
    for x, y in zip(one, two):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("offset,pad", [(0, 64), (8, 24), (1, 3)])
def test_strided_rows(dt, offset, pad):
    """Rows of a wider buffer, on and off 16-byte boundaries."""
    B, T, H, Hkv, D = 2, 37, 3, 1, 64
    qkv, qw, kw, cos, sin = _inputs(B, T, H, Hkv, D, dt, BF, 0)
    W = qkv.shape[2]
    big = torch.full((B, T, W + pad + offset), 7.0, dtype=dt, device=DEV)
    view = big[:, :, offset:offset + W]
    view.copy_(qkv)
    view.requires_grad_(True)
    out = qk_norm_rope(view, qw, kw, cos, sin, H, num_kv_heads=Hkv)
    _check_forward(tuple(o.detach() for o in out), qkv, qw, kw, cos, sin, H, Hkv, 0)
    grads = _grads(out)
    (dqkv,) = torch.autograd.grad(out, view, grads)
    want = torch.autograd.grad(
        qk_norm_rope(qkv.requires_grad_(True), qw, kw, cos, sin, H, num_kv_heads=Hkv), qkv, grads)
    assert torch.equal(dqkv, want[0])


def test_gradient_layouts():
    """Gradients in [B, T, H, D] storage, expanded, off a boundary, and absent."""
    B, T, H, D = 2, 21, 4, 64
    qkv, qw, kw, cos, sin = _inputs(B, T, H, H, D, BF, BF, 0)
    leaves = [t.requires_grad_(True) for t in (qkv, qw, kw)]

    def run(grads):
        return torch.autograd.grad(qk_norm_rope(*leaves, cos, sin, H), leaves, grads)

    g = _grads(qk_norm_rope(*leaves, cos, sin, H))
    want = run(g)
    turned = tuple(x.transpose(1, 2).contiguous().transpose(1, 2) for x in g)
    shifted = tuple(torch.cat((x.new_zeros(1), x.reshape(-1)))[1:].view(x.shape) for x in g)
    for other in (turned, shifted):
        for a, b in zip(run(other), want):
            assert torch.equal(a, b)
    ones = tuple(torch.ones_like(x) for x in g)
    flat = tuple(torch.ones((), dtype=BF, device=DEV).expand_as(x) for x in g)
    for a, b in zip(run(flat), run(ones)):
        assert torch.equal(a, b)
    # only q is used: k and v get zero gradients
    q, _, _ = qk_norm_rope(*leaves, cos, sin, H)
    dqkv, _, dkw = torch.autograd.grad(q, leaves, g[0])
    _, dk, dv = _split(dqkv, H, H)
    assert not dk.any() and not dv.any() and not dkw.any()


def test_gradient_against_differences():
    """d/dt f(inputs + t u) of the plain form in 64 bits, f = <out, grads>, by
    central differences (h = 1e-5: truncation h^2 times a third derivative of
    order 1e2 and cancellation 2^-53 |f| / h, both under 1e-6 of the sum of
    |gradient u| here) against the kernel's float32 gradients."""
    B, T, H, Hkv, D = 1, 9, 4, 2, 32
    qkv, qw, kw, cos, sin = _inputs(B, T, H, Hkv, D, F32, F32, 0)
    leaves = [t.requires_grad_(True) for t in (qkv, qw, kw)]
    out = qk_norm_rope(*leaves, cos, sin, H, num_kv_heads=Hkv, eps=EPS)
    grads = _grads(out)
    got = torch.autograd.grad(out, leaves, grads)
    c, s = cos[:T].double(), sin[:T].double()

    def f(x, a, b):
        q, k, v = _split(x, H, Hkv)
        o = (_forward_ref(q, a, c, s)[0], _forward_ref(k, b, c, s)[0], v)
        return sum((y * g.double()).sum() for y, g in zip(o, grads))

    base = [t.detach().double() for t in leaves]
    gen = torch.Generator().manual_seed(3)
    for i in range(3):
        for _ in range(3):
            u = torch.randn(base[i].shape, generator=gen, dtype=torch.float64).to(DEV)
            h = 1e-5
            hi, lo = ([b + sgn * h * u if j == i else b for j, b in enumerate(base)]
                      for sgn in (1, -1))
            diff = float((f(*hi) - f(*lo)) / (2 * h))
            size = float((got[i].double().abs() * u.abs()).sum())
            assert abs(diff - float((got[i].double() * u).sum())) <= 1e-5 * size


def test_zero_rows_and_values_that_are_not_finite():
    B, T, H, D = 1, 6, 2, 64
    qkv, qw, kw, cos, sin = _inputs(B, T, H, H, D, BF, BF, 0)
    clean = qk_norm_rope(qkv, qw, kw, cos, sin, H)
    bad = qkv.clone()
    bad[0, 1, :D] = 0                      # a query row of zeros
    bad[0, 2, D + 3] = float("nan")        # head 1 of the query
    bad[0, 3, H * D + 5] = float("inf")    # head 0 of the key
    q, k, v = qk_norm_rope(bad, qw, kw, cos, sin, H)
    assert not q[0, 0, 1].any()
    assert q[0, 1, 2].isnan().all()
    # inf / rms(inf) is not a number there; the other values become 0
    assert k[0, 0, 3].isnan().any()
    keep = torch.ones(B, H, T, dtype=torch.bool, device=DEV)
    keep[0, 0, 1] = keep[0, 1, 2] = False
    assert torch.equal(q[keep], clean[0][keep])
    keep = torch.ones(B, H, T, dtype=torch.bool, device=DEV)
    keep[0, 0, 3] = False
    assert torch.equal(k[keep], clean[1][keep])
    assert torch.equal(v, clean[2])


def test_no_tokens():
    for B, T in ((0, 5), (2, 0)):
        qkv, qw, kw, cos, sin = _inputs(1, 1, 2, 2, 64, BF, F32, 4)
        qkv = qkv.new_empty(B, T, 6 * 64).requires_grad_(True)
        qw.requires_grad_(True)
        q, k, v = qk_norm_rope(qkv, qw, kw, cos, sin, 2)
        assert q.shape == (B, 2, T, 64)
        dqkv, dqw = torch.autograd.grad((q, k, v), (qkv, qw), (q, k, v))
        assert dqkv.shape == qkv.shape and not dqw.any()


def test_second_order_is_refused():
    qkv, qw, kw, cos, sin = _inputs(1, 3, 1, 1, 32, F32, F32, 0)
    qkv.requires_grad_(True)
    q, _, _ = qk_norm_rope(qkv, qw, kw, cos, sin, 1)
    (d,) = torch.autograd.grad(q.sum(), qkv, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), qkv)


# ---- new tokens into a cache

@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("B,M,H,Hkv,D", [(1, 1, 12, 12, 64), (3, 4, 6, 2, 48), (2, 8, 4, 4, 128)])
def test_append_writes_the_prologues_rows(B, M, H, Hkv, D, dt):
    cap = 40
    qkv, qw, kw, _, _ = _inputs(B, M, H, Hkv, D, dt, BF, 0)
    cos, sin = rope_tables(D, cap, DEV)
    filled = [torch.randn(B, Hkv, cap, D, device=DEV).to(dt) for _ in range(2)]
    first = [(7 * b) % (cap - M + 1) for b in range(B)]
    want_q = torch.cat([qk_norm_rope(qkv[b:b + 1], qw, kw, cos, sin, H, Hkv, pos0=first[b])[0]
                        for b in range(B)])
    want_k, want_v = (c.clone() for c in filled)
    for b in range(B):
        _, k, v = qk_norm_rope(qkv[b:b + 1], qw, kw, cos, sin, H, Hkv, pos0=first[b])
        want_k[b, :, first[b]:first[b] + M], want_v[b, :, first[b]:first[b] + M] = k[0], v[0]
    pos = torch.tensor(first, device=DEV)[:, None] + torch.arange(M, device=DEV)
    kc, vc = (c.clone() for c in filled)
    q = qk_norm_rope_append(qkv, qw, kw, cos, sin, H, pos, kc, vc)
    assert torch.equal(q, want_q) and torch.equal(kc, want_k) and torch.equal(vc, want_v)
    # one list of positions for all sequences, and a first position
    kc, vc = (c.clone() for c in filled)
    at = pos[0] + 3 if first[0] + M + 3 <= cap else pos[0]
    q = qk_norm_rope_append(qkv, qw, kw, cos, sin, H, at, kc, vc)
    k2, v2 = (c.clone() for c in filled)
    q2 = qk_norm_rope_append(qkv, qw, kw, cos, sin, H, int(at[0]), k2, v2)
    assert torch.equal(q, q2) and torch.equal(kc, k2) and torch.equal(vc, v2)


def test_append_of_many_rows_and_a_strided_cache():
    B, M, H, Hkv, D, cap = 1, 100, 4, 2, 64, 160
    qkv, qw, kw, _, _ = _inputs(B, M, H, Hkv, D, BF, BF, 0)
    cos, sin = rope_tables(D, 128, DEV)
    store = torch.zeros(2, B, cap, Hkv, D, dtype=BF, device=DEV)  # [B, cap, Hkv, D] storage
    kc, vc = store[0].transpose(1, 2), store[1].transpose(1, 2)
    q = qk_norm_rope_append(qkv, qw, kw, cos, sin, H, 28, kc, vc)
    wq, wk, wv = qk_norm_rope(qkv, qw, kw, cos, sin, H, Hkv, pos0=28)
    assert torch.equal(q, wq) and torch.equal(kc[:, :, 28:128], wk)
    assert torch.equal(vc[:, :, 28:128], wv)
    assert not kc[:, :, :28].any() and not kc[:, :, 128:].any() and not vc[:, :, 128:].any()


def test_append_positions_without_a_row_and_twice_the_same():
    B, M, H, D, cap = 2, 5, 2, 64, 16
    qkv, qw, kw, _, _ = _inputs(B, M, H, H, D, BF, BF, 0)
    cos, sin = rope_tables(D, 64, DEV)  # more table rows than cache rows
    kc, vc = (torch.randn(B, H, cap, D, device=DEV).to(BF) for _ in range(2))
    k0, v0 = kc.clone(), vc.clone()
    pos = torch.tensor([[3, -1, 3, 16, 15], [0, 1 << 40, 2, 2, -(1 << 62)]], device=DEV)
    q = qk_norm_rope_append(qkv, qw, kw, cos, sin, H, pos, kc, vc)
    for b, m, p in ((0, 2, 3), (0, 4, 15), (1, 0, 0), (1, 3, 2)):
        wq, wk, wv = qk_norm_rope(qkv[b:b + 1, m:m + 1], qw, kw, cos, sin, H, pos0=p)
        assert torch.equal(q[b, :, m], wq[0, :, 0])
        assert torch.equal(kc[b, :, p], wk[0, :, 0]) and torch.equal(vc[b, :, p], wv[0, :, 0])
        k0[b, :, p], v0[b, :, p] = wk[0, :, 0], wv[0, :, 0]
    assert torch.equal(kc, k0) and torch.equal(vc, v0)
    for b, m in ((0, 1), (0, 3), (1, 1), (1, 4)):
        assert not q[b, :, m].any()
    # rows that share a position all get their query
    assert q[0, :, 0].any() and q[1, :, 2].any()


# ---- graphs and streams

def test_captured_forward_and_backward():
    """A captured training call, replayed on new values beside eager work."""
    shape = (1, 200, 6, 2, 64, BF, F32, 0)
    qkv, qw, kw, cos, sin = _inputs(*shape)
    leaves = [t.clone().requires_grad_(True) for t in (qkv, qw, kw)]
    grads = _grads(qk_norm_rope(qkv, qw, kw, cos, sin, 6, 2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = qk_norm_rope(*leaves, cos, sin, 6, 2)
        torch.autograd.grad(out, leaves, grads)
        del out
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = qk_norm_rope(*leaves, cos, sin, 6, 2)
        got = torch.autograd.grad(out, leaves, grads)
    for seed in range(3):
        new = _inputs(*shape, seed=10 + seed)[:3]
        with torch.no_grad():
            for leaf, n in zip(leaves, new):
                leaf.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        fresh = [n.clone().requires_grad_(True) for n in new]
        eager = qk_norm_rope(*fresh, cos, sin, 6, 2)
        want = torch.autograd.grad(eager, fresh, grads)
        for a, b in zip((*out, *got), (*eager, *want)):
            assert torch.equal(a, b)


def test_offsets_past_32_bits():
    """Rows and cache heads more than 2^32 elements apart."""
    H, Hkv, D, T, cap = 2, 2, 64, 3, 8
    qkv, qw, kw, _, _ = _inputs(1, T, H, Hkv, D, BF, BF, 0)
    cos, sin = rope_tables(D, cap, DEV)
    far = (1 << 32) + 64
    store = torch.empty(2 * far + 4096, dtype=BF, device=DEV)
    rows = store.as_strided((1, T, 6 * D), (0, far, 1))
    rows.copy_(qkv)
    leaf = rows.requires_grad_(True)
    out = qk_norm_rope(leaf, qw, kw, cos, sin, H)
    near = qkv.clone().requires_grad_(True)
    want = qk_norm_rope(near, qw, kw, cos, sin, H)
    grads = _grads(want)
    for a, b in zip(out, want):
        assert torch.equal(a, b)
    # (autograd.grad of a strided leaf gives its gradient contiguous)
    assert torch.equal(torch.autograd.grad(out, leaf, grads)[0],
                       torch.autograd.grad(want, near, grads)[0])
    kc, vc = (store[1024 * (i + 1):].as_strided((1, Hkv, cap, D), (0, far, D, 1)) for i in (0, 1))
    with torch.no_grad():
        q = qk_norm_rope_append(qkv, qw, kw, cos, sin, H, 0, kc, vc)
    for a, b in zip((q, kc[:, :, :T], vc[:, :, :T]), want):
        assert torch.equal(a, b.detach())


def _append_case():
    qkv, qw, kw, cos, sin = _inputs(1, 2, 2, 2, 64, BF, BF, 6)
    kc, vc = (torch.randn(1, 2, 8, 64, device=DEV).to(BF) for _ in range(2))
    return (qkv, qw, kw, cos, sin), kc, vc


@pytest.mark.parametrize("which", [0, 1])
def test_append_is_seen_by_graphs_that_saved_the_cache(which):
    """The append changes the caches in place: a graph that saved rows of one
    refuses to be differentiated afterwards, as behind torch's own writes."""
    args, *caches = _append_case()
    w = torch.ones(64, device=DEV, dtype=BF, requires_grad=True)
    y = (caches[which][:, :, 3:5] * w).sum()  # w's gradient needs the rows
    at = torch.tensor([3, 4], device=DEV)
    with torch.no_grad():
        versions = [c._version for c in caches]
        qk_norm_rope_append(*args, 2, at, *caches)
        assert all(c._version > v for c, v in zip(caches, versions))
    with pytest.raises(RuntimeError, match="modified"):
        y.backward()
    # a refused call changes nothing
    versions = [c._version for c in caches]
    with pytest.raises(ValueError, match="cache rows"):
        qk_norm_rope_append(*args, 2, 7, *caches)
    assert [c._version for c in caches] == versions


def test_append_into_caches_made_for_inference():
    """Inference tensors have no versions; a cache of them takes the append, in
    and behind inference mode, and so does a plain cache in inference mode."""
    args, kc, vc = _append_case()
    want = [kc.clone(), vc.clone()]
    qk_norm_rope_append(*args, 2, 1, *want)
    with torch.inference_mode():
        mine = [kc.clone(), vc.clone()]
        qk_norm_rope_append(*args, 2, 1, *mine)
        qk_norm_rope_append(*args, 2, 1, kc, vc)
    with torch.no_grad():
        qk_norm_rope_append(*args, 2, 1, *mine)
    for a, b, c in zip(want, mine, (kc, vc)):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_captured_append():
    B, M, H, D, cap = 1, 1, 4, 64, 32
    qkv, qw, kw, _, _ = _inputs(B, M, H, H, D, BF, BF, 0)
    cos, sin = rope_tables(D, cap, DEV)
    kc, vc = (torch.zeros(B, H, cap, D, dtype=BF, device=DEV) for _ in range(2))
    pos = torch.zeros(1, dtype=torch.int64, device=DEV)
    with torch.no_grad():
        qk_norm_rope_append(qkv, qw, kw, cos, sin, H, pos, kc, vc)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            q = qk_norm_rope_append(qkv, qw, kw, cos, sin, H, pos, kc, vc)
    kc.zero_()
    for p in (0, 31, 7, 32):
        pos.fill_(p)
        qkv.copy_(_inputs(B, M, H, H, D, BF, BF, 0, seed=p)[0])
        graph.replay()
        torch.cuda.synchronize()
        if p < cap:
            wq, wk, _ = qk_norm_rope(qkv, qw, kw, cos, sin, H, pos0=p)
            assert torch.equal(q, wq) and torch.equal(kc[:, :, p:p + 1], wk)
        else:
            assert not q.any()


def test_traced_append():
    """A trace, and a call that a dispatch mode watches, hold the append."""
    B, M, H, Hkv, D, cap = 2, 3, 4, 2, 64, 16
    qkv, qw, kw, _, _ = _inputs(B, M, H, Hkv, D, BF, BF, 0)
    cos, sin = rope_tables(D, cap, DEV)
    caches = [torch.zeros(B, Hkv, cap, D, dtype=BF, device=DEV) for _ in range(2)]
    pos = torch.tensor([4, 5, 6], device=DEV)

    def call(x, at, kc, vc):
        return qk_norm_rope_append(x, qw, kw, cos, sin, H, at, kc, vc)

    with torch.no_grad():
        traced = torch.jit.trace(call, (qkv, pos, *caches), check_trace=False)
        for seed in (1, 2):
            x = _inputs(B, M, H, Hkv, D, BF, BF, 0, seed=seed)[0]
            want, got = ([c.clone() for c in caches] for _ in range(2))
            assert torch.equal(traced(x, pos + seed, *got), call(x, pos + seed, *want))
            for a, b in zip(got, want):
                assert torch.equal(a, b) and b[:, :, 4 + seed:7 + seed].any()
    torch.library.opcheck(torch.ops.t2t.qk_norm_rope_append,
                          (qkv, qw, kw, cos, sin, H, pos, 0, *caches, EPS))


def test_another_stream():
    qkv, qw, kw, cos, sin = _inputs(1, 512, 4, 4, 64, BF, BF, 0)
    want = qk_norm_rope(qkv, qw, kw, cos, sin, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        moved = qkv.clone()  # made on the stream that the call has to follow
        got = qk_norm_rope(moved, qw, kw, cos, sin, 4)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_custom_op():
    qkv, qw, kw, cos, sin = _inputs(2, 10, 4, 2, 64, BF, F32, 1)
    for t in (qkv, qw, kw):
        t.requires_grad_(True)
    out = torch.ops.t2t.qk_norm_rope(qkv, qw, kw, cos, sin, 4, 2, 1, EPS)
    grads = _grads(out)
    got = torch.autograd.grad(out, (qkv, qw, kw), grads)
    eager = qk_norm_rope(qkv, qw, kw, cos, sin, 4, 2, pos0=1, eps=EPS)
    want = torch.autograd.grad(eager, (qkv, qw, kw), grads)
    for a, b in zip((*out, *got), (*eager, *want)):
        assert torch.equal(a, b)
    torch.library.opcheck(torch.ops.t2t.qk_norm_rope,
                          (qkv.detach(), qw.detach(), kw.detach(), cos, sin, 4, 2, 1, EPS))


def test_what_else_may_watch_a_call():
    """Traces hold the call, forward-mode levels and batched calls are refused."""
    qkv, qw, kw, cos, sin = _inputs(1, 12, 4, 2, 64, BF, BF, 0)

    def call(x):
        return qk_norm_rope(x, qw, kw, cos, sin, 4, 2)[0]

    other = torch.randn_like(qkv)
    with torch.no_grad():
        traced = torch.jit.trace(call, qkv, check_trace=False)
        assert torch.equal(traced(other), call(other))
    with torch.no_grad(), fwad.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            call(fwad.make_dual(qkv, torch.ones_like(qkv)))
    with torch.no_grad(), pytest.raises(RuntimeError):
        torch.func.vmap(call)(torch.stack([qkv, qkv]))
    q = call(qkv.requires_grad_(True))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(q, qkv, torch.stack([q, q]).detach(), is_grads_batched=True)


def test_leaves_keep_their_gradients_and_hooks():
    """Accumulated gradients, a hook on an output, saved tensors kept elsewhere."""
    qkv, qw, kw, cos, sin = _inputs(1, 30, 4, 4, 64, BF, BF, 0)
    leaves = [t.requires_grad_(True) for t in (qkv, qw, kw)]
    out = qk_norm_rope(*leaves, cos, sin, 4)
    grads = _grads(out)
    want = torch.autograd.grad(out, leaves, grads)
    seen = []
    with torch.autograd.graph.save_on_cpu():
        out = qk_norm_rope(*leaves, cos, sin, 4)
    out[0].register_hook(lambda g: seen.append(g))
    torch.autograd.backward(out, grads)
    assert len(seen) == 1 and torch.equal(seen[0], grads[0])
    for leaf, w in zip(leaves, want):
        assert torch.equal(leaf.grad, w)
    torch.autograd.backward(qk_norm_rope(*leaves, cos, sin, 4), grads)
    for leaf, w in zip(leaves, want):
        assert torch.equal(leaf.grad, w + w)


# ---- refusals that need GPU tensors

def test_refusals():
    qkv, qw, kw, cos, sin = _inputs(1, 4, 2, 1, 64, BF, BF, 0)
    ok = dict(num_kv_heads=1)
    with pytest.raises(ValueError, match="positions"):
        qk_norm_rope(qkv, qw, kw, cos, sin, 2, pos0=cos.shape[0] - 3, **ok)
    with pytest.raises(ValueError, match="positions"):
        qk_norm_rope(qkv, qw, kw, cos, sin, 2, pos0=-1, **ok)
    with pytest.raises(ValueError, match="dtype"):
        qk_norm_rope(qkv, qw, kw.float(), cos, sin, 2, **ok)
    with pytest.raises(RuntimeError, match="GPU"):
        qk_norm_rope(qkv, qw, kw, cos.cpu(), sin.cpu(), 2, **ok)
    with pytest.raises(RuntimeError, match="head dim"):
        qk_norm_rope(qkv[:, :, :4 * 24].contiguous(), qw[:24], kw[:24], cos[:, :12].contiguous(),
                     sin[:, :12].contiguous(), 2, **ok)
    kc, vc = (torch.zeros(1, 1, 8, 64, dtype=BF, device=DEV) for _ in range(2))
    with pytest.raises(ValueError, match="exceed"):
        qk_norm_rope_append(qkv, qw, kw, cos, sin, 2, 5, kc, vc)
    with pytest.raises(ValueError, match="pos"):
        qk_norm_rope_append(qkv, qw, kw, cos, sin, 2, torch.arange(3, device=DEV), kc, vc)
    with pytest.raises(ValueError, match="pos"):
        qk_norm_rope_append(qkv, qw, kw, cos, sin, 2, torch.arange(4), kc, vc)
    with pytest.raises(ValueError, match="dtype"):
        qk_norm_rope_append(qkv, qw, kw, cos, sin, 2, 0, kc.float(), vc.float())
    with pytest.raises(RuntimeError, match="overlap"):
        qk_norm_rope_append(qkv, qw, kw, cos, sin, 2, 0, kc[:, :, :1].expand(1, 1, 8, 64), vc)
    with pytest.raises(RuntimeError, match="are one"):
        qk_norm_rope_append(qkv, qw, kw, cos, sin, 2, 0, kc, kc)
    with pytest.raises(RuntimeError, match="boundary"):
        odd = torch.zeros(8 * 64 + 1, dtype=BF, device=DEV)[1:].view(1, 1, 8, 64)
        qk_norm_rope_append(qkv, qw, kw, cos, sin, 2, 0, odd, vc)
    with pytest.raises(RuntimeError, match="at most 8"):
        wide = qkv.new_zeros(1, 9, 4 * 64)
        big = torch.zeros(1, 1, 16, 64, dtype=BF, device=DEV)
        cos, sin = rope_tables(64, 16, DEV)
        qk_norm_rope_append(wide, qw, kw, cos, sin, 2, torch.arange(9, device=DEV), big,
                            big.clone())
    with pytest.raises(RuntimeError, match="no gradient"):
        qk_norm_rope_append(qkv.requires_grad_(True), qw, kw, cos, sin, 2, 0, kc, vc)


@pytest.mark.parametrize("which", [0, 1])
def test_append_refuses_caches_with_a_gradient(which):
    args, *caches = _append_case()
    caches[which].requires_grad_(True)
    before = [c.detach().clone() for c in caches]
    with pytest.raises(RuntimeError, match="no gradient"):
        qk_norm_rope_append(*args, 2, 1, *caches)
    assert all(torch.equal(a, b) for a, b in zip(before, caches))
    with torch.no_grad():  # as torch's own writes into a leaf
        qk_norm_rope_append(*args, 2, 1, *caches)
    assert not torch.equal(before[which], caches[which])
