"""GPU checks of the scaled embedding (t2t_embedding) and its weight gradient
(t2t_embedding_backward) against sums in 64 bits.

Tolerances count roundings, U = 2^-24 for a step of fp32: the lookup rounds the
scale and the product (2 U) and once to the type (eps / 2); a gradient row of n
positions adds n terms (each addition U of the sum of |terms| at most) and
scales (2 U), then rounds once.
"""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from tagseq2tagseq_amd.embedding import ScaledEmbedding, embedding

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
U = 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32


def _case(N, V, C, dt, seed=0, skew=True):
    g = torch.Generator().manual_seed(seed + 7 * N + V + C)
    if skew:  # frequent low ids, as token ids are
        u = torch.rand(N, generator=g, dtype=torch.float64)
        tokens = ((V + 1.0) ** u - 1).long().clamp_(max=V - 1)
    else:
        tokens = torch.randint(0, V, (N,), generator=g)
    w = torch.randn(V, C, generator=g).to(dt)
    dy = torch.randn(N, C, generator=g).to(dt)
    return tokens.to(DEV), w.to(DEV), dy.to(DEV)


def _check_rows(out, tokens, w, scale):
    ref = w.double()[tokens] * scale
    tol = (torch.finfo(w.dtype).eps / 2 + 3 * U) * ref.abs() + 1e-37
    assert out.dtype == w.dtype and out.shape == ref.shape
    assert bool(((out.double() - ref).abs() <= tol).all())


def _check_grad(dw, tokens, dy, V, scale, skip=()):
    keep = torch.ones_like(tokens, dtype=torch.bool)
    for t in skip:
        keep &= tokens != t
    t, d = tokens[keep], dy.double()[keep]
    shape = (V, dy.shape[1])
    ref = torch.zeros(shape, dtype=torch.float64, device=DEV).index_add_(0, t, d) * scale
    size = torch.zeros(shape, dtype=torch.float64, device=DEV).index_add_(0, t, d.abs())
    n = torch.bincount(t, minlength=V).double()[:, None]
    tol = (torch.finfo(dy.dtype).eps / 2 * ref.abs() + (n + 4) * U * abs(scale) * size + 1e-37)
    assert dw.dtype == dy.dtype and dw.shape == shape
    err = (dw.double() - ref).abs()
    assert bool((err <= tol).all()), f"{float((err / tol).max()):.3g} of the tolerance"
    # rows without a position are zero, not small
    assert not dw[n[:, 0] == 0].any()


@pytest.mark.parametrize("N,V,C,dt,scale", [
    (1, 1, 8, BF, 1.0), (1, 50257, 768, BF, 27.7), (2, 3, 1, F32, 2.0), (5, 11, 7, BF, -1.5),
    (17, 600, 64, F32, 1.0), (300, 40, 520, BF, 22.6), (1537, 8192, 512, F32, 22.6),
    (4096, 50257, 768, BF, 27.7), (2049, 1000, 100, BF, 3.0), (333, 513, 30, F32, 0.1),
    (16384, 700, 96, BF, 9.8), (40000, 3000, 24, F32, 1.0), (33000, 200000, 264, BF, 1.0),
    (3, 5, 1 << 20, BF, 1.0), (2500, 5, 30001, F32, 1.0), (3, 1 << 20, 8, BF, 2.0),
    (2100, 1 << 20, 8, F32, 2.0),
])
def test_rows_and_gradient(N, V, C, dt, scale):
    tokens, w, dy = _case(N, V, C, dt)
    w.requires_grad_(True)
    out = embedding(tokens, w, scale)
    _check_rows(out.detach(), tokens, w.detach(), scale)
    (dw,) = torch.autograd.grad(out, w, dy)
    _check_grad(dw, tokens, dy, V, scale)
    # the same bits again, and without autograd
    (again,) = torch.autograd.grad(embedding(tokens, w, scale), w, dy)
    assert torch.equal(dw, again)
    assert torch.equal(out.detach(), embedding(tokens, w.detach(), scale))


@pytest.mark.parametrize("N", [1, 15, 16, 17, 63, 64, 65, 66, 1000, 2047, 2048, 2049, 2064, 2065,
                               4097, 32768, 32769, 32800, 70000])
def test_one_token_throughout(N):
    """A token that crosses every piece of the list; its neighbours get zeros."""
    C = 40
    _, w, dy = _case(N, 9, C, F32)
    tokens = torch.full((N,), 4, device=DEV)
    w.requires_grad_(True)
    (dw,) = torch.autograd.grad(embedding(tokens, w, 1.0), w, dy)
    _check_grad(dw, tokens, dy, 9, 1.0)


@pytest.mark.parametrize("more", [0, 2048, 32768])
@pytest.mark.parametrize("lengths", [(16, 16, 16), (15, 1, 16), (1, 31, 1), (40, 3, 50, 5),
                                     (17, 64, 15, 1, 1, 1), (5, 200, 5), (64, 65, 66),
                                     (32, 32, 33, 31, 600, 1)])
def test_runs_that_end_at_and_cross_pieces(lengths, more):
    """Runs of equal tokens (ids of one work-group, in ascending order) of
    given lengths behind one of `more`, in shuffled positions: short lists, and
    longer ones with pieces of 16 and of 32."""
    lengths = (more,) * (more > 0) + lengths
    ids = torch.cat([torch.full((n,), 512 * i + 3) for i, n in enumerate(lengths)])
    g = torch.Generator().manual_seed(len(ids))
    tokens = ids[torch.randperm(len(ids), generator=g)].to(DEV)
    V, C = 512 * len(lengths), 24
    _, w, _ = _case(1, V, C, F32)
    dy = torch.randn(len(ids), C, generator=g).to(DEV)
    w.requires_grad_(True)
    (dw,) = torch.autograd.grad(embedding(tokens, w, 1.0), w, dy)
    _check_grad(dw, tokens, dy, V, 1.0)


@pytest.mark.parametrize("more", [0, 3000])
def test_order_of_the_positions(more):
    """Additions in the order of the positions: 2^24 + 1 - 2^24 is 0 in fp32, and
    2^24 - 2^24 + 1 is 1."""
    big = 2.0 ** 24
    tokens = torch.tensor([5, 9, 5, 9, 5, 9] + [3] * more, device=DEV)
    vals = torch.tensor([big, big, 1.0, -big, -big, 1.0] + [0.0] * more, device=DEV)
    w = torch.zeros(10, 4, device=DEV, requires_grad=True)
    (dw,) = torch.autograd.grad(embedding(tokens, w), w, vals[:, None].expand(6 + more, 4))
    assert dw[5].tolist() == [0.0] * 4 and dw[9].tolist() == [1.0] * 4


@pytest.mark.parametrize("N", [400, 5000])
@pytest.mark.parametrize("pad", [0, 7, -1])
def test_padding_row(pad, N):
    V, C = 50, 32
    tokens, w, dy = _case(N, V, C, BF)
    tokens[::3] = pad % V
    w.requires_grad_(True)
    out = embedding(tokens, w, 2.0, padding_idx=pad)
    _check_rows(out.detach(), tokens, w.detach(), 2.0)  # it is looked up like any row
    (dw,) = torch.autograd.grad(out, w, dy)
    _check_grad(dw, tokens, dy, V, 2.0, skip=(pad % V,))
    assert not dw[pad].any()


@pytest.mark.parametrize("N", [64, 3000, 40000])
def test_ids_outside_the_table(N):
    V, C = 20, 16
    tokens, w, dy = _case(N, V, C, BF)
    bad = {3: -1, 10: V, 40: 1 << 40, 41: -(1 << 62), 63: (1 << 32) + 2}
    for i, t in bad.items():
        tokens[i] = t
    w.requires_grad_(True)
    out = embedding(tokens, w, 1.0)
    rows = torch.zeros(N, dtype=torch.bool, device=DEV)
    rows[list(bad)] = True
    assert out[rows].isnan().all() and not out[~rows].isnan().any()
    _check_rows(out.detach()[~rows], tokens[~rows], w.detach(), 1.0)
    (dw,) = torch.autograd.grad(out, w, dy)
    _check_grad(dw, tokens[~rows], dy[~rows], V, 1.0)


def test_values_that_are_not_finite_stay_in_their_rows():
    tokens, w, dy = _case(200, 30, 24, F32, skew=False)
    dy[7] = float("nan")
    dy[9, 3] = float("inf")
    w.requires_grad_(True)
    (dw,) = torch.autograd.grad(embedding(tokens, w), w, dy)
    a, b = int(tokens[7]), int(tokens[9])
    assert dw[a].isnan().all()
    if a != b:
        assert dw[b, 3] == float("inf") and dw[b].isinf().sum() == 1
    rest = torch.ones(30, dtype=torch.bool, device=DEV)
    rest[[a, b]] = False
    assert dw[rest].isfinite().all()


@pytest.mark.parametrize("dt", [BF, F32])
def test_strides_and_alignments(dt):
    N, V, C = 77, 90, 48
    tokens, w, dy = _case(N, V, C, dt)
    want = embedding(tokens, w, 3.0)
    leaf = w.clone().requires_grad_(True)
    (want_dw,) = torch.autograd.grad(embedding(tokens, leaf, 3.0), leaf, dy)
    for pad, off in ((16, 0), (5, 1)):
        big = torch.zeros(V, C + pad, dtype=dt, device=DEV)
        view = big[:, off:off + C]
        view.copy_(w)
        assert torch.equal(embedding(tokens, view, 3.0), want)
        grad = torch.zeros(N, C + pad, dtype=dt, device=DEV)[:, off:off + C]
        grad.copy_(dy)
        (dw,) = torch.autograd.grad(embedding(tokens, leaf, 3.0), leaf, grad)
        assert torch.equal(dw, want_dw)
    turned = w.t().contiguous().t()
    assert torch.equal(embedding(tokens, turned, 3.0), want)
    (dw,) = torch.autograd.grad(embedding(tokens, leaf, 3.0), leaf, dy.t().contiguous().t())
    assert torch.equal(dw, want_dw)
    strided = torch.stack((tokens, tokens + 1), 1)[:, 0]
    assert torch.equal(embedding(strided, w, 3.0), want)
    assert torch.equal(embedding(tokens.int(), w, 3.0), want)
    # one gradient for all rows
    one = torch.ones((), dtype=dt, device=DEV)
    (a,) = torch.autograd.grad(embedding(tokens, leaf, 3.0), leaf, one.expand(N, C))
    (b,) = torch.autograd.grad(embedding(tokens, leaf, 3.0), leaf, torch.ones_like(dy))
    assert torch.equal(a, b)
    (a,) = torch.autograd.grad(embedding(tokens, leaf, 3.0), leaf, dy[:1].expand(N, C))
    (b,) = torch.autograd.grad(embedding(tokens, leaf, 3.0), leaf, dy[:1].repeat(N, 1))
    assert torch.equal(a, b)


def test_shapes():
    w = torch.randn(12, 16, device=DEV, requires_grad=True)
    for shape in ((), (3,), (2, 0), (0,), (2, 3, 4)):
        tokens = torch.randint(0, 12, shape, device=DEV)
        out = embedding(tokens, w, 2.0)
        assert out.shape == (*shape, 16)
        (dw,) = torch.autograd.grad(out, w, torch.ones_like(out))
        n = torch.bincount(tokens.reshape(-1), minlength=12).float()
        assert torch.equal(dw, (2 * n)[:, None].expand(12, 16))


def test_gradient_against_differences():
    """The lookup is linear in the table, so central differences of the plain
    form in 64 bits are exact to 2^-53; the float32 gradient has the tolerance
    of its sums (at most 50 positions a token: 54 U of the sum of |terms|)."""
    tokens, w, dy = _case(50, 6, 8, F32)
    w.requires_grad_(True)
    (dw,) = torch.autograd.grad(embedding(tokens, w, 1.25), w, dy)
    base, gen = w.detach().double(), torch.Generator().manual_seed(2)
    f = lambda x: (1.25 * x[tokens] * dy.double()).sum()  # noqa: E731
    for _ in range(4):
        u = torch.randn(w.shape, generator=gen, dtype=torch.float64).to(DEV)
        diff = float(f(base + 0.5 * u) - f(base - 0.5 * u))
        size = float((1.25 * u.abs()[tokens] * dy.double().abs()).sum())
        assert abs(diff - float((dw.double() * u).sum())) <= 54 * U * size + 1e-12 * size


def test_offsets_past_32_bits():
    """A table and a gradient of more than 2^32 elements, rows of dy as far apart."""
    V, C = 1 << 20, 4104
    ids = torch.tensor([V - 1, 0, V - 2, V - 1, 1 << 19], device=DEV)
    w = torch.empty(V, C, dtype=BF, device=DEV)
    g = torch.Generator().manual_seed(3)
    rows, dy = (torch.randn(5, C, generator=g).to(BF).to(DEV) for _ in range(2))
    w[ids] = rows
    out = embedding(ids, w, 2.0)
    assert torch.equal(out, w[ids] * 2)
    far = torch.empty(4 * (1 << 30) + C, dtype=BF, device=DEV).as_strided((5, C), (1 << 30, 1))
    far.copy_(dy)
    w.requires_grad_(True)
    (dw,) = torch.autograd.grad(embedding(ids, w, 2.0), w, far)
    d = dy.double()
    want = {V - 1: d[0] + d[3], 0: d[1], V - 2: d[2], 1 << 19: d[4]}
    for v, ref in want.items():
        tol = (torch.finfo(BF).eps / 2 + 6 * U) * 2 * ref.abs() + 4 * U * 16
        assert bool(((dw[v].double() - 2 * ref).abs() <= tol).all())
    dw[ids] = 0
    assert not any(bool(part.any()) for part in dw.split(1 << 17))


def test_captured_lookup_and_gradient():
    tokens, w, dy = _case(1000, 500, 64, BF)
    w.requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = embedding(tokens, w, 2.0)
        torch.autograd.grad(out, w, dy)
        del out
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = embedding(tokens, w, 2.0)
        (dw,) = torch.autograd.grad(out, w, dy)
    for seed in range(4):
        t, _, d = _case(1000, 500, 64, BF, seed=50 + seed)
        tokens.copy_(t if seed != 2 else torch.full_like(t, 7))
        dy.copy_(d)
        graph.replay()
        torch.cuda.synchronize()
        fresh = w.detach().clone().requires_grad_(True)
        eager = embedding(tokens, fresh, 2.0)
        assert torch.equal(out, eager)
        assert torch.equal(dw, torch.autograd.grad(eager, fresh, dy)[0])


def test_another_stream():
    tokens, w, dy = _case(3000, 800, 64, BF)
    leaf = w.clone().requires_grad_(True)
    (want,) = torch.autograd.grad(embedding(tokens, leaf), leaf, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        moved = w.clone().requires_grad_(True)
        (got,) = torch.autograd.grad(embedding(tokens.clone(), moved), moved, dy.clone())
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_module_and_custom_op():
    m = ScaledEmbedding(60, 32, scale=5.5, padding_idx=3, device=DEV, dtype=BF)
    tokens = torch.randint(0, 60, (4, 9), device=DEV)
    out = m(tokens)
    _check_rows(out.detach().reshape(-1, 32), tokens.reshape(-1), m.weight.detach(), 5.5)
    dy = torch.randn_like(out)
    (dw,) = torch.autograd.grad(out, m.weight, dy)
    w = m.weight.detach().clone().requires_grad_(True)
    op = torch.ops.t2t.embedding(tokens, w, 5.5, 3)
    assert torch.equal(op, out) and torch.equal(torch.autograd.grad(op, w, dy)[0], dw)
    torch.library.opcheck(torch.ops.t2t.embedding, (tokens, w.detach(), 5.5, 3))


def test_what_else_may_watch_a_call():
    """Traces hold the call, forward-mode levels and batched calls are refused."""
    tokens, w, dy = _case(30, 20, 16, BF)

    def call(x):
        return embedding(tokens, x, 2.0)

    other = torch.randn_like(w)
    with torch.no_grad():
        traced = torch.jit.trace(call, w, check_trace=False)
        assert torch.equal(traced(other), call(other))
    with torch.no_grad(), fwad.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            call(fwad.make_dual(w, torch.ones_like(w)))
    with torch.no_grad(), pytest.raises(RuntimeError):
        torch.func.vmap(call)(torch.stack([w, w]))
    out = call(w.requires_grad_(True))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, w, torch.stack([dy, dy]), is_grads_batched=True)


def test_second_order_is_refused():
    tokens, w, _ = _case(5, 6, 8, F32)
    w.requires_grad_(True)
    (d,) = torch.autograd.grad((embedding(tokens, w) ** 2).sum(), w, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), w)


def test_refusals():
    tokens, w, _ = _case(5, 6, 8, F32)
    with pytest.raises(RuntimeError, match="GPU"):
        embedding(tokens.cpu(), w)
    with pytest.raises(ValueError, match="tokens must"):
        embedding(tokens.float(), w)
    with pytest.raises(NotImplementedError, match="dtype"):
        embedding(tokens, w.half())
