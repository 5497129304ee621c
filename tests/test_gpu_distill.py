"""GPU checks of the distillation loss (t2t_distill_rows) and its gradient, for
given logits and with the linear head, against a plain implementation in 64
bits.

Tolerances count roundings, U = 2^-24 for a step of fp32.  With x = (z - max) / T:
  e^x      the difference (U |z - max| / T), two products, the exponential (2 U):
           a relative error of (3 |x| + 4) U.
  S        the sum of e^x: E[3 |x|] + 4 under the softmax, and the chain of
           additions, at most ceil(V / 256) + 20: a relative error rel(S).
  ln S     rel(S) + 4 (1 + ln S) U.
  KD       the weighted sum of differences, each of a weight with a relative
           error of (3 |x_t| + 8 + K) U, and the two logarithms.
  grad_j   each of its terms (soft, hard, the slots', the target's) with its
           exponential's, its sum's and 10 more roundings; one rounding to the
           type (half a step, eps / 2); exponentials under 2^-126 are 0.
"""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwad
import torch.utils.checkpoint

from tagseq2tagseq_amd.distill import LinearDistillLoss, distill_loss, head_distill
from tagseq2tagseq_amd.head_loss import head_cross_entropy

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
U = 2.0 ** -24
BF, F32, I32, I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64
IGNORE = -100


def _case(N, V, K, dt, tdt=F32, idt=I64, seed=0, empty=True):
    g = torch.Generator().manual_seed(seed + 13 * N + V + K)
    z = 2.5 * torch.randn(N, V, generator=g)
    # distinct columns: a walk with a step that K of them fit
    step = torch.randint(1, max(1, V // max(K, 1)) + 1, (N, 1), generator=g)
    idx = (torch.randint(0, V, (N, 1), generator=g) + step * torch.arange(K)) % V
    t = 6 - 1.5 * torch.log1p(torch.arange(K, dtype=F32)) + torch.randn(N, K, generator=g)
    if K <= V:
        z.scatter_(1, idx, 0.6 * t + torch.randn(N, K, generator=g))
    if empty and K > 1:
        keep = torch.where(torch.rand(N, 1, generator=g) < 0.4,
                           torch.randint(0, K + 1, (N, 1), generator=g), K)
        idx = torch.where(torch.arange(K) < keep, idx, -1 - torch.arange(K))
    target = torch.randint(0, V, (N,), generator=g)
    if K:
        target = torch.where((idx[:, 0] >= 0) & (torch.rand(N, generator=g) < 0.5), idx[:, 0],
                             target)
    target[torch.rand(N, generator=g) < 0.2] = IGNORE
    target[0] = 0
    return (z.to(dt).to(DEV), idx.to(idt).to(DEV), t.to(tdt).to(DEV), target.to(DEV))


def _reference(z, idx, t, target, tau, alpha):
    """In 64 bits: row losses, their tolerance, gradients (of each row's own
    loss), and what their roundings are relative to, in units of U."""
    tau, alpha = float(tau), float(alpha)
    z, t = z.double(), t.double()
    N, V = z.shape
    K = idx.shape[1]
    valid = idx >= 0
    at = torch.where(valid, idx.long(), 0)
    m = z.amax(1, keepdim=True)

    def softmax(T):
        x = (z - m) / T
        e = torch.exp(x)
        S = e.sum(1, keepdim=True)
        q = e / S
        # (0 of a masked column is exact)
        far = torch.where(q > 0, x.abs(), 0.0)
        rel = 3 * (q * far).sum(1, keepdim=True) + 4 + math.ceil(V / 256) + 20
        return q, S, far, rel

    q, S, far, rel = softmax(tau)
    h, Sh, farh, relh = softmax(1.0)
    mt = torch.where(valid, t, -math.inf).amax(1, keepdim=True) if K else z.new_zeros(N, 1)
    taught = valid.any(1, keepdim=True) & (mt != -math.inf)
    mt = torch.where(taught, mt, 0.0)
    xt = torch.where(valid, (t - mt) / tau, -math.inf)
    w = torch.exp(xt)
    St = w.sum(1, keepdim=True).clamp(min=1e-300)
    p = w / St
    live = p > 0
    xt = torch.where(live, xt, 0.0)
    zs = torch.where(live, (z.gather(1, at) - m) / tau, 0.0)
    kd = (torch.where(live, p * (xt - zs), 0.0).sum(1, keepdim=True) - St.log() + S.log())
    tol_f = torch.where(live, p * (3 * xt.abs() + 8 + K) * (xt.abs() + zs.abs() + 1), 0.0).sum(
        1, keepdim=True)
    rel_t = (p * 3 * xt.abs()).sum(1, keepdim=True) + 4 + K
    tol_kd = tol_f + rel + rel_t + 4 * (2 + S.log() + St.log().abs()) + tol_f / 4
    rows = torch.where(taught, alpha * tau ** 2 * kd, 0.0)
    tol = torch.where(taught, alpha * tau ** 2 * (tol_kd + 6 * kd.abs()), 0.0)
    # gradient terms
    soft = torch.where(taught, alpha * tau * q, 0.0)
    grad = soft.clone()
    size = soft * (3 * far + rel + 14)
    pk = torch.where(taught & live, alpha * tau * p, 0.0)
    grad.scatter_add_(1, at, -pk)
    size.scatter_add_(1, at, pk * (3 * xt.abs() + rel_t + 14 + K))
    if alpha < 1:
        tgt = torch.where(target == IGNORE, 0, target)[:, None]
        zt = (z - m).gather(1, tgt)
        rows = rows + (1 - alpha) * (Sh.log() - zt)
        tol = tol + (1 - alpha) * (relh + 4 * (1 + Sh.log()) + 3 * zt.abs())
        grad += (1 - alpha) * h
        size += (1 - alpha) * h * (3 * farh + relh + 14)
        one = torch.full_like(tgt, 1, dtype=torch.float64) * (1 - alpha)
        grad.scatter_add_(1, tgt, -one)
        size.scatter_add_(1, tgt, 14 * one)
    rows, tol = rows[:, 0], tol[:, 0] + 4 * rows[:, 0].abs()
    if target is not None:
        out = target == IGNORE
        rows, tol = rows.masked_fill(out, 0), tol.masked_fill(out, 0)
        grad, size = grad.masked_fill(out[:, None], 0), size.masked_fill(out[:, None], 0)
    return rows, tol * U, grad, size * U


def _within(got, ref, tol, what):
    err = (got.double() - ref).abs()
    assert got.shape == ref.shape and bool((err <= tol).all()), (
        f"{what}: {float((err / tol.clamp(min=1e-300)).max()):.3g} of the tolerance")


def _grad_tol(dt, ref, size):
    return torch.finfo(dt).eps / 2 * ref.abs() + size + 1e-37


def _check(z, idx, t, target, tau, alpha):
    """Row losses, and mean and sum with their gradients."""
    kw = dict(temperature=tau, alpha=alpha, ignore_index=IGNORE)
    rows, tol, grad, size = _reference(z, idx, t, target, tau, alpha)
    got = distill_loss(z, idx, t, target, reduction="none", **kw)
    assert got.dtype == F32
    _within(got, rows, tol + 1e-37, "rows")
    n = rows.numel() if target is None else int((target != IGNORE).sum())
    leaf = z.clone().requires_grad_(True)
    loss = distill_loss(leaf, idx, t, target, **kw)
    # the sum is in 64 bits; 1 / n, the product and the result round
    _within(loss.detach(), rows.sum() / n, (tol.sum() + 4 * U * rows.abs().sum()) / n, "mean")
    (dz,) = torch.autograd.grad(loss, leaf)
    assert dz.dtype == z.dtype
    _within(dz, grad / n, _grad_tol(z.dtype, grad / n, size / n), "gradient")
    assert torch.equal(loss.detach(), distill_loss(z, idx, t, target, **kw))
    return loss.detach(), dz


SHAPES = [
    # N, V, K, logits, teacher, indices, tau, alpha
    (1, 1, 1, BF, BF, I64, 1.0, 1.0),
    (5, 7, 3, BF, F32, I32, 2.0, 0.5),
    (6, 8, 8, F32, F32, I64, 0.7, 0.3),
    (33, 300, 8, F32, BF, I32, 0.5, 1.0),
    (17, 1003, 64, BF, BF, I64, 2.0, 0.5),
    (9, 1003, 300, F32, F32, I64, 1.0, 0.4),
    (9, 50257, 64, BF, BF, I32, 2.0, 0.5),
    (7, 50257, 32, BF, F32, I64, 1.0, 1.0),
    (4, 8193, 1024, F32, F32, I64, 3.0, 0.9),
    (3, 5000, 5, BF, BF, I64, 1.0, 0.0),
    (3, 140001, 40, BF, F32, I64, 1.7, 0.5),  # wider than the registers hold
    (2, 70003, 40, F32, F32, I64, 1.0, 1.0),
]


@pytest.mark.parametrize("N,V,K,dt,tdt,idt,tau,alpha", SHAPES)
def test_loss_and_gradient(N, V, K, dt, tdt, idt, tau, alpha):
    _check(*_case(N, V, K, dt, tdt, idt), tau, alpha)


@pytest.mark.parametrize("V", [2047, 4097, 8200, 16391, 33001, 41000, 49160, 57400, 65537, 98304,
                               131077])
def test_every_width_of_the_held_row(V):
    _check(*_case(3, V, 16, BF, seed=1), 1.5, 0.5)


@pytest.mark.parametrize("V", [1023, 2049, 4101, 8203, 16390, 20480, 24570, 28676, 32769, 49153,
                               65539])
def test_every_width_of_the_held_float32_row(V):
    _check(*_case(2, V, 16, F32, seed=1), 1.0, 0.5)


@pytest.mark.parametrize("dt", [BF, F32])
def test_widest_row(dt):
    V = 1 << 28
    g = torch.Generator(device=DEV).manual_seed(1)
    z = torch.randn(1, V, generator=g, device=DEV, dtype=dt)
    idx = torch.tensor([[V - 1, 5, -1, V // 2]], device=DEV)
    _check(z, idx, torch.tensor([[2.0, 1.0, 9.0, 0.5]], device=DEV),
           torch.tensor([V - 1], device=DEV), 2.0, 0.5)


def test_without_targets():
    z, idx, t, _ = _case(40, 777, 12, BF)
    _check(z, idx, t, None, 2.0, 1.0)


def test_targets_only_mask_at_alpha_one():
    z, idx, t, target = _case(40, 777, 12, BF)
    loss, dz = _check(z, idx, t, target, 2.0, 1.0)
    moved = torch.where(target == IGNORE, target, (target + 5) % 777)
    again, dz2 = _check(z, idx, t, moved, 2.0, 1.0)
    assert torch.equal(loss, again) and torch.equal(dz, dz2)


def test_no_slots_is_the_cross_entropy():
    z, idx, t, target = _case(12, 500, 4, F32)
    a = distill_loss(z, idx[:, :0], t[:, :0], target, alpha=0.25, ignore_index=IGNORE)
    b = distill_loss(z, torch.full_like(idx, -1), t, target, alpha=0.25, ignore_index=IGNORE)
    assert torch.equal(a, b)
    _check(z, torch.full_like(idx, -1), t, target, 2.0, 0.25)
    # and nothing without hard labels
    leaf = z.clone().requires_grad_(True)
    loss = distill_loss(leaf, torch.full_like(idx, -1), t, target)
    (dz,) = torch.autograd.grad(loss, leaf)
    assert float(loss) == 0.0 and not dz.any()


def test_slots_of_the_same_column_add_up():
    z, idx, t, target = _case(8, 64, 6, F32, empty=False)
    idx[:, 3] = idx[:, 1]
    idx[::2, 5] = idx[::2, 1]
    idx[1] = idx[1, 0]
    _check(z, idx, t, target, 1.5, 0.5)


def test_teacher_masks():
    z, idx, t, target = _case(6, 90, 5, F32, empty=False)
    inf = math.inf
    t[0, 2] = -inf                      # a slot without mass
    t[1] = -inf                         # no slot with mass
    t[2] = torch.finfo(F32).min         # all at the lowest value: uniform
    t[3, 1:] = torch.finfo(F32).min     # mass on one slot
    idx[4] = -1
    target[:] = torch.arange(6, device=DEV)
    _check(z, idx, t, target, 2.0, 0.5)
    none = distill_loss(z, idx, t, reduction="none")
    assert none[1] == 0 and none[4] == 0
    t[5, 3] = float("nan")
    assert distill_loss(z, idx, t, reduction="none")[5].isnan()
    t[5] = float("nan")
    assert distill_loss(z, idx, t, reduction="none")[5].isnan()


@pytest.mark.parametrize("dt", [BF, F32])
def test_masked_logits(dt):
    """Columns of -inf and of the lowest value, off the slots and the target."""
    z, idx, t, target = _case(8, 203, 4, dt, empty=False)
    used = torch.zeros_like(z, dtype=torch.bool).scatter_(1, idx, True)
    used.scatter_(1, target.clamp(min=0)[:, None], True)
    gone = ~used & (torch.rand_like(z, dtype=F32) < 0.5)
    for value in (-math.inf, torch.finfo(dt).min):
        zz = z.masked_fill(gone, value)
        _, dz = _check(zz, idx, t, target, 2.0, 0.5)
        assert not dz[gone].any()
    # a whole row at the lowest value is uniform
    zz = torch.full_like(z, torch.finfo(dt).min)
    _check(zz, idx, t, target, 2.0, 0.5)


@pytest.mark.parametrize("tau", [1 / 64, 0.5, 1.0, 2.0, 4.0])
@pytest.mark.parametrize("dt,V", [(BF, 203), (F32, 203), (BF, 131080), (F32, 65544)])
def test_rows_far_from_zero(dt, V, tau):
    """Rows wholly, or but for one column, at a value far from 0, and columns far
    above the others.  A sum's exponentials are those of differences to the row's
    maximum, whatever its size, so the tolerances at the head hold as they are
    (temperatures are powers of two: T and 1 / T are exact)."""
    far = (-1e4, -1e9, -1e10, -1e12, -1e30)
    z, idx, t, target = _case(2 * len(far) + 3, V, 4, dt, empty=False)
    for i, value in enumerate(far):
        z[i] = value
        z[len(far) + i] = value
        z[len(far) + i, 17] = 0.5
    z[-3, 17], z[-2, 17] = 1e10, 1e20
    target[:] = torch.arange(len(target), device=DEV)
    for alpha in (0.5, 1.0):
        _check(z, idx, t, target, tau, alpha)
        _, _, grad, size = _reference(z, idx, t, target, tau, alpha)
        leaf, g = z.clone().requires_grad_(True), torch.tensor(-1 / 3, device=DEV)
        loss = distill_loss(leaf, idx, t, target, temperature=tau, alpha=alpha, reduction="sum")
        (dz,) = torch.autograd.grad(loss, leaf, g)
        f = g.double()
        _within(dz, grad * f, _grad_tol(dt, grad * f, size * f.abs()), "scaled gradient")


def test_rows_that_are_not_numbers():
    z, idx, t, target = _case(8, 99, 4, F32, empty=False)
    target[:] = 7
    clean = distill_loss(z, idx, t, target, alpha=0.5, reduction="none")
    leaf = z.clone()
    leaf[1, 50] = float("nan")
    leaf[2] = -math.inf
    leaf[3, 20] = math.inf
    leaf[4, int(idx[4, 1])] = -math.inf     # the teacher wants what the student excludes
    leaf.requires_grad_(True)
    rows = distill_loss(leaf, idx, t, target, alpha=0.5, reduction="none")
    assert rows[1:4].isnan().all() and rows[4] == math.inf
    keep = [0, 5, 6, 7]
    assert torch.equal(rows[keep].detach(), clean[keep])
    (dz,) = torch.autograd.grad(rows, leaf, torch.ones_like(rows))
    assert dz[1].isnan().all() and dz[2].isnan().all() and dz[4:].isfinite().all()
    # rows that do not count are not read
    target[1:4] = IGNORE
    loss = distill_loss(leaf, idx, t, target, alpha=0.5, reduction="none", ignore_index=IGNORE)
    assert torch.equal(loss[1:4], torch.zeros(3, device=DEV))
    (dz,) = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
    assert not dz[1:4].any()


def test_columns_and_targets_outside_the_vocabulary():
    z, idx, t, target = _case(6, 120, 4, BF, empty=False)
    target[:] = 3
    idx[1, 2] = 120
    idx[2, 0] = 1 << 40
    target[3] = 120
    target[4] = -7
    leaf = z.clone().requires_grad_(True)
    rows = distill_loss(leaf, idx, t, target, alpha=0.5, reduction="none", ignore_index=IGNORE)
    assert rows[1:5].isnan().all() and rows[[0, 5]].isfinite().all()
    (dz,) = torch.autograd.grad(rows, leaf, torch.ones_like(rows))
    assert not dz[1:5].any() and dz[[0, 5]].any()
    assert distill_loss(z, idx, t, target, alpha=0.5).isnan()
    # alpha 0: the teacher has no say, whatever its columns
    target[:] = 3
    idx[:, 0] = (1 << 32) + 3
    idx[:, 1] = 3
    want = distill_loss(leaf, idx[:, :0], t[:, :0], target, alpha=0.0)
    got = distill_loss(leaf, idx, t, target, alpha=0.0)
    assert torch.equal(got, want) and got.isfinite()
    assert torch.equal(*(torch.autograd.grad(x, leaf)[0] for x in (got, want)))


def test_more_rows_than_a_launch_takes():
    """The rows at and behind the end of a launch, against the same rows alone."""
    N, V, K = (1 << 21) + 70, 40, 2
    g = torch.Generator(device=DEV).manual_seed(5)
    z = torch.randn(N, V, generator=g, device=DEV).to(BF).requires_grad_(True)
    idx = torch.randint(-1, V, (N, K), generator=g, device=DEV)
    t = torch.randn(N, K, generator=g, device=DEV)
    target = torch.randint(0, V, (N,), generator=g, device=DEV)
    up = torch.randn(N, generator=g, device=DEV)
    kw = dict(temperature=2.0, alpha=0.5, reduction="none")
    rows = distill_loss(z, idx, t, target, **kw)
    (dz,) = torch.autograd.grad(rows, z, up)
    for part in (slice(0, 64), slice((1 << 21) - 64, N)):
        alone = z.detach()[part].clone().requires_grad_(True)
        want = distill_loss(alone, idx[part], t[part], target[part], **kw)
        (d,) = torch.autograd.grad(want, alone, up[part])
        # (rows of 80 bytes: whole pieces from the same column on in both)
        assert torch.equal(rows[part], want) and torch.equal(dz[part], d)


def test_offsets_past_32_bits():
    """Logit rows, ids and teacher rows more than 2^32 elements apart in all."""
    z, idx, t, target = _case(5, 1000, 8, BF)

    def far(x):
        step = 1 << 30
        rows = torch.empty(4 * step + x.shape[1], dtype=x.dtype, device=DEV).as_strided(
            x.shape, (step, 1))
        rows.copy_(x)
        return rows

    kw = dict(temperature=2.0, alpha=0.5, reduction="none")
    a, b = far(z).requires_grad_(True), z.clone().requires_grad_(True)
    got = distill_loss(a, far(idx.int()), far(t.to(BF)), target, **kw)
    want = distill_loss(b, idx.int(), t.to(BF), target, **kw)
    up = torch.arange(1.0, 6.0, device=DEV)
    assert torch.equal(got, want)  # (rows of 2000 bytes: 16-byte boundaries in both)
    assert torch.equal(torch.autograd.grad(got, a, up)[0], torch.autograd.grad(want, b, up)[0])


def test_no_counted_rows_and_no_rows():
    z, idx, t, target = _case(5, 60, 3, F32)
    leaf = z.clone().requires_grad_(True)
    target[:] = IGNORE
    loss = distill_loss(leaf, idx, t, target, alpha=0.5, ignore_index=IGNORE)
    assert loss.isnan()  # 0 / 0, as torch's mean cross-entropy
    (dz,) = torch.autograd.grad(loss, leaf)
    assert not dz.any()
    assert distill_loss(z, idx, t, target, alpha=0.5, reduction="sum") == 0
    e = slice(0, 0)
    leaf = z[e].clone().requires_grad_(True)
    for reduction, want in (("mean", None), ("sum", 0.0)):
        loss = distill_loss(leaf, idx[e], t[e], target[e], alpha=0.5, reduction=reduction)
        assert loss.isnan() if want is None else float(loss) == want
        assert torch.autograd.grad(loss, leaf)[0].shape == (0, 60)
    assert distill_loss(z[e], idx[e], t[e], reduction="none").shape == (0,)
    assert distill_loss(z[e], idx[e], t[e]).isnan()


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_incoming_gradients(reduction):
    """Gradients other than 1 are folded in before the only rounding; a second
    backward, with the graph kept, gives the same."""
    z, idx, t, target = _case(30, 400, 10, BF)
    leaf = z.clone().requires_grad_(True)
    loss = distill_loss(leaf, idx, t, target, temperature=2.0, alpha=0.5, reduction=reduction)
    _, _, grad, size = _reference(z, idx, t, target, 2.0, 0.5)
    n = int((target != IGNORE).sum()) if reduction == "mean" else 1
    g = (torch.randn(30, generator=torch.Generator().manual_seed(0)).to(DEV)
         if reduction == "none" else torch.tensor(-1 / 3, device=DEV))
    f = (g[:, None] if reduction == "none" else g).double() / n
    (one,) = torch.autograd.grad(loss, leaf, g, retain_graph=True)
    _within(one, grad * f, _grad_tol(BF, grad * f, size * f.abs()), "gradient")
    (two,) = torch.autograd.grad(loss, leaf, g, retain_graph=True)
    assert torch.equal(one, two)
    ones = torch.ones_like(g)
    (a,) = torch.autograd.grad(loss, leaf, ones, retain_graph=True)
    fresh = z.clone().requires_grad_(True)
    again = distill_loss(fresh, idx, t, target, temperature=2.0, alpha=0.5, reduction=reduction)
    (b,) = torch.autograd.grad(again, fresh, ones)
    assert torch.equal(a, b)


def test_gradient_is_not_shared_between_backwards():
    z, idx, t, target = _case(10, 100, 4, F32)
    leaf = z.clone().requires_grad_(True)
    loss = distill_loss(leaf, idx, t, target, alpha=0.5)
    loss.backward(retain_graph=True)
    first = leaf.grad.clone()
    loss.backward()
    assert torch.equal(leaf.grad, 2 * first)


def test_logits_changed_before_the_backward_are_refused():
    z, idx, t, target = _case(10, 100, 4, F32)
    leaf = z.clone().requires_grad_(True)
    y = leaf * 1.0
    loss = distill_loss(y, idx, t, target, alpha=0.5)
    with torch.no_grad():
        y.zero_()
    with pytest.raises(RuntimeError, match="modified"):
        loss.backward()


@pytest.mark.parametrize("dt", [BF, F32])
def test_strides_alignments_and_leading_dimensions(dt):
    N, V, K = 12, 333, 7
    z, idx, t, target = _case(N, V, K, dt)
    kw = dict(temperature=2.0, alpha=0.5)

    def run(zz, ii, tt, gg):
        leaf = zz.detach().requires_grad_(True)
        loss = distill_loss(leaf, ii, tt, gg, **kw)
        return loss.detach(), torch.autograd.grad(loss, leaf)[0].reshape(N, V)

    want = run(z, idx, t, target)
    # Where a row starts between two 16-byte boundaries, the columns that a thread
    # adds up are others: another order of the same additions.  Each order's
    # result is within the tolerance of the sums (rel(S) holds for any chain of
    # that length), so that is what both have to keep.
    rows, tol, grad, size = _reference(z, idx, t, target, 2.0, 0.5)
    n = int((target != IGNORE).sum())
    wide = torch.full((N, V + 20), float("nan"), dtype=dt, device=DEV)
    for off in (0, 1, 8):
        view = wide[:, off:off + V]
        view.copy_(z)
        loss, dz = run(view, idx, t, target)
        _within(loss, rows.sum() / n, (tol.sum() + 4 * U * rows.abs().sum()) / n, "mean")
        _within(dz, grad / n, _grad_tol(dt, grad / n, size / n), "gradient")
    pad = torch.cat((idx, idx), 1)[:, :K], torch.cat((t, t), 1)[:, :K]
    for a, b in zip(run(z, *pad, target.int()), want):
        assert torch.equal(a, b)
    for a, b in zip(run(z.t().contiguous().t(), idx.t().contiguous().t(), t, target), want):
        assert torch.equal(a, b)
    lead = (3, 4)
    for a, b in zip(run(z.view(*lead, V), idx.view(*lead, K), t.view(*lead, K),
                        target.view(lead)), want):
        assert torch.equal(a, b)
    # one teacher for all rows
    a = run(z, idx[:1].expand(N, K), t[:1].expand(N, K), target)
    b = run(z, idx[:1].repeat(N, 1), t[:1].repeat(N, 1), target)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # a single row without leading dimensions
    x = distill_loss(z[0], idx[0], t[0], target[0], reduction="none", **kw)
    y = distill_loss(z[:1], idx[:1], t[:1], target[:1], reduction="none", **kw)
    assert x.shape == () and torch.equal(x, y[0])


def test_gradient_against_differences():
    """Central differences (h = 1e-4) of the row losses in 64 bits against the
    float32 gradient: the truncation, h^2 / 6 times a third derivative of at most
    a few |u|^3, is under 1e-7 of the sum taken here, the gradient's own
    tolerance under 1e-5 of it."""
    z, idx, t, target = _case(6, 40, 5, F32)
    leaf = z.clone().requires_grad_(True)
    rows = distill_loss(leaf, idx, t, target, temperature=2.0, alpha=0.6, reduction="none")
    (dz,) = torch.autograd.grad(rows, leaf, torch.ones_like(rows))
    gen = torch.Generator().manual_seed(5)
    f = lambda x: _reference(x, idx, t, target, 2.0, 0.6)[0].sum()  # noqa: E731
    for _ in range(5):
        u = torch.randn(z.shape, generator=gen, dtype=torch.float64).to(DEV)
        h = 1e-4
        diff = float((f(z.double() + h * u) - f(z.double() - h * u)) / (2 * h))
        size = float((dz.double() * u).abs().sum())
        assert abs(diff - float((dz.double() * u).sum())) <= 2e-5 * size


@pytest.mark.parametrize("tau", [0.01, 0.05, 30.0, 100.0])
def test_extreme_temperatures(tau):
    _check(*_case(6, 300, 8, F32), tau, 0.5)


def test_captured_loss_and_gradient():
    z, idx, t, target = _case(20, 1000, 8, BF)
    leaf = z.clone().requires_grad_(True)

    def step():
        loss = distill_loss(leaf, idx, t, target, temperature=2.0, alpha=0.5)
        return loss, torch.autograd.grad(loss, leaf)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, dz = step()
    for seed in range(3):
        new = _case(20, 1000, 8, BF, seed=60 + seed)
        with torch.no_grad():
            leaf.copy_(new[0])
        for a, b in zip((idx, t, target), new[1:]):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        fresh = new[0].clone().requires_grad_(True)
        want = distill_loss(fresh, *new[1:], temperature=2.0, alpha=0.5)
        assert torch.equal(loss, want.detach())
        assert torch.equal(dz, torch.autograd.grad(want, fresh)[0])


def test_another_stream():
    z, idx, t, target = _case(64, 5000, 8, BF)
    want = distill_loss(z, idx, t, target, alpha=0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaf = z.clone().requires_grad_(True)
        loss = distill_loss(leaf, idx.clone(), t.clone(), target.clone(), alpha=0.5)
        (dz,) = torch.autograd.grad(loss, leaf)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(loss.detach(), want) and dz.isfinite().all()


def test_custom_op():
    z, idx, t, target = _case(9, 100, 4, BF)
    for tg, alpha, red in ((target, 0.5, 2), (None, 1.0, 1), (target, 0.5, 0)):
        leaf = z.clone().requires_grad_(True)
        loss = torch.ops.t2t.distill_loss(leaf, idx, t, tg, 2.0, alpha, IGNORE, red)
        (dz,) = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
        other = z.clone().requires_grad_(True)
        want = distill_loss(other, idx, t, tg, temperature=2.0, alpha=alpha,
                            reduction=("none", "sum", "mean")[red])
        assert torch.equal(loss, want)
        assert torch.equal(dz, torch.autograd.grad(want, other, torch.ones_like(want))[0])
    torch.library.opcheck(torch.ops.t2t.distill_loss, (z, idx, t, target, 2.0, 0.5, IGNORE, 2))


def test_what_else_may_watch_a_call():
    """Traces hold the call, forward-mode levels and batched calls are refused;
    a function mode and recorded hooks see an ordinary call."""
    z, idx, t, target = _case(9, 100, 4, F32)

    def call(x):
        return distill_loss(x, idx, t, target, alpha=0.5)

    other = torch.randn_like(z)
    with torch.no_grad():
        traced = torch.jit.trace(call, z, check_trace=False)
        assert torch.equal(traced(other), call(other))
    with torch.no_grad(), fwad.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            call(fwad.make_dual(z, torch.ones_like(z)))
    with torch.no_grad(), pytest.raises(RuntimeError):
        torch.func.vmap(call)(torch.stack([z, z]))
    loss = call(z.requires_grad_(True))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, z, torch.ones(2, device=DEV), is_grads_batched=True)
    loss = call(z)
    (want,) = torch.autograd.grad(loss, z)
    with torch.autograd.graph.save_on_cpu():
        loss = call(z)
    assert torch.equal(torch.autograd.grad(loss, z)[0], want)
    again = torch.utils.checkpoint.checkpoint(call, z, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(again, z)[0], want)


@pytest.mark.parametrize("watched", [False, True])
def test_offloaded_graphs_keep_no_gradient(watched):
    """Where a user's hooks take what a graph saves, nothing of the logits' size
    stays on the GPU beside the logits themselves, and the gradient is the same."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    z, idx, t, target = _case(512, 8192, 4, F32)
    leaf = z.clone().requires_grad_(True)
    kw = dict(temperature=2.0, alpha=0.5, ignore_index=IGNORE)
    (want,) = torch.autograd.grad(distill_loss(leaf, idx, t, target, **kw), leaf)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    with torch.autograd.graph.save_on_cpu():
        if watched:
            with Watch():
                loss = distill_loss(leaf, idx, t, target, **kw)
        else:
            loss = distill_loss(leaf, idx, t, target, **kw)
    assert torch.cuda.memory_allocated() - before < z.numel() * 4 // 2
    assert torch.equal(torch.autograd.grad(loss, leaf)[0], want)


def test_second_order_is_refused():
    z, idx, t, target = _case(4, 50, 3, F32)
    leaf = z.clone().requires_grad_(True)
    loss = distill_loss(leaf, idx, t, target, alpha=0.5)
    (d,) = torch.autograd.grad(loss, leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), leaf)


def test_refusals():
    z, idx, t, target = _case(4, 50, 3, F32)
    with pytest.raises(RuntimeError, match="GPU"):
        distill_loss(z, idx.cpu(), t)
    with pytest.raises(RuntimeError, match="detach"):
        distill_loss(z, idx, t.clone().requires_grad_(True))
    with pytest.raises(RuntimeError, match="at most 1024"):
        distill_loss(z, idx.repeat(1, 400), t.repeat(1, 400))
    with pytest.raises(NotImplementedError, match="dtype"):
        distill_loss(z.half(), idx, t)
    with pytest.raises(RuntimeError, match="bf16 rows"):
        head_distill(z, z, idx, t)


# ---- with the head

def _head_case(N, C, V, K, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, C, generator=g).to(BF).to(DEV)
    w = (torch.randn(V, C, generator=g) * C ** -0.5).to(BF).to(DEV)
    _, idx, t, target = _case(N, V, K, BF, seed=seed)
    return x, w, idx, t, target


@pytest.mark.parametrize("chunk", [None, 7])
@pytest.mark.parametrize("wdt", [BF, F32])
def test_head_is_the_loss_of_its_logits(chunk, wdt):
    """head_distill against the row kernel on the same bf16 logits and products
    in 64 bits of the same bf16 logit gradients.  The chunk changes the library
    product that makes the logits at most, so losses agree to bf16 logits."""
    x, w, idx, t, target = _head_case(40, 64, 515, 6)
    w = w.to(wdt)
    kw = dict(temperature=2.0, alpha=0.5)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = head_distill(xl, wl, idx, t, target, chunk=chunk, **kw)
    gx, gw = torch.autograd.grad(loss, (xl, wl))
    logits = (x @ w.to(BF).t()).requires_grad_(True)
    rows = distill_loss(logits, idx, t, target, reduction="none", **kw)
    # a logit rounded the other way moves by 2^-7 of itself at most (one step),
    # and a loss by the sum of |gradient| that step
    _, _, grad, _ = _reference(logits.detach(), idx, t, target, 2.0, 0.5)
    n = int((target != IGNORE).sum())
    move = (grad.abs() * logits.detach().double().abs()).sum() * 2.0 ** -7 / n
    want = distill_loss(logits, idx, t, target, **kw)
    assert abs(float(loss) - float(want)) <= float(move) + 1e-6
    (d,) = torch.autograd.grad(want, logits)
    d64, x64, w64 = d.double(), x.double(), w.to(BF).double()
    # 2^-6: a moved logit's gradient, on top of bf16 sums and results
    for got, ref, size in ((gx, d64 @ w64, d64.abs() @ w64.abs()),
                           (gw, d64.t() @ x64, d64.abs().t() @ x64.abs())):
        assert got.dtype in (BF, wdt)
        _within(got, ref, 2.0 ** -6 * (ref.abs() + size) + 1e-6, "head gradient")
    with torch.no_grad():
        assert torch.equal(head_distill(x, w, idx, t, target, chunk=chunk, **kw), loss)
    assert rows.shape == (40,)


def test_head_gradients_of_a_third():
    """A loss divided by three: dx and dW are those of an incoming gradient of 1
    times g in fp32, rounded once more (U, and half a step of bf16 for dx)."""
    x, w, idx, t, target = _head_case(60, 64, 512, 6)
    kw = dict(temperature=2.0, alpha=0.5)
    w = w.float()
    g = torch.tensor(1 / 3, device=DEV)

    def grads(up):
        xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        return torch.autograd.grad(head_distill(xl, wl, idx, t, target, **kw), (xl, wl), up)

    for one, third in zip(grads(torch.ones_like(g)), grads(g)):
        ref = one.double() * g.double()
        tol = (torch.finfo(one.dtype).eps / 2 + U) * ref.abs()
        _within(third, ref, tol + 1e-37, "a third")


def test_head_gradients_of_a_batch():
    x, w, idx, t, target = _head_case(30, 64, 400, 5)
    x.requires_grad_(True), w.requires_grad_(True)
    loss = head_distill(x, w, idx, t, target, temperature=2.0, alpha=0.5)
    many = torch.tensor([1.0, 1 / 3, -2.0], device=DEV)
    dx, dw = torch.autograd.grad(loss, (x, w), many, is_grads_batched=True, retain_graph=True)
    for i, g in enumerate(many):
        a, b = torch.autograd.grad(loss, (x, w), g, retain_graph=True)
        assert torch.equal(dx[i], a) and torch.equal(dw[i], b)



@pytest.mark.parametrize("V", [512, 515])
def test_head_rows_that_do_not_count_may_hold_anything(V):
    """Rows of ignored targets with infinities and NaN: no share of the loss, and a
    gradient of zeros (that of the weight has 0 times them, as in torch)."""
    x, w, idx, t, target = _head_case(40, 64, V, 6)
    target[:] = torch.where(target == IGNORE, 1, target)
    target[3:5] = IGNORE
    kw = dict(temperature=2.0, alpha=0.5, ignore_index=IGNORE)
    want = head_distill(x, w, idx, t, target, **kw)
    x[3], x[4] = math.inf, math.nan
    xl = x.clone().requires_grad_(True)
    loss = head_distill(xl, w, idx, t, target, **kw)
    assert torch.equal(loss.detach(), want)
    (gx,) = torch.autograd.grad(loss, xl)
    assert not gx[3:5].any() and gx.isfinite().all() and gx[5].any()


def test_head_without_a_teacher_is_the_cross_entropy():
    """alpha 0: the loss of head_cross_entropy's logits, to the roundings of
    both row kernels (each under 1e-5 of a loss of about ln V)."""
    x, w, idx, t, target = _head_case(50, 64, 512, 4)
    a = head_distill(x, w, idx, t, target, alpha=0.0)
    b = head_cross_entropy(x, w, target, IGNORE)
    assert abs(float(a) - float(b)) <= 2e-5 * float(b)


def test_module():
    x, w, idx, t, target = _head_case(30, 64, 400, 5)
    m = LinearDistillLoss(64, 400, temperature=2.0, alpha=0.5, weight=torch.nn.Parameter(w))
    want = head_distill(x, w, idx, t, target, temperature=2.0, alpha=0.5)
    assert torch.equal(m(x.view(2, 15, 64), target.view(2, 15), idx.view(2, 15, 5),
                         t.view(2, 15, 5)).detach(), want)
    assert torch.equal(m(x, target).detach(), head_cross_entropy(x, w, target, IGNORE))
    with pytest.raises(ValueError, match="together"):
        m(x, target, idx)
    # no slots at all: the second part alone
    assert torch.equal(m(x, target, idx[:, :0], t[:, :0]).detach(),
                       head_distill(x, w, idx[:, :0], t[:, :0], target, temperature=2.0,
                                    alpha=0.5))
    # float32 rows: chunks of logits in float32, gradients by recomputation
    f = LinearDistillLoss(64, 400, temperature=2.0, alpha=0.5,
                          weight=torch.nn.Parameter(w.float()), chunk=8)
    xf = x.float().requires_grad_(True)
    loss = f(xf, target, idx, t)
    gx, gw = torch.autograd.grad(loss, (xf, f.weight))
    x64, w64 = xf.detach().double(), w.double()
    rows, tol, grad, _ = _reference(x64 @ w64.t(), idx, t, target, 2.0, 0.5)
    n = int((target != IGNORE).sum())
    # products of 64 terms in float32: logits within 64 U of their sums, a few
    # units each; 1e-4 holds 20 times that
    assert abs(float(loss) - float(rows.sum() / n)) <= 1e-4 * float(rows.sum() / n)
    _within(gx, grad @ w64 / n, 1e-4 * (grad.abs() @ w64.abs()) / n + 1e-9, "dx")
    _within(gw, grad.t() @ x64 / n, 1e-4 * (grad.abs().t() @ x64.abs()) / n + 1e-9, "dw")


def test_recomputed_chunks_keep_no_logits():
    """float32 rows of LinearDistillLoss: what lives between forward and backward
    is less than one chunk's logits, and at no time more than a few chunks'."""
    N, V, chunk = 2048, 8192, 256
    _, idx, t, target = _case(N, V, 4, F32)
    m = LinearDistillLoss(64, V, temperature=2.0, alpha=0.5, chunk=chunk).to(DEV)
    x = torch.randn(N, 64, device=DEV, requires_grad=True)
    torch.autograd.grad(m(x, target, idx, t), (x, m.weight))  # (what a first call loads stays)
    one = chunk * V * 4
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    loss = m(x, target, idx, t)
    assert torch.cuda.memory_allocated() - before < one
    torch.autograd.grad(loss, (x, m.weight))
    # a chunk's logits and their gradient, the weight's gradients (2 MB each)
    assert torch.cuda.max_memory_allocated() - before < 3 * one
